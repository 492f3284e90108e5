// linear_attention_core.h -- device side of linear attention with a decay for each head (linear_attention.hip).
//
// One head of one sequence, w = its decay, S the [d1][d2] state, tokens taken in chunks of C (in reverse time for the
// gradients of k and v):
//     P[i][j] = w^{i-j} (q_i . k_j) scale      for j <= i, else 0
//     O[i]    = w^{i+1-late} read * q_i S + sum_j P[i][j] v_j
//     S      <- w^C S + sum_j w^{C-1-j+late} write * k_j v_j^T
// A workgroup of four waves keeps the d1 x (64 NT) part of S in fp32 accumulators for its whole run over the tokens, so
// that the state never travels: q, k, v are read and o is written once.  Wave w owns 16 NT columns of S and of O.
//
// Every product is laid out so that accumulators become operands in place: S as accumulated (lane: column n = lane & 15,
// rows 4g .. 4g+3 of each 16-row tile, g = lane >> 4) is the A operand of O^T = S^T Q^T once the contraction index runs
// in the order {4g .. 4g+3, 16 + 4g .. 16 + 4g+3} of each 32 -- the order in which every fragment here is read, from rows
// (two 8-byte reads) or, transposed, from columns (two transposing LDS reads).  The V fragments serve O and S alike.
//
// Rounding (bf16): S and P are rounded to bf16 as operands of O -- each as much as the rounding of O itself -- while the
// running S takes w^{..} write v split into three bf16 parts (24 bits), so the state keeps fp32's accuracy over any
// length.  fp32 and fp16 samples are multiplied in fp32 (v_mfma_f32_16x16x4_f32): an fp16 state would overflow.
#pragma once

#include <type_traits>

#include "common.h"

namespace dspgpu {
namespace la {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kMaxHeads = 256;
constexpr int kMaxRoles = 3;

// One run of the operator: the forward pass has one, the backward pass three (gradients of q, k, v).
struct Role {
    const void *q, *k, *v;
    void *o;                       // sample type, or fp32 [row][heads][d2] where o_partial
    long long qs[3], ks[3], vs[3], os[3];  // strides in elements: sequence, token, head
    int q_group, k_group, v_group;  // heads that share one head of q / k / v
    int d1, d2, tiles;             // tiles of 64 NT columns
    int late;                      // 1: reverse time
    int o_partial;
    int vec;                       // bit 0..3: q, k, v, o take 16-byte (o: 4-element) accesses
    float read, write, pscale;
    const float *s_in;             // [sequence][head] blocks of d1 * d2, element (d, n) at d * s_in_d + n * s_in_n; or null
    int s_in_d, s_in_n;
    float *s_out;                  // [sequence][head][d1][d2] or null
    float *seg;                    // [sequence * heads + head][segments][d1][d2]: states of the segments (null: one segment)
};

struct Args {
    Role role[kMaxRoles];
    int roles;
    int heads, batch;
    int segments;
    long long seg_len;             // tokens of a segment, a multiple of the chunk
    long long n;                   // tokens of a sequence at most
    long long rows;                // rows of a packed batch
    const long long *offsets, *lengths;
    float log2_decay[kMaxHeads];
};

// Rows [start, start + len) of sequence b.  Offsets and lengths are data: whatever they hold, the rows stay inside.
__device__ __forceinline__ void sequence_rows(const Args &a, int b, long long &start, long long &len) {
    start = 0;
    len = a.n;
    if (a.offsets) {
        long long s = a.offsets[b], e = a.offsets[b + 1];
        s = s < 0 ? 0 : s > a.rows ? a.rows : s;
        e = e < s ? s : e > a.rows ? a.rows : e;
        start = s;
        len = e - s < a.n ? e - s : a.n;
    } else if (a.lengths) {
        const long long l = a.lengths[b];
        len = l < 0 ? 0 : l < a.n ? l : a.n;
    }
}

// w^n for n >= 0, from log2 w (-inf for w = 0: w^0 is still 1)
__device__ __forceinline__ float power(float log2w, float n) { return n == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(log2w * n); }

// w^n to 48 bits, for what multiplies a state again and again: rounded to 24 bits, w^C of a slow decay would be off by
// 2^-25 every C tokens, and the state by that times the number of chunks it remembers
struct Decay {
    float hi, lo;
};
__device__ __forceinline__ Decay decay_over(float log2w, long long n) {
    const double w = n == 0 ? 1.0 : exp2(static_cast<double>(log2w) * static_cast<double>(n));
    const float hi = static_cast<float>(w);
    return {hi, static_cast<float>(w - hi)};
}

template <typename Tc>
struct Cfg;
template <>
struct Cfg<__bf16> {
    typedef bf16x8 frag;
    static constexpr int kVe = 8, kPad = 8;
};
template <>
struct Cfg<float> {
    typedef f32x8 frag;
    static constexpr int kVe = 4, kPad = 4;
};

__device__ __forceinline__ void mma(f32x4 &acc, bf16x8 a, bf16x8 b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void mma(f32x4 &acc, f32x8 a, f32x8 b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
}

// 8 contraction elements of one row: columns 4g .. 4g+3 and 16 + 4g .. of the 32 at p (p: the row's first of these 32)
__device__ __forceinline__ bf16x8 row_frag(const __bf16 *p, int g) {
    const bf16x4 a = *reinterpret_cast<const bf16x4 *>(p + 4 * g), b = *reinterpret_cast<const bf16x4 *>(p + 16 + 4 * g);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 row_frag(const float *p, int g) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p + 4 * g), b = *reinterpret_cast<const f32x4 *>(p + 16 + 4 * g);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// 8 contraction elements of one column: rows 4g .. 4g+3 and 16 + 4g .. of the 32 rows at p, column lane & 15.
// The transposing read: the 16 lanes of a group fetch four rows of 16 elements, lane m gets column m of the four.
template <int STRIDE>
__device__ __forceinline__ bf16x8 col_frag(const __bf16 *p, int g, int m) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const __bf16 *r = p + (4 * g + (m >> 2)) * STRIDE + 4 * (m & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(r));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(r + 16 * STRIDE));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 ab = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, ab);
}
template <int STRIDE>
__device__ __forceinline__ f32x8 col_frag(const float *p, int g, int m) {
    f32x8 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        f[r] = p[(4 * g + r) * STRIDE + m];
        f[4 + r] = p[(16 + 4 * g + r) * STRIDE + m];
    }
    return f;
}

__device__ __forceinline__ bf16x8 operand(const f32x4 &a, const f32x4 &b, __bf16) {
    bf16x8 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        f[r] = static_cast<__bf16>(a[r]);
        f[4 + r] = static_cast<__bf16>(b[r]);
    }
    return f;
}
__device__ __forceinline__ f32x8 operand(const f32x4 &a, const f32x4 &b, float) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// ---- global <-> registers ----------------------------------------------------------------------------------------------

template <typename T, int N>
struct Pack {
    T e[N];
};

// VE consecutive elements of a row, zeros from column `cols` on
template <typename Ti, int VE>
__device__ __forceinline__ Pack<Ti, VE> load_pack(const Ti *row, int col, int cols, bool vec) {
    Pack<Ti, VE> r;
    typedef int raw __attribute__((ext_vector_type(VE * sizeof(Ti) / 4)));
    if (vec) {  // cols is a multiple of VE and the row aligned
        raw v = {};
        if (col < cols) v = *reinterpret_cast<const raw *>(row + col);
        __builtin_memcpy(&r, &v, sizeof r);
    } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) r.e[e] = col + e < cols ? row[col + e] : static_cast<Ti>(0.0f);
    }
    return r;
}

__device__ __forceinline__ void to_lds(__bf16 *p, const Pack<__bf16, 8> &v) { *reinterpret_cast<bf16x8 *>(p) = __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ void to_lds(float *p, const Pack<float, 4> &v) { *reinterpret_cast<f32x4 *>(p) = __builtin_bit_cast(f32x4, v); }
__device__ __forceinline__ void to_lds(float *p, const Pack<_Float16, 4> &v) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{static_cast<float>(v.e[0]), static_cast<float>(v.e[1]), static_cast<float>(v.e[2]), static_cast<float>(v.e[3])};
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const f32x4 &v, int left, bool vec) {
    if (vec) {
        if (left >= 4) {
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(v[r]);
            *reinterpret_cast<t4 *>(p) = o;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < left) p[r] = static_cast<T>(v[r]);
    }
}

// ---- the kernel ------------------------------------------------------------------------------------------------------

template <typename Tc, int D1P, int NT, int C>
struct Lds {
    static constexpr int kPad = Cfg<Tc>::kPad;
    static constexpr int kD = D1P + kPad, kN = 64 * NT + kPad, kP = C + kPad;
    Tc q[C * kD];
    Tc k[C * kD];
    Tc v[C * kN];
    Tc p[C * kP];
    float pw[C + 4];
};
template <typename Tc, int D1P, int NT, int C>
struct LdsState {  // no queries
    static constexpr int kPad = Cfg<Tc>::kPad;
    static constexpr int kD = D1P + kPad, kN = 64 * NT + kPad, kP = 0;
    Tc k[C * kD];
    Tc v[C * kN];
    float pw[C + 4];
};

// STATE_ONLY: the state a segment leaves behind when it starts from zero -> seg[segment]
template <typename Ti, typename Tc, int D1P, int NT, int C, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads, 2) linear_attention_kernel(const Args a) {
    using F = typename Cfg<Tc>::frag;
    using L = typename std::conditional<STATE_ONLY, LdsState<Tc, D1P, NT, C>, Lds<Tc, D1P, NT, C>>::type;
    constexpr int VE = Cfg<Tc>::kVe;
    constexpr int KB = D1P / 32, DT = D1P / 16, IT = C / 16, JB = C / 32, NB = 64 * NT;
    constexpr int QV = C * D1P / VE / kThreads, VV = C * NB / VE / kThreads;  // packs a thread moves
    static_assert(QV * VE * kThreads == C * D1P && VV * VE * kThreads == C * NB, "whole packs");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    L &lds = *reinterpret_cast<L *>(smem);

    // workgroup -> (segment, sequence, head, role, tile): the tiles and roles of a head next to each other
    unsigned id = blockIdx.x;
    int role_tiles = 0;
    for (int r = 0; r < a.roles; ++r) role_tiles += a.role[r].tiles;
    int t = id % role_tiles;
    id /= role_tiles;
    const int head = id % a.heads;
    id /= a.heads;
    const int b = id % a.batch;
    const int segment = id / a.batch;
    int ri = 0;
    while (t >= a.role[ri].tiles) t -= a.role[ri++].tiles;
    const Role &role = a.role[ri];
    const int n0 = t * NB;

    long long start, len;
    sequence_rows(a, b, start, len);
    const long long u0 = segment * a.seg_len, u1 = min(len, u0 + a.seg_len);  // in the order of traversal
    const bool split = role.seg != nullptr;
    if (u0 >= u1 && (split || !role.s_out)) return;  // an empty sequence still hands its state on

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
    const int d1 = role.d1, d2 = role.d2;
    const float log2w = a.log2_decay[head];
    const size_t bh = static_cast<size_t>(b) * a.heads + head;
    const long long base = a.offsets ? 0 : b;  // packed rows have no sequence stride
    const Ti *q = static_cast<const Ti *>(role.q) + base * role.qs[0] + start * role.qs[1] + (head / role.q_group) * role.qs[2];
    const Ti *k = static_cast<const Ti *>(role.k) + base * role.ks[0] + start * role.ks[1] + (head / role.k_group) * role.ks[2];
    const Ti *v = static_cast<const Ti *>(role.v) + base * role.vs[0] + start * role.vs[1] + (head / role.v_group) * role.vs[2] + n0;
    const bool qvec = role.vec & 1, kvec = role.vec & 2, vvec = role.vec & 4, ovec = role.vec & 8;

    if (tid <= C) lds.pw[tid] = power(log2w, static_cast<float>(tid));

    // the state: lane holds rows 16 dt + 4g + r, column n0 + 16 (NT wave + nt) + m
    f32x4 S[DT][NT];
    {
        const float *s_in = nullptr;
        size_t sd = 0, sn = 1;
        if constexpr (!STATE_ONLY) {
            if (split) {
                s_in = role.seg + (bh * a.segments + segment) * d1 * d2;
                sd = d2;
            } else if (role.s_in) {
                s_in = role.s_in + bh * d1 * d2;
                sd = role.s_in_d;
                sn = role.s_in_n;
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = n0 + 16 * (NT * wave + nt) + m;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r;
                    S[dt][nt][r] = s_in && d < d1 && n < d2 ? s_in[d * sd + n * sn] : 0.0f;
                }
            }
    }

    Pack<Ti, VE> rq[STATE_ONLY ? 1 : QV], rk[QV], rv[VV];
    // rows u .. u + C of the traversal into registers, zeros behind the last one
    auto fetch = [&](long long u) {
#pragma unroll
        for (int x = 0; x < QV; ++x) {
            const int at = (x * kThreads + tid) * VE, row = at / D1P, col = at % D1P;
            const long long uu = u + row, tt = role.late ? len - 1 - uu : uu;
            const bool in = uu < u1;
            rk[x] = load_pack<Ti, VE>(k + (in ? tt : 0) * role.ks[1], col, in ? d1 : 0, kvec);
            if constexpr (!STATE_ONLY) rq[x] = load_pack<Ti, VE>(q + (in ? tt : 0) * role.qs[1], col, in ? d1 : 0, qvec);
        }
#pragma unroll
        for (int x = 0; x < VV; ++x) {
            const int at = (x * kThreads + tid) * VE, row = at / NB, col = at % NB;
            const long long uu = u + row, tt = role.late ? len - 1 - uu : uu;
            const bool in = uu < u1;
            rv[x] = load_pack<Ti, VE>(v + (in ? tt : 0) * role.vs[1], col, in ? d2 - n0 : 0, vvec);
        }
    };
    auto commit = [&]() {
#pragma unroll
        for (int x = 0; x < QV; ++x) {
            const int at = (x * kThreads + tid) * VE, row = at / D1P, col = at % D1P;
            to_lds(lds.k + row * L::kD + col, rk[x]);
            if constexpr (!STATE_ONLY) to_lds(lds.q + row * L::kD + col, rq[x]);
        }
#pragma unroll
        for (int x = 0; x < VV; ++x) {
            const int at = (x * kThreads + tid) * VE, row = at / NB, col = at % NB;
            to_lds(lds.v + row * L::kN + col, rv[x]);
        }
    };

    const Decay whole = decay_over(log2w, C);
    if (u0 < u1) {
        fetch(u0);
        commit();
    }
    __syncthreads();

    for (long long u = u0; u < u1; u += C) {
        const int size = static_cast<int>(min(static_cast<long long>(C), u1 - u));
        const bool more = u + C < u1;
        if (more) fetch(u + C);

        f32x4 O[STATE_ONLY ? 1 : IT][NT];
        if constexpr (!STATE_ONLY) {
            // P^T = K Q^T: wave w takes the keys of tile w % IT for every (4 / IT)-th tile of queries
            const int jt = wave % IT;
            F sf[KB][NT], kf[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                kf[kb] = row_frag(lds.k + (16 * jt + m) * L::kD + 32 * kb, g);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sf[kb][nt] = operand(S[2 * kb][nt], S[2 * kb + 1][nt], Tc());
            }
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                F qf[KB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) qf[kb] = row_frag(lds.q + (16 * it + m) * L::kD + 32 * kb, g);
                const float rd = role.read * lds.pw[16 * it + m + 1 - role.late];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    f32x4 acc = {};
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) mma(acc, sf[kb][nt], qf[kb]);
                    O[it][nt] = acc * rd;
                }
                if (it % (4 / IT) == wave / IT && jt / 2 <= it / 2) {
                    f32x4 p = {};
                    if (jt <= it) {
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) mma(p, kf[kb], qf[kb]);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int gap = 16 * (it - jt) + m - 4 * g - r;
                        p[r] = gap >= 0 ? p[r] * (role.pscale * lds.pw[gap < 0 ? 0 : gap]) : 0.0f;
                    }
                    store4(lds.p + (16 * it + m) * L::kP + 16 * jt + 4 * g, p, 4, true);
                }
            }
            __syncthreads();
        }

        F vf[JB][NT];
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) vf[jb][nt] = col_frag<L::kN>(lds.v + 32 * jb * L::kN + 16 * (NT * wave + nt), g, m);

        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int it = 0; it < IT; ++it) {
#pragma unroll
                for (int jb = 0; jb <= it / 2; ++jb) {
                    const F pf = row_frag(lds.p + (16 * it + m) * L::kP + 32 * jb, g);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma(O[it][nt], vf[jb][nt], pf);
                }
                if (16 * it + m < size) {
                    const long long uu = u + 16 * it + m, tt = start + (role.late ? len - 1 - uu : uu);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int n = n0 + 16 * (NT * wave + nt) + 4 * g;
                        const long long at = base * role.os[0] + tt * role.os[1] + head * role.os[2] + n;
                        if (role.o_partial) store4(static_cast<float *>(role.o) + at, O[it][nt], d2 - n, ovec);
                        else store4(static_cast<Ti *>(role.o) + at, O[it][nt], d2 - n, ovec);
                    }
                }
            }
        }

        // S <- w^size S + K^T diag(w^{size-1-j+late} write) V, the weighted V in three bf16 parts (fp32: in one)
        const Decay wc = size == C ? whole : decay_over(log2w, size);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) S[dt][nt] = S[dt][nt] * wc.hi + S[dt][nt] * wc.lo;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
            float wj[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = 32 * jb + 16 * (e >> 2) + 4 * g + (e & 3);
                wj[e] = j < size ? role.write * lds.pw[size - 1 - j + role.late] : 0.0f;
            }
            constexpr int PARTS = sizeof(Tc) == 2 ? 3 : 1;
            F part[PARTS][NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = static_cast<float>(vf[jb][nt][e]) * wj[e];
#pragma unroll
                    for (int s = 0; s < PARTS; ++s) {
                        part[s][nt][e] = static_cast<Tc>(x);
                        x -= static_cast<float>(part[s][nt][e]);
                    }
                }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const F kt = col_frag<L::kD>(lds.k + 32 * jb * L::kD + 16 * dt, g, m);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int s = PARTS - 1; s >= 0; --s) mma(S[dt][nt], kt, part[s][nt]);
            }
        }
        __syncthreads();
        if (more) {
            commit();
            __syncthreads();
        }
    }

    float *s_out = nullptr;
    if constexpr (STATE_ONLY) s_out = role.seg + (bh * a.segments + segment) * d1 * d2;
    else if (!split && role.s_out) s_out = role.s_out + bh * d1 * d2;
    if (s_out) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = n0 + 16 * (NT * wave + nt) + m;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r;
                    if (d < d1 && n < d2) s_out[static_cast<size_t>(d) * d2 + n] = S[dt][nt][r];
                }
            }
    }
}

// D1P and NT by the host's rule; C by the type: 64 tokens, 32 where an element is four bytes or a row 256 of them (LDS)
template <typename Ti, typename Tc, int D1P, int NT>
int launch_one(const Args &a, unsigned blocks, bool state_only, hipStream_t s) {
    constexpr int C = sizeof(Tc) == 2 && D1P <= 128 ? 64 : 32;
    if (state_only) {
        using L = LdsState<Tc, D1P, NT, C>;
        const auto fn = linear_attention_kernel<Ti, Tc, D1P, NT, C, true>;
        if (sizeof(L) > 65536)
            if (int rc = allow_full_lds(reinterpret_cast<const void *>(fn))) return rc;
        fn<<<blocks, kThreads, sizeof(L), s>>>(a);
    } else {
        using L = Lds<Tc, D1P, NT, C>;
        const auto fn = linear_attention_kernel<Ti, Tc, D1P, NT, C, false>;
        if (sizeof(L) > 65536)
            if (int rc = allow_full_lds(reinterpret_cast<const void *>(fn))) return rc;
        fn<<<blocks, kThreads, sizeof(L), s>>>(a);
    }
    return check_launch("linear_attention_kernel");
}

template <typename Ti, typename Tc>
int launch_any(const Args &a, int d1p, int nt, unsigned blocks, bool state_only, hipStream_t s) {
    if (d1p == 64) return nt == 1 ? launch_one<Ti, Tc, 64, 1>(a, blocks, state_only, s) : launch_one<Ti, Tc, 64, 2>(a, blocks, state_only, s);
    if (d1p == 128) return nt == 1 ? launch_one<Ti, Tc, 128, 1>(a, blocks, state_only, s) : launch_one<Ti, Tc, 128, 2>(a, blocks, state_only, s);
    return launch_one<Ti, Tc, 256, 1>(a, blocks, state_only, s);
}

// one translation unit each
int launch_bf16(const Args &a, int d1p, int nt, unsigned blocks, bool state_only, hipStream_t s);
int launch_f16(const Args &a, int d1p, int nt, unsigned blocks, bool state_only, hipStream_t s);
int launch_f32(const Args &a, int d1p, int nt, unsigned blocks, bool state_only, hipStream_t s);

}  // namespace la
}  // namespace dspgpu
