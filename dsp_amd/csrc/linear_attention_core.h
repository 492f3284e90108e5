// linear_attention_core.h -- device side of linear attention with a decay for each head (linear_attention.hip).
//
// One head of one sequence, w = its decay, S the [d1][d2] state, tokens taken in chunks of C (in reverse time for the
// gradients of k and v):
//     P[i][j] = w^{i-j} (q_i . k_j) scale      for j <= i, else 0
//     O[i]    = w^{i+1} read * q_i S + sum_j P[i][j] v_j
//     S      <- w^C S + sum_j w^{C-1-j} write * k_j v_j^T
// In reverse time the chunks come last to first, the tokens of one stay in their places, and every weight is mirrored:
//     P[i][j] = w^{j-i} ... for j >= i,   O[i] = w^{C-1-i} read ...,   S <- w^C S + sum_j w^{j+1} write ...
// A workgroup of four waves keeps the d1 x (64 NT) part of S in fp32 accumulators for its whole run over the tokens, so
// that the state never travels: q, k, v are read and o is written once.  Wave w owns 16 NT columns of S and of O.
//
// Every product is laid out so that accumulators become operands in place: S as accumulated (lane: column n = lane & 15,
// rows 4g .. 4g+3 of each 16-row tile, g = lane >> 4) is the A operand of O^T = S^T Q^T once the contraction index runs
// in the order {4g .. 4g+3, 16 + 4g .. 16 + 4g+3} of each 32 -- the order in which every fragment here is read, from rows
// (two 8-byte reads) or, transposed, from columns (two transposing LDS reads).  The V fragments serve O and S alike.
//
// Rounding (bf16): S and P are rounded to bf16 as operands of O -- together they add as much error as the rounding of O
// itself (0.0023 against 0.0017 relative) -- while the running S takes w^{..} write v split into three bf16 parts (24 bits),
// so the state keeps fp32's accuracy over any length (two parts: 6e-7 of it lost for 13 % of the time).  fp32 and fp16
// samples are multiplied in fp32 (v_mfma_f32_16x16x4_f32): an fp16 state would overflow.
//
// What bounds it, at 32,768 tokens x 16 heads of 128 x 128 bf16 (32 segments, two workgroups of four waves a CU): 148 us for
// 537 MB of q, k, v and o, 3.6 TB/s; the same walk over memory without the arithmetic takes 95 us.  The matrix pipes are busy
// in a quarter of the SIMDs' cycles, and a wave issues vector instructions in a fifth of its own; the rest waits for LDS, for
// the partner wave and for memory.  The pass that finds the segments' states: 74 us for 268 MB of k and v.  Measured and not
// kept, when the same took 140 us: eight waves of 128 registers (160 us), chunks of 32 tokens (three workgroups a CU, spills:
// 285 us), LDS reads a step ahead of the products (140 us), workgroups dealt to the XCDs by segment (140 us), q and P stored
// in the order they are read (142 us).
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
// Up to so many segments a workgroup of the last pass joins the states before its own itself: that reads them
// segments / 2 times instead of twice and a write, but saves a kernel that runs by itself.
constexpr int kJoinSelf = 6;

// One run of the operator: the forward pass has one, the backward pass three (gradients of q, k, v).
struct Role {
    const void *q, *k, *v;
    void *o;                       // sample type, or fp32 [row][heads][d2] where o_partial
    long long qs[3], ks[3], vs[3], os[3];  // strides in elements: sequence, token, head
    int q_group, k_group, v_group;  // heads that share one head of q / k / v
    int d1, d2, tiles;             // tiles of 64 NT columns
    int late;                      // 1: reverse time
    int o_partial;
    int vec;                       // rows of q, k, v are whole aligned packs, rows of o whole aligned quads
    float read, write, pscale;
    const float *s_in;             // [sequence][head] blocks of d1 * d2, element (d, n) at d * s_in_d + n * s_in_n; or null
    int s_in_d, s_in_n;
    float *s_out;                  // [sequence][head][d1][d2] or null
    float *seg;                    // [head][slot][d1][d2]: states between the segments (Slots)
};

struct Args {
    Role role[kMaxRoles];
    int roles;
    int heads, batch;
    unsigned blocks;               // workgroups that have work
    int segments;                  // of the longest sequence that there can be
    unsigned slots;                // states between the segments, for each head
    int in_place;                  // s_out is s_in, and there are segments (copy_states_kernel)
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

// The last sequence of a packed batch that starts at or before `row` (or the first one).
__device__ __forceinline__ int sequence_at(const Args &a, long long row) {
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.offsets[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Segments of a sequence with another one behind them: those that leave a state between the segments.
__device__ __forceinline__ int inner_segments(const Args &a, long long len) {
    return len > 0 ? static_cast<int>(static_cast<unsigned>(len - 1) / static_cast<unsigned>(a.seg_len)) : 0;
}

// Which slot holds the state that segment s of a sequence leaves behind: first + s * step.  A dense batch has segments - 1
// slots for each sequence.  The inner segments of a packed one are seg_len rows each that no other has, so the numbers
// (first row of it) / seg_len are all different and below rows / seg_len: that many slots, however the rows are dealt out.
struct Slots {
    int first, step;
};
__device__ __forceinline__ Slots slots_of(const Args &a, int late, int b, long long start, long long len) {
    if (!a.offsets) return {b * (a.segments - 1), 1};
    const unsigned l = static_cast<unsigned>(a.seg_len);
    return late ? Slots{static_cast<int>(static_cast<unsigned>(start + len) / l) - 1, -1} : Slots{static_cast<int>(static_cast<unsigned>(start) / l), 1};
}

// w^n for n >= 0, from log2 w (-inf for w = 0: w^0 is still 1)
__device__ __forceinline__ float power(float log2w, float n) { return n == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(log2w * n); }

// w^n as a sum of two floats, for what multiplies a state again and again: rounded to 24 bits, w^C of a slow decay would be
// off by 2^-25 every C tokens, and the state by that times the number of chunks it remembers.  (log2 w itself has 24 bits,
// like the weights within a chunk: the rate of the decay is off by 2^-25 of itself, over any number of tokens.)  Both parts
// are positive, so that an infinite state times each of them is no NaN; the least lo adds nothing to a finite product.
struct Decay {
    float hi, lo;
};
__host__ __device__ inline Decay two_parts(double w) {
    float hi = static_cast<float>(w);
    if (hi > w) hi = __builtin_bit_cast(float, __builtin_bit_cast(int, hi) - 1);
    const float lo = static_cast<float>(w - hi), least = hi * 0x1p-40f;
    return {hi, lo > least ? lo : least};
}
__device__ __forceinline__ Decay decay_over(float log2w, long long n) {
    return two_parts(n == 0 ? 1.0 : exp2(static_cast<double>(log2w) * static_cast<double>(n)));
}

template <typename Tc>
struct Cfg;
template <>
struct Cfg<__bf16> {
    typedef bf16x8 frag;
    static constexpr int kVe = 8, kPad = 8, kPadT = 16;  // of rows read along / across: no two lanes of 32 share a bank
};
template <>
struct Cfg<float> {
    typedef f32x8 frag;
    static constexpr int kVe = 4, kPad = 4, kPadT = 4;
};

__device__ __forceinline__ void mma(f32x4 &acc, bf16x8 a, bf16x8 b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void mma(f32x4 &acc, f32x8 a, f32x8 b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
}

// Sixteen wait states between matrix products and whatever reads their results after them (eleven are needed).  hipcc 7.2
// leaves them out where the reader opens a block behind two uniform branches: halves of accumulators were stored stale.
__device__ __forceinline__ void settle(f32x4 &a) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(a)); }
__device__ __forceinline__ void settle(f32x4 &a, f32x4 &b) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void settle(f32x4 &a, f32x4 &b, f32x4 &c, f32x4 &d) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(a), "+v"(b), "+v"(c), "+v"(d)); }
template <int N>
__device__ __forceinline__ void settle(f32x4 (&x)[N]) {
    if constexpr (N >= 8) asm volatile("s_nop 7\n\ts_nop 7" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
    if constexpr (N == 16) asm volatile("s_nop 7\n\ts_nop 7" : "+v"(x[8]), "+v"(x[9]), "+v"(x[10]), "+v"(x[11]), "+v"(x[12]), "+v"(x[13]), "+v"(x[14]), "+v"(x[15]));
    if constexpr (N == 4) settle(x[0], x[1], x[2], x[3]);
    if constexpr (N == 2) settle(x[0], x[1]);
    if constexpr (N == 1) settle(x[0]);
}

// Two wait states between what inline assembly has written and the matrix products that read it: hipcc puts them behind vector
// instructions that it knows of.
template <int N>
__device__ __forceinline__ void ready(f32x4 (&x)[N]) {
    static_assert(N == 4 || N == 8 || N == 16, "states of 64, 128, 256 rows");
    if constexpr (N >= 8) asm volatile("s_nop 1" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
    if constexpr (N == 16) asm volatile("s_nop 1" : "+v"(x[8]), "+v"(x[9]), "+v"(x[10]), "+v"(x[11]), "+v"(x[12]), "+v"(x[13]), "+v"(x[14]), "+v"(x[15]));
    if constexpr (N == 4) asm volatile("s_nop 1" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
}

// adds 0 if all of a lane group's elements are finite, else NaN somewhere
__device__ __forceinline__ void times_zero(f32x4 &acc, bf16x8 a) { mma(acc, a, bf16x8{}); }
__device__ __forceinline__ void times_zero(f32x4 &acc, f32x8 a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e & 3] += a[e] * 0.0f;
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

// part[0] + part[1] + part[2] = v w to 24 bits, two elements at a time
template <int NT>
__device__ __forceinline__ void split(bf16x8 (&part)[3][NT], int nt, const bf16x8 &v, const float (&w)[8]) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const u32x4 in = __builtin_bit_cast(u32x4, v);
    u32x4 out[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x = __uint_as_float(in[i] << 16) * w[2 * i], y = __uint_as_float(in[i] & 0xffff0000u) * w[2 * i + 1];
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            const unsigned xy = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{x, y}), bf16x2));
            out[s][i] = xy;
            x -= __uint_as_float(xy << 16);
            y -= __uint_as_float(xy & 0xffff0000u);
        }
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) part[s][nt] = __builtin_bit_cast(bf16x8, out[s]);
}
template <int NT>
__device__ __forceinline__ void split(f32x8 (&part)[1][NT], int nt, const f32x8 &v, const float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) part[0][nt][e] = v[e] * w[e];
}

// ---- global <-> registers ----------------------------------------------------------------------------------------------

template <typename T, int N>
struct Pack {
    T e[N];
};

// Rows are reached through buffer descriptors that start at a chunk's first row: a lane whose row or column lies outside
// gets an offset past the descriptor's end, reads zeros and writes nothing, and no load or store sits behind a branch.
// (Offset and step are below 2^29 each for everything inside, so the end is out of reach for those.)
constexpr int kRecords = 0x7fffffff;
constexpr unsigned kOutside = 0xc0000000u;  // with or without a step

__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, kRecords, 0x00027000);
}

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <typename Ti, int VE>
__device__ __forceinline__ Pack<Ti, VE> load_pack(__amdgpu_buffer_rsrc_t r, unsigned offset, int step) {
    if constexpr (sizeof(Ti) * VE == 16) return __builtin_bit_cast(Pack<Ti, VE>, __builtin_amdgcn_raw_buffer_load_b128(r, offset, step, 0));
    else return __builtin_bit_cast(Pack<Ti, VE>, __builtin_amdgcn_raw_buffer_load_b64(r, offset, step, 0));
}
// the same element by element, for rows that are not whole aligned packs: the first `left` of VE, zeros behind them
template <typename Ti, int VE>
__device__ __forceinline__ Pack<Ti, VE> load_elements(const Ti *p, int left) {
    Pack<Ti, VE> r;
#pragma unroll
    for (int e = 0; e < VE; ++e) r.e[e] = e < left ? p[e] : static_cast<Ti>(0.0f);
    return r;
}

__device__ __forceinline__ void to_lds(__bf16 *p, const Pack<__bf16, 8> &v) { *reinterpret_cast<bf16x8 *>(p) = __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ void to_lds(float *p, const Pack<float, 4> &v) { *reinterpret_cast<f32x4 *>(p) = __builtin_bit_cast(f32x4, v); }
__device__ __forceinline__ void to_lds(float *p, const Pack<_Float16, 4> &v) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{static_cast<float>(v.e[0]), static_cast<float>(v.e[1]), static_cast<float>(v.e[2]), static_cast<float>(v.e[3])};
}

template <typename T>
__device__ __forceinline__ void to_lds4(T *p, const f32x4 &v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(v[r]);
    *reinterpret_cast<t4 *>(p) = o;
}
template <typename T>
__device__ __forceinline__ void store_quad(__amdgpu_buffer_rsrc_t r, unsigned offset, int step, const f32x4 &v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(v[e]);
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, o), r, offset, step, 0);
    else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i32x2, o), r, offset, step, 0);
}
template <typename T>
__device__ __forceinline__ void store_elements(T *p, const f32x4 &v, int left) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < left) p[r] = static_cast<T>(v[r]);
}

// ---- the kernel ------------------------------------------------------------------------------------------------------

template <typename Tc, int D1P, int NT, int C>
struct Lds {
    static constexpr int kPad = Cfg<Tc>::kPad, kPadT = Cfg<Tc>::kPadT;
    static constexpr int kQ = D1P + kPad, kD = D1P + kPadT, kN = 64 * NT + kPadT, kP = C + kPad;
    float pw[2 * C + 4];  // w^|x| at C + x; in front, where the offsets of paired reads reach
    float pm[2 * C + 4];  // the same, below zero on the side that P leaves out (a weight may itself come to zero)
    Tc q[C * kQ];
    Tc k[C * kD];
    Tc v[C * kN];
    Tc p[C * kP];
};
template <typename Tc, int D1P, int NT, int C>
struct LdsState {  // no queries
    static constexpr int kPadT = Cfg<Tc>::kPadT;
    static constexpr int kQ = 0, kD = D1P + kPadT, kN = 64 * NT + kPadT, kP = 0;
    float pw[2 * C + 4];
    Tc k[C * kD];
    Tc v[C * kN];
};

// STATE_ONLY: the state a segment leaves behind when it starts from zero -> seg[segment], for all but a sequence's last.
// VEC: rows of q, k, v are whole aligned packs, rows of o whole aligned quads, and a chunk of any of them spans < 2^29 bytes.
template <typename Ti, typename Tc, int D1P, int NT, int C, bool STATE_ONLY, bool VEC, bool late>
__device__ __forceinline__ void linear_attention_body(const Args &a, const Role &role, int n0, int head, int b, long long start, long long len, int segment, Slots slots) {
    using F = typename Cfg<Tc>::frag;
    using L = typename std::conditional<STATE_ONLY, LdsState<Tc, D1P, NT, C>, Lds<Tc, D1P, NT, C>>::type;
    constexpr int VE = Cfg<Tc>::kVe;
    constexpr int KB = D1P / 32, DT = D1P / 16, IT = C / 16, JB = C / 32, NB = 64 * NT;
    constexpr int QV = C * D1P / VE / kThreads, VV = C * NB / VE / kThreads;      // packs a thread moves
    constexpr int QROWS = kThreads * VE / D1P, VROWS = kThreads * VE / NB;        // rows between them
    static_assert(QV * QROWS == C && VV * VROWS == C, "whole packs");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    L &lds = *reinterpret_cast<L *>(smem);

    const long long u0 = segment * a.seg_len, u1 = min(len, u0 + a.seg_len);  // in the order of traversal
    if (STATE_ONLY && u1 >= len) return;
    if (u0 >= u1 && (segment > 0 || !role.s_out)) return;  // an empty sequence still hands its state on

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, m = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same in all its lanes: branches on it are scalar
    const int d1 = role.d1, d2 = role.d2;
    // fp32 products are a sixteenth as fast as bf16's, and what bounds their kernels: steps behind d1, and waves behind d2,
    // leave them out (gradients of 11 x 1200 tokens of 14 heads of 192 x 16 in fp16: 485 us, with them 621).
    constexpr bool kTrim = sizeof(Tc) == 4;
    const bool busy = n0 + 16 * NT * wave < d2;
    const float log2w = a.log2_decay[head], read = role.read, write = role.write, pscale = role.pscale;
    const size_t bh = static_cast<size_t>(b) * a.heads + head;
    const long long base = a.offsets ? 0 : b;  // packed rows have no sequence stride
    const long long qt = role.qs[1], kt = role.ks[1], vt = role.vs[1], ot = role.os[1];
    const Ti *q = static_cast<const Ti *>(role.q) + base * role.qs[0] + start * qt + (head / role.q_group) * role.qs[2];
    const Ti *k = static_cast<const Ti *>(role.k) + base * role.ks[0] + start * kt + (head / role.k_group) * role.ks[2];
    const Ti *v = static_cast<const Ti *>(role.v) + base * role.vs[0] + start * vt + (head / role.v_group) * role.vs[2] + n0;
    const bool partial = role.o_partial;
    const int osize = partial ? 4 : static_cast<int>(sizeof(Ti));
    char *o = static_cast<char *>(role.o) + (base * role.os[0] + start * ot + head * role.os[2] + n0) * osize;

    for (int x = tid; x <= 2 * C; x += kThreads) {
        const float w = power(log2w, static_cast<float>(x < C ? C - x : x - C));
        lds.pw[x] = w;
        if constexpr (!STATE_ONLY) lds.pm[x] = (late ? x <= C : x >= C) ? w : -1.0f;
    }

    // the state: lane holds rows 16 dt + 4g + r, column n0 + 16 (NT wave + nt) + m
    f32x4 S[DT * NT];
    auto load_state = [&](f32x4(&x)[DT * NT], const float *p, int sd, int sn) {
        const auto from = descriptor(p);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = n0 + 16 * (NT * wave + nt) + m;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r;
                    const unsigned at = p && d < d1 && n < d2 ? (d * sd + n * sn) * 4u : kOutside;
                    x[dt * NT + nt][r] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
                }
            }
    };
    auto seg = [&](int s) { return role.seg + (static_cast<size_t>(head) * a.slots + slots.first + s * slots.step) * d1 * d2; };
    const bool joined = a.segments > kJoinSelf;
    if (STATE_ONLY) {
        load_state(S, nullptr, 0, 0);
    } else if (segment > 0 && joined) {
        load_state(S, seg(segment - 1), d2, 1);
    } else {
        load_state(S, role.s_in ? role.s_in + bh * d1 * d2 : nullptr, role.s_in_d, role.s_in_n);
        if (segment > 0) {  // the few segments before this one, joined on the spot
            const Decay w = decay_over(log2w, a.seg_len);
            for (int s = 0; s < segment; ++s) {
                f32x4 local[DT * NT];
                load_state(local, seg(s), d2, 1);
#pragma unroll
                for (int i = 0; i < DT * NT; ++i) S[i] = S[i] * w.hi + (S[i] * w.lo + local[i]);
            }
        }
    }

    const int qrow = tid * VE / D1P, qcol = tid * VE % D1P, vrow = tid * VE / NB, vcol = tid * VE % NB;
    constexpr int es = sizeof(Ti);
    unsigned qoff = 0, koff = 0, voff = 0;
    if constexpr (VEC) {
        qoff = qcol < d1 ? (qrow * static_cast<int>(qt) + qcol) * es : kOutside;
        koff = qcol < d1 ? (qrow * static_cast<int>(kt) + qcol) * es : kOutside;
        voff = n0 + vcol < d2 ? (vrow * static_cast<int>(vt) + vcol) * es : kOutside;
    }

    // the `size` tokens from u on in the order of traversal: the lowest of them
    auto lowest = [&](long long u, int size) { return late ? len - u - size : u; };
    Pack<Ti, VE> rq[STATE_ONLY ? 1 : QV], rk[QV], rv[VV];
    // their rows into registers, zeros behind the last one
    auto fetch = [&](long long u, int size) {
        const long long low = lowest(u, size);
        if constexpr (VEC) {
            const auto dq = descriptor(q + low * qt), dk = descriptor(k + low * kt), dv = descriptor(v + low * vt);
#pragma unroll
            for (int x = 0; x < QV; ++x) {
                const bool in = qrow < size - x * QROWS;
                rk[x] = load_pack<Ti, VE>(dk, in ? koff : kOutside, x * QROWS * es * static_cast<int>(kt));
                if constexpr (!STATE_ONLY) rq[x] = load_pack<Ti, VE>(dq, in ? qoff : kOutside, x * QROWS * es * static_cast<int>(qt));
            }
#pragma unroll
            for (int x = 0; x < VV; ++x)
                rv[x] = load_pack<Ti, VE>(dv, vrow < size - x * VROWS ? voff : kOutside, x * VROWS * es * static_cast<int>(vt));
        } else {
#pragma unroll
            for (int x = 0; x < QV; ++x) {
                const int row = qrow + x * QROWS;
                rk[x] = load_elements<Ti, VE>(k + (low + row) * kt + qcol, row < size ? d1 - qcol : 0);
                if constexpr (!STATE_ONLY) rq[x] = load_elements<Ti, VE>(q + (low + row) * qt + qcol, row < size ? d1 - qcol : 0);
            }
#pragma unroll
            for (int x = 0; x < VV; ++x) {
                const int row = vrow + x * VROWS;
                rv[x] = load_elements<Ti, VE>(v + (low + row) * vt + vcol, row < size ? d2 - n0 - vcol : 0);
            }
        }
    };
    auto commit = [&]() {
#pragma unroll
        for (int x = 0; x < QV; ++x) {
            to_lds(lds.k + (qrow + x * QROWS) * L::kD + qcol, rk[x]);
            if constexpr (!STATE_ONLY) to_lds(lds.q + (qrow + x * QROWS) * L::kQ + qcol, rq[x]);
        }
#pragma unroll
        for (int x = 0; x < VV; ++x) to_lds(lds.v + (vrow + x * VROWS) * L::kN + vcol, rv[x]);
    };
    auto size_at = [&](long long u) { return static_cast<int>(min(static_cast<long long>(C), u1 - u)); };

    // of a whole chunk and of the last one
    const Decay whole = decay_over(log2w, C), rest = u0 < u1 ? decay_over(log2w, (u1 - u0 - 1) % C + 1) : whole;

    if (u0 < u1) {
        fetch(u0, size_at(u0));
        commit();
    }
    __syncthreads();
    settle(S);  // loaded here: in the loop the wait for it would be one for the rows on their way, too

    for (long long u = u0; u < u1; u += C) {
        const int size = size_at(u);
        const bool more = u + C < u1;
        if (more) fetch(u + C, size_at(u + C));

        const float *const pw_mirrored = lds.pw + C - (size - 1), *const pw_plain = lds.pw + C + 1;
        const float *const pw_read = late ? pw_mirrored : pw_plain, *const pw_write = late ? pw_plain : pw_mirrored;
        f32x4 O[STATE_ONLY ? 2 : IT * NT];
        if constexpr (!STATE_ONLY) {
            // O^T = S^T Q^T, and P^T = K Q^T, of which wave w takes the keys of tile w % IT for every (4 / IT)-th tile of
            // queries -- all of them: leaving out the tiles that the mask empties costs more in branches than it saves.
            // The contraction is the outer loop: S becomes an operand 32 rows at a time.
            constexpr int PT = IT * IT / 4;
            const int jt = wave % IT;
            f32x4 p[PT];
#pragma unroll
            for (int x = 0; x < PT; ++x) p[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < IT * NT; ++x) O[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if (kTrim && 32 * kb >= d1) break;
                F sf[NT];
                const F kf = row_frag(lds.k + (16 * jt + m) * L::kD + 32 * kb, g);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sf[nt] = operand(S[2 * kb * NT + nt], S[(2 * kb + 1) * NT + nt], Tc());
#pragma unroll
                for (int it = 0; it < IT; ++it) {
                    const F qf = row_frag(lds.q + (16 * it + m) * L::kQ + 32 * kb, g);
                    if (!kTrim || busy) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma(O[it * NT + nt], sf[nt], qf);
                    }
                    if constexpr (PT == IT) mma(p[it], kf, qf);
                }
                if constexpr (PT == 1) mma(p[0], kf, row_frag(lds.q + (16 * (wave / IT) + m) * L::kQ + 32 * kb, g));
            }
            settle(p);
#pragma unroll
            for (int x = 0; x < PT; ++x) {
                const int it = PT == 1 ? wave / IT : x;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = lds.pm[C + 16 * (it - jt) + m - 4 * g - r];
                    p[x][r] = w >= 0.0f ? p[x][r] * (w * pscale) : 0.0f;  // what is left out may be anything, NaN too
                }
                to_lds4(lds.p + (16 * it + m) * L::kP + 16 * jt + 4 * g, p[x]);
            }
            settle(O);
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                const float rd = read * pw_read[16 * it + m];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) O[it * NT + nt] *= rd;
            }
            __syncthreads();
        }

        F vf[JB][NT];
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) vf[jb][nt] = col_frag<L::kN>(lds.v + 32 * jb * L::kN + 16 * (NT * wave + nt), g, m);

        if constexpr (!STATE_ONLY) {
            char *const op = o + lowest(u, size) * ot * osize;
            const auto dout = descriptor(op);
            // 0 * NaN is NaN: a product with P would carry what is not finite in V to tokens that P leaves it out for.
            f32x4 none = {};
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) times_zero(none, vf[jb][nt]);
            settle(none);
            const bool finite = none[0] == 0.0f && none[1] == 0.0f && none[2] == 0.0f && none[3] == 0.0f;
            if (__builtin_expect(__all(finite), 1)) {
#pragma unroll
                for (int it = 0; it < IT; ++it) {
#pragma unroll
                    for (int jb = 0; jb < JB; ++jb) {
                        if (late ? jb < it / 2 : jb > it / 2) continue;
                        const F pf = row_frag(lds.p + (16 * it + m) * L::kP + 32 * jb, g);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma(O[it * NT + nt], vf[jb][nt], pf);
                    }
                }
                settle(O);
            } else {  // token by token, by those that see it
#pragma unroll 1
                for (int j = 0; j < C; ++j) {
                    const Tc *const vj = lds.v + j * L::kN + 16 * NT * wave + 4 * g;
#pragma unroll
                    for (int it = 0; it < IT; ++it) {
                        const int i = 16 * it + m;
                        if (late ? j < i : j > i) continue;
                        const float pij = static_cast<float>(lds.p[i * L::kP + j]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) O[it * NT + nt][r] += pij * static_cast<float>(vj[16 * nt + r]);
                    }
                }
            }
#pragma unroll
            for (int it = 0; it < IT; ++it) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int n = 16 * (NT * wave + nt) + 4 * g;
                    if constexpr (VEC) {
                        const unsigned at = m < size - 16 * it && n0 + n < d2 ? (m * static_cast<int>(ot) + n) * osize : kOutside;
                        const int step = 16 * it * static_cast<int>(ot) * osize;
                        if (partial) store_quad<float>(dout, at, step, O[it * NT + nt]);
                        else store_quad<Ti>(dout, at, step, O[it * NT + nt]);
                    } else if (16 * it + m < size) {
                        char *const to = op + ((16 * it + m) * ot + n) * osize;
                        if (partial) store_elements(reinterpret_cast<float *>(to), O[it * NT + nt], d2 - n0 - n);
                        else store_elements(reinterpret_cast<Ti *>(to), O[it * NT + nt], d2 - n0 - n);
                    }
                }
            }
        }

        // S <- w^size S + K^T (weighted V), the weighted V in three bf16 parts (fp32: in one); rows behind the last are zeros.
        // Every weight is one at most and S is as large as it is: to put the decay off, and to weight V the more for it, would
        // save 2 to 5 % of the time but lose the largest numbers.
        const float hi = more ? whole.hi : rest.hi, lo = more ? whole.lo : rest.lo;
#pragma unroll
        for (int i = 0; i < DT * NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // x hi + x lo in x's own register: the compiler would take another 64
                float x = S[i][r], t;
                asm("v_mul_f32 %1, %2, %0\n\tv_fma_f32 %0, %0, %3, %1" : "+v"(x), "=&v"(t) : "v"(lo), "v"(hi));
                S[i][r] = x;
            }
        ready(S);
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
            float wj[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) wj[e] = write * pw_write[32 * jb + 16 * (e >> 2) + 4 * g + (e & 3)];
            constexpr int PARTS = sizeof(Tc) == 2 ? 3 : 1, GROUP = 4;
            F part[PARTS][NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                split(part, nt, vf[jb][nt], wj);
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += GROUP) {
                if (kTrim && (16 * d0 >= d1 || !busy)) break;  // four tiles of rows at a time: products that do not wait for each other
                F kc[GROUP];
#pragma unroll
                for (int i = 0; i < GROUP; ++i) kc[i] = col_frag<L::kD>(lds.k + 32 * jb * L::kD + 16 * (d0 + i), g, m);
#pragma unroll
                for (int s = PARTS - 1; s >= 0; --s)
#pragma unroll
                    for (int i = 0; i < GROUP; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma(S[(d0 + i) * NT + nt], kc[i], part[s][nt]);
            }
        }
        settle(S);
        __syncthreads();
        if (more) {
            commit();
            __syncthreads();
        }
    }

    float *s_out = nullptr;
    if constexpr (STATE_ONLY) s_out = seg(segment);
    else if (role.s_out && u1 == len) s_out = a.in_place && segment > 0 ? seg(segment - 1) : role.s_out + bh * d1 * d2;
    if (s_out) {
        int rows = d1, cols = d2;  // hidden from the compiler, which would keep 64 comparisons of the loads above for the stores
        asm volatile("" : "+s"(rows), "+s"(cols));
        const auto to = descriptor(s_out);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = n0 + 16 * (NT * wave + nt) + m;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r;
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(S[dt * NT + nt][r]), to,
                                                          d < rows && n < cols ? (d * cols + n) * 4u : kOutside, 0, 0);
                }
            }
    }
}

template <typename Ti, typename Tc, int D1P, int NT, int C, bool STATE_ONLY, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) linear_attention_kernel(const Args a) {
    // workgroup -> (segment of a sequence, head, role, tile): the tiles and roles of a head next to each other
    unsigned id = static_cast<unsigned>(block_index());
    if (id >= a.blocks) return;
    unsigned role_tiles = 0;
    for (int r = 0; r < a.roles; ++r) role_tiles += a.role[r].tiles;
    int t = id % role_tiles;
    id /= role_tiles;
    const int head = id % a.heads;
    id /= a.heads;
    int ri = 0;
    while (t >= a.role[ri].tiles) t -= a.role[ri++].tiles;
    const Role &role = a.role[ri];
    const int n0 = t * 64 * NT;
    int b, segment;
    long long start, len;
    Slots slots;
    if (a.offsets && a.segments > 1) {  // the slots' segments first, then the last segment of every sequence
        if (id < a.slots) {
            // seg_len rows from one in [id, id + 1) * seg_len on hold the last row of that range, whatever the offsets are
            b = sequence_at(a, (id + 1) * a.seg_len - 1);
            sequence_rows(a, b, start, len);
            slots = slots_of(a, role.late, b, start, len);
            segment = (static_cast<int>(id) - slots.first) * slots.step;
            if (segment < 0 || segment >= inner_segments(a, len)) return;  // no segment has this slot
        } else {
            b = id - a.slots;
            sequence_rows(a, b, start, len);
            slots = slots_of(a, role.late, b, start, len);
            segment = inner_segments(a, len);
        }
    } else {
        b = id % a.batch;
        segment = id / a.batch;
        sequence_rows(a, b, start, len);
        slots = slots_of(a, role.late, b, start, len);
    }
    if (role.late) linear_attention_body<Ti, Tc, D1P, NT, C, STATE_ONLY, VEC, true>(a, role, n0, head, b, start, len, segment, slots);
    else linear_attention_body<Ti, Tc, D1P, NT, C, STATE_ONLY, VEC, false>(a, role, n0, head, b, start, len, segment, slots);
}

// D1P and NT by the host's rule; C by the type: 64 tokens, 32 where an element is four bytes or a row 256 of them (LDS)
template <typename Ti, typename Tc, int D1P, int NT, bool STATE_ONLY, bool VEC>
int launch_kernel_as(const Args &a, hipStream_t s) {
    constexpr int C = sizeof(Tc) == 2 && D1P <= 128 ? 64 : 32;
    using L = typename std::conditional<STATE_ONLY, LdsState<Tc, D1P, NT, C>, Lds<Tc, D1P, NT, C>>::type;
    const auto fn = linear_attention_kernel<Ti, Tc, D1P, NT, C, STATE_ONLY, VEC>;
    if (sizeof(L) > 65536)
        if (int rc = allow_full_lds(reinterpret_cast<const void *>(fn))) return rc;
    fn<<<grid_of(a.blocks), kThreads, sizeof(L), s>>>(a);
    return check_launch("linear_attention_kernel");
}

struct Variant {
    int d1p, nt;
    bool vec, state_only;
};

template <typename Ti, typename Tc, int D1P, int NT>
int launch_one(const Args &a, const Variant &v, hipStream_t s) {
    if (v.state_only) return v.vec ? launch_kernel_as<Ti, Tc, D1P, NT, true, true>(a, s) : launch_kernel_as<Ti, Tc, D1P, NT, true, false>(a, s);
    return v.vec ? launch_kernel_as<Ti, Tc, D1P, NT, false, true>(a, s) : launch_kernel_as<Ti, Tc, D1P, NT, false, false>(a, s);
}

template <typename Ti, typename Tc>
int launch_any(const Args &a, const Variant &v, hipStream_t s) {
    if (v.d1p == 64) return v.nt == 1 ? launch_one<Ti, Tc, 64, 1>(a, v, s) : launch_one<Ti, Tc, 64, 2>(a, v, s);
    if (v.d1p == 128) return v.nt == 1 ? launch_one<Ti, Tc, 128, 1>(a, v, s) : launch_one<Ti, Tc, 128, 2>(a, v, s);
    return launch_one<Ti, Tc, 256, 1>(a, v, s);
}

// one translation unit each
int launch_bf16(const Args &a, const Variant &v, hipStream_t s);
int launch_f16(const Args &a, const Variant &v, hipStream_t s);
int launch_f32(const Args &a, const Variant &v, hipStream_t s);

}  // namespace la
}  // namespace dspgpu
