// linear_attention.hip -- linear attention with a decay for each head: entry points, the plan of a call, and the small
// kernels around linear_attention_core.h (joining segments, adding up shared heads' gradients, the single-token step).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "linear_attention_core.h"

namespace dspgpu {
namespace la {
namespace {

// ---- segments -> states ------------------------------------------------------------------------------------------------

// The slot of segment s holds what it leaves behind from a zero state; afterwards, the state that segment s + 1 starts from.
// A thread has kJoin elements of the state, 256 apart; the loads do not depend on the recurrence.
constexpr int kJoin = 4;
__global__ void __launch_bounds__(256) join_segments_kernel(const Args a) {
    const Role &role = a.role[blockIdx.z];
    const int count = role.d1 * role.d2, blocks = (count + 256 * kJoin - 1) / (256 * kJoin);
    const unsigned id = static_cast<unsigned>(block_index());
    if (id / blocks >= static_cast<unsigned>(a.batch * a.heads)) return;
    const int bh = id / blocks, e0 = (id % blocks) * 256 * kJoin + threadIdx.x;
    long long start, len;
    sequence_rows(a, bh / a.heads, start, len);
    const int full = inner_segments(a, len);
    if (full == 0) return;
    const Slots slots = slots_of(a, role.late, bh / a.heads, start, len);
    float run[kJoin];
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
        const int e = e0 + 256 * j;
        run[j] = role.s_in && e < count ? role.s_in[static_cast<size_t>(bh) * count + (e / role.d2) * role.s_in_d + (e % role.d2) * role.s_in_n] : 0.0f;
    }
    float *seg = role.seg + (static_cast<size_t>(bh % a.heads) * a.slots + slots.first) * count + e0;
    const int step = slots.step * count;
    const Decay w = decay_over(a.log2_decay[bh % a.heads], a.seg_len);
    for (int s0 = 0; s0 < full; s0 += 4, seg += 4 * step) {
        float local[4][kJoin];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kJoin; ++j) local[i][j] = s0 + i < full && e0 + 256 * j < count ? seg[i * step + 256 * j] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i >= full) break;
#pragma unroll
            for (int j = 0; j < kJoin; ++j) {
                run[j] = fmaf(run[j], w.hi, fmaf(run[j], w.lo, local[i][j]));
                if (e0 + 256 * j < count) seg[i * step + 256 * j] = run[j];
            }
        }
    }
}

// A state in place: where a sequence has several segments, others may still read the state before its first token when the
// last one is done.  That one leaves its state in the slot of the segment before it, which nobody else reads any more (of the
// columns that are its own), and this brings it to its place.
__global__ void __launch_bounds__(256) copy_states_kernel(const Args a) {
    const Role &role = a.role[0];
    const int count = role.d1 * role.d2, blocks = (count + 256 * kJoin - 1) / (256 * kJoin);
    const unsigned id = static_cast<unsigned>(block_index());
    if (id / blocks >= static_cast<unsigned>(a.batch * a.heads)) return;
    const int bh = id / blocks, e0 = (id % blocks) * 256 * kJoin + threadIdx.x;
    long long start, len;
    sequence_rows(a, bh / a.heads, start, len);
    const int full = inner_segments(a, len);
    if (full == 0) return;
    const Slots slots = slots_of(a, role.late, bh / a.heads, start, len);
    const float *from = role.seg + (static_cast<size_t>(bh % a.heads) * a.slots + slots.first + (full - 1) * slots.step) * count;
    float *to = role.s_out + static_cast<size_t>(bh) * count;
#pragma unroll
    for (int j = 0; j < kJoin; ++j)
        if (e0 + 256 * j < count) to[e0 + 256 * j] = from[e0 + 256 * j];
}

// ---- gradients of shared heads -----------------------------------------------------------------------------------------

// Whether a sequence holds `row` (of [batch][n], or of the packed batch) -- what the kernel above wrote.
__device__ __forceinline__ bool row_taken(const Args &a, long long row) {
    if (a.batch == 0) return false;
    long long start, len;
    if (a.offsets) {
        sequence_rows(a, sequence_at(a, row), start, len);
        return row >= start && row < start + len;
    }
    sequence_rows(a, static_cast<int>(row / a.n), start, len);
    return row % a.n < len;
}

struct Shared {
    const float *part[3];
    void *out[3];
    int group[3], dim[3];
    long long rows;
};

// part [row][heads][dim] fp32 -> out [row][heads / group][dim], heads of a group added in their order
template <typename T>
__global__ void __launch_bounds__(256) add_heads_kernel(const Args a, const Shared g) {
    const long long row = static_cast<long long>(block_index());
    if (row >= g.rows || !row_taken(a, row)) return;
    const int i = blockIdx.z, group = g.group[i], dim = g.dim[i], heads = a.heads / group;
    for (int e = threadIdx.x; e < heads * dim; e += 256) {
        const float *p = g.part[i] + (row * a.heads + (e / dim) * group) * dim + e % dim;
        float sum = 0.0f;
        for (int h = 0; h < group; ++h) sum += p[static_cast<size_t>(h) * dim];
        static_cast<T *>(g.out[i])[row * heads * dim + e] = static_cast<T>(sum);
    }
}

// ---- rows of no sequence -----------------------------------------------------------------------------------------------

struct Rest {
    void *p[3];
    long long stride[3][3];
    int heads[3], dim[3];
    int wide;  // 4-byte samples
    long long rows;
};

// zeros into the rows that no sequence holds (all samples are zero where their bits are): a thread looks at a row, and the
// workgroup clears what its threads found
__global__ void __launch_bounds__(256) zero_rest_kernel(const Args a, const Rest z) {
    __shared__ int list[256], count;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const long long first = static_cast<long long>(block_index()) * 256, mine = first + threadIdx.x;
    if (mine < z.rows && !row_taken(a, mine)) list[atomicAdd(&count, 1)] = threadIdx.x;
    __syncthreads();
    const int i = blockIdx.z;
    for (int r = 0; r < count; ++r) {
        const long long row = first + list[r];
        const long long at = a.offsets ? row * z.stride[i][1] : row / a.n * z.stride[i][0] + row % a.n * z.stride[i][1];
        for (int e = threadIdx.x; e < z.heads[i] * z.dim[i]; e += 256) {
            const long long to = at + e / z.dim[i] * z.stride[i][2] + e % z.dim[i];
            if (z.wide) static_cast<unsigned *>(z.p[i])[to] = 0;
            else static_cast<unsigned short *>(z.p[i])[to] = 0;
        }
    }
}

int zero_rest(const Args &a, Rest &z, int count, hipStream_t s) {
    zero_rest_kernel<<<grid_of(static_cast<size_t>((z.rows + 255) / 256), count), 256, 0, s>>>(a, z);
    return check_launch("zero_rest_kernel");
}

// ---- one token ---------------------------------------------------------------------------------------------------------

struct StepArgs {
    const void *q, *k, *v;
    void *o;
    long long qs[2], ks[2], vs[2], os[2];  // strides: row, head
    int q_group, k_group, v_group;
    int heads, d1, d2, batch;
    float scale;
    int vec;                               // states in 16-byte accesses
    float *state;                          // [slots][heads][d1][d2]
    const long long *slots;                // or null: row b has state b
    long long n_slots;
    float decay_hi[kMaxHeads], decay_lo[kMaxHeads];  // the decay in two parts: rounded to 24 bits it would drift over long answers
};

constexpr int kStepCols = 64;

// S <- w S + k v^T, o = scale q S.  Bound by the state's traffic (8 d1 d2 bytes a head): a workgroup takes 64 columns of one
// head, each thread four columns of every 16th row, all its rows in flight at once, and the operands beside them.  64 rows
// of 16 heads of 128 x 128: 28 us for 134 MB, 4.8 TB/s; one row of 8 heads of 64 x 64: 5 us, a launch and three latencies.
// A slot that several rows name is taken by the workgroup of the first of them, for all of them in their order.
template <typename T, int ROWS>
__global__ void __launch_bounds__(256) step_kernel(const StepArgs a) {
    __shared__ float part[4][kStepCols];
    __shared__ int first, more;
    const int tiles = (a.d2 + kStepCols - 1) / kStepCols;
    const unsigned id = static_cast<unsigned>(block_index());
    const int tile = id % tiles, head = id / tiles % a.heads;
    int b = id / tiles / a.heads;
    if (b >= a.batch) return;
    const int tid = threadIdx.x, cx = tid & 15, ry = tid >> 4, lane = tid & 63, wave = tid >> 6;
    const int n0 = tile * kStepCols + 4 * cx;

    long long slot = b;
    if (a.slots) {
        slot = a.slots[b];
        if (slot < 0 || slot >= a.n_slots) {  // an empty row
            if (tid < kStepCols && tile * kStepCols + tid < a.d2)
                static_cast<T *>(a.o)[b * a.os[0] + head * a.os[1] + tile * kStepCols + tid] = static_cast<T>(0.0f);
            return;
        }
    }
    const float w = a.decay_hi[head], w_lo = a.decay_lo[head];
    float *state = a.state + ((slot * a.heads + head) * a.d1) * a.d2 + n0;
    f32x4 s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int d = ry + 16 * i;
        s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (d < a.d1) {
            if (a.vec) {
                if (n0 < a.d2) s[i] = *reinterpret_cast<const f32x4 *>(state + static_cast<size_t>(d) * a.d2);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n0 + c < a.d2) s[i][c] = state[static_cast<size_t>(d) * a.d2 + c];
            }
        }
    }
    float kd[ROWS], qd[ROWS];
    f32x4 vv;
    auto operands = [&]() {
        const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + (head / a.q_group) * a.qs[1];
        const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + (head / a.k_group) * a.ks[1];
        const T *v = static_cast<const T *>(a.v) + b * a.vs[0] + (head / a.v_group) * a.vs[1] + n0;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int d = ry + 16 * i;
            kd[i] = d < a.d1 ? static_cast<float>(k[d]) : 0.0f;
            qd[i] = d < a.d1 ? static_cast<float>(q[d]) : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) vv[c] = n0 + c < a.d2 ? static_cast<float>(v[c]) : 0.0f;
    };
    operands();  // on their way while the slots are looked through
    bool again = false;
    if (a.slots) {
        if (tid == 0) {
            first = b;
            more = 0;
        }
        __syncthreads();
        for (int r = tid; r < a.batch; r += 256)
            if (r != b && a.slots[r] == slot) {
                if (r < b) first = r;  // any earlier row: this workgroup is not the slot's
                else more = 1;
            }
        __syncthreads();
        if (first != b) return;
        again = more != 0;
    }
    for (;;) {
        f32x4 acc = {};
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            s[i] = s[i] * w + (s[i] * w_lo + kd[i] * vv);
            acc += qd[i] * s[i];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            acc[c] += __shfl_xor(acc[c], 16);
            acc[c] += __shfl_xor(acc[c], 32);
        }
        if (lane < 16) *reinterpret_cast<f32x4 *>(&part[wave][4 * cx]) = acc;
        __syncthreads();
        if (tid < kStepCols && tile * kStepCols + tid < a.d2) {
            T *o = static_cast<T *>(a.o) + b * a.os[0] + head * a.os[1] + tile * kStepCols + tid;
            *o = static_cast<T>(a.scale * ((part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid])));
        }
        if (!again) break;
        __syncthreads();
        for (++b; b < a.batch; ++b)
            if (a.slots[b] == slot) break;
        if (b >= a.batch) break;
        operands();
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int d = ry + 16 * i;
        if (d < a.d1) {
            if (a.vec) {
                if (n0 < a.d2) *reinterpret_cast<f32x4 *>(state + static_cast<size_t>(d) * a.d2) = s[i];
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n0 + c < a.d2) state[static_cast<size_t>(d) * a.d2 + c] = s[i][c];
            }
        }
    }
}

template <typename T>
int launch_step(const StepArgs &a, hipStream_t s) {
    const dim3 grid = grid_of(static_cast<size_t>(a.batch) * a.heads * ((a.d2 + kStepCols - 1) / kStepCols));
    if (a.d1 <= 64) step_kernel<T, 4><<<grid, 256, 0, s>>>(a);
    else if (a.d1 <= 128) step_kernel<T, 8><<<grid, 256, 0, s>>>(a);
    else step_kernel<T, 16><<<grid, 256, 0, s>>>(a);
    return check_launch("step_kernel");
}

// ---- host --------------------------------------------------------------------------------------------------------------

typedef dsp_gpu_linear_attention_shape Shape;

size_t sample_bytes(int type) { return type == DSP_GPU_F32 ? 4 : 2; }

struct Range {
    const char *p;
    size_t bytes;
};
bool meet(const Range &a, const Range &b) { return a.p && b.p && a.bytes && b.bytes && a.p < b.p + b.bytes && b.p < a.p + a.bytes; }

// bytes from the first to the last element of a strided [batch][n][heads][dim] array
size_t extent(const long long *stride, size_t batch, size_t n, size_t heads, size_t dim, size_t size) {
    if (batch == 0 || n == 0) return 0;
    return ((batch - 1) * stride[0] + (n - 1) * stride[1] + (heads - 1) * stride[2] + dim) * size;
}

int check_heads(const char *who, int heads, int heads_q, int heads_k, int heads_v, int dim_k, int dim_v, int type) {
    if (type != DSP_GPU_F32 && type != DSP_GPU_F16 && type != DSP_GPU_BF16) return fail(DSP_GPU_EINVAL, "%s: sample type %d (F32, F16 or BF16)", who, type);
    if (heads < 1 || heads > kMaxHeads) return fail(DSP_GPU_EINVAL, "%s: %d heads outside [1,%d]", who, heads, kMaxHeads);
    for (int h : {heads_q, heads_k, heads_v})
        if (h < 1 || heads % h) return fail(DSP_GPU_EINVAL, "%s: %d heads of q, k or v do not divide %d", who, h, heads);
    if (dim_k < 1 || dim_k > 256 || dim_v < 1 || dim_v > 256)
        return fail(DSP_GPU_EINVAL, "%s: dimensions %d, %d outside [1,256]", who, dim_k, dim_v);
    return DSP_GPU_OK;
}

int check_decay(const char *who, const double *log_decay, int heads, double scale, float *log2_decay) {
    for (int h = 0; h < heads; ++h) {
        if (!(log_decay[h] <= 0.0)) return fail(DSP_GPU_EINVAL, "%s: log_decay[%d] = %g is not <= 0", who, h, log_decay[h]);
        log2_decay[h] = static_cast<float>(log_decay[h] * 1.4426950408889634);
    }
    if (!std::isfinite(scale)) return fail(DSP_GPU_EINVAL, "%s: non-finite scale", who);
    return DSP_GPU_OK;
}

int check_shape(const char *who, const Shape &p) {
    if (int rc = check_heads(who, p.heads, p.heads_q, p.heads_k, p.heads_v, p.dim_k, p.dim_v, p.sample_type)) return rc;
    if (p.offsets && p.lengths) return fail(DSP_GPU_EINVAL, "%s: offsets and lengths exclude each other", who);
    if (p.batch > (1u << 24) || p.n > (1ull << 31) || p.rows > (1ull << 31)) return fail(DSP_GPU_EINVAL, "%s: too many sequences or tokens", who);
    for (const long long *s : {p.q_stride, p.k_stride, p.v_stride, p.o_stride})
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0 || s[i] > (1ll << 40)) return fail(DSP_GPU_EINVAL, "%s: stride %lld", who, s[i]);
    const size_t batch = p.offsets ? 1 : p.batch, n = p.offsets ? p.rows : p.n;
    if (!extent_fits(p.q_stride, batch, n, p.heads_q, p.dim_k) || !extent_fits(p.k_stride, batch, n, p.heads_k, p.dim_k) ||
        !extent_fits(p.v_stride, batch, n, p.heads_v, p.dim_v) || !extent_fits(p.o_stride, batch, n, p.heads, p.dim_v))
        return fail(DSP_GPU_EINVAL, "%s: a tensor is larger than any memory", who);
    return DSP_GPU_OK;
}

// Ranges that a call reads or writes: what it writes must not meet any other.  Empty and null ranges meet nothing.
struct Buffers {
    Range r[12];
    int count = 0;
    void add(const void *p, size_t bytes) { r[count++] = {static_cast<const char *>(p), bytes}; }
    bool meet(const void *p, size_t bytes) const {
        for (int i = 0; i < count; ++i)
            if (la::meet({static_cast<const char *>(p), bytes}, r[i])) return true;
        return false;
    }
};

// the inputs that forward and backward share
Buffers inputs(const Shape &p, const void *q, const void *k, const void *v) {
    const size_t batch = p.offsets ? 1 : p.batch, n = p.offsets ? p.rows : p.n, size = sample_bytes(p.sample_type);
    Buffers b;
    b.add(q, extent(p.q_stride, batch, n, p.heads_q, p.dim_k, size));
    b.add(k, extent(p.k_stride, batch, n, p.heads_k, p.dim_k, size));
    b.add(v, extent(p.v_stride, batch, n, p.heads_v, p.dim_v, size));
    b.add(p.offsets, sizeof(long long) * (p.batch + 1));
    b.add(p.lengths, sizeof(long long) * p.batch);
    return b;
}

// One launch of the kernel: up to three roles that share the padded first dimension and the columns of a workgroup.
struct Plan {
    int d1p, nt, segments;
    long long seg_len;
    size_t slots;  // segments that leave a state to the next one, of all sequences together
};

constexpr long long kSlots = 512;     // workgroups the chip runs at once: two on each of 256 CUs
// Tokens of a segment at least: a state is written and read for each.  (2 x 1000 tokens of 12 heads of 48 x 80, backward:
// 55 us; 256: 65 us, 64: 56 us.  2 x 2048 of 8 heads, fp32: 47 us; 256: 66 us, 64: 48 us.  1 x 600 of 4 heads: 34 us; 256:
// 48 us, 64: 30 us.)
constexpr long long kLeast = 128;

// How the work of `roles` runs over batch * heads sequences is spread.  A workgroup that owns 128 columns reads q and k half
// as often as two that own 64.  Where the runs do not fill the chip the time axis is cut into segments, which costs a
// second pass over k and v (about kAgain of the first): dense batches take the number of segments with the least
// ceil(workgroups / slots) * tokens of a segment; of packed ones only the sum of the lengths is known, and a segment is
// its share of a slot (20,011 tokens of 16 heads in 16 sequences: 175 us; half of it 191 us, a third 197 us).
Plan make_plan(const Shape &p, int d1, const int *d2, int roles) {
    Plan pl{};
    pl.d1p = d1 <= 64 ? 64 : d1 <= 128 ? 128 : 256;
    bool wide = false;
    for (int r = 0; r < roles; ++r) wide = wide || d2[r] > 64;
    pl.nt = pl.d1p < 256 && wide ? 2 : 1;
    long long groups = 0;
    for (int r = 0; r < roles; ++r) groups += (d2[r] + 64 * pl.nt - 1) / (64 * pl.nt);
    groups *= p.heads;
    const long long batch = static_cast<long long>(p.batch), n = static_cast<long long>(p.offsets ? std::min(p.n, p.rows) : p.n);
    auto up = [](long long x) { return (x + 63) / 64 * 64; };  // whole chunks
    pl.seg_len = std::max<long long>(64, up(n));
    if (n >= 2 * kLeast) {
        constexpr double kAgain = 0.4;
        if (p.offsets) {
            pl.seg_len = std::min(pl.seg_len, std::max(kLeast, up(static_cast<long long>(p.rows) * groups / kSlots)));
        } else {
            double best = 0.0;
            for (long long s = 1; s <= 64 && s <= n / kLeast; ++s) {
                const long long len = up((n + s - 1) / s), rounds = (batch * groups * ((n + len - 1) / len) + kSlots - 1) / kSlots;
                const double cost = static_cast<double>(rounds * (len + 64)) * (s > 1 ? 1.0 + kAgain : 1.0);
                if (s == 1 || cost < 0.9 * best) {
                    best = cost;
                    pl.seg_len = std::max<long long>(64, len);
                }
            }
        }
    }
    pl.segments = static_cast<int>(std::max<long long>(1, (n + pl.seg_len - 1) / pl.seg_len));
    if (pl.segments > 1) pl.slots = p.offsets ? p.rows / static_cast<size_t>(pl.seg_len) : p.batch * (pl.segments - 1);
    return pl;
}

size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

size_t segment_bytes(const Shape &p, const Plan &pl) {
    return align256(sizeof(float) * pl.slots * p.heads * p.dim_k * p.dim_v);
}
size_t total_rows(const Shape &p) { return p.offsets ? p.rows : p.batch * p.n; }
size_t part_bytes(const Shape &p, int heads_x, int dim) {
    return heads_x < p.heads ? align256(sizeof(float) * total_rows(p) * p.heads * dim) : 0;
}

int launch_kernel(Args &a, const Variant &v, int type, size_t blocks, hipStream_t s) {
    a.blocks = static_cast<unsigned>(blocks);
    if (type == DSP_GPU_BF16) return launch_bf16(a, v, s);
    if (type == DSP_GPU_F16) return launch_f16(a, v, s);
    return launch_f32(a, v, s);
}

// roles: a.role[0 .. a.roles) with everything but tiles and seg filled in; seg_ws: a.roles * segment_bytes
int run(const Shape &p, Args &a, const Plan &pl, char *seg_ws, hipStream_t s) {
    a.heads = p.heads;
    a.batch = static_cast<int>(p.batch);
    a.n = static_cast<long long>(p.n);
    a.rows = static_cast<long long>(p.rows);
    a.offsets = p.offsets;
    a.lengths = p.lengths;
    a.segments = pl.segments;
    a.seg_len = pl.seg_len;
    a.slots = static_cast<unsigned>(pl.slots);
    size_t tiles = 0, most = 0;
    Variant v{pl.d1p, pl.nt, true, false};
    for (int r = 0; r < a.roles; ++r) {
        Role &x = a.role[r];
        x.tiles = (x.d2 + 64 * pl.nt - 1) / (64 * pl.nt);
        x.seg = pl.segments > 1 ? reinterpret_cast<float *>(seg_ws + r * segment_bytes(p, pl)) : nullptr;
        tiles += x.tiles;
        most = std::max<size_t>(most, (static_cast<size_t>(x.d1) * x.d2 + 256 * kJoin - 1) / (256 * kJoin));
        v.vec = v.vec && x.vec;
    }
    const size_t runs = p.batch * p.heads, inner = pl.slots * p.heads * tiles, blocks = inner + runs * tiles;
    if (runs == 0) return DSP_GPU_OK;
    if (blocks > 0x7fffffffu || runs * most > 0x7fffffffu) return fail(DSP_GPU_EINVAL, "linear attention: %zu workgroups", blocks);
    if (pl.segments > 1) {
        v.state_only = true;
        if (int rc = launch_kernel(a, v, p.sample_type, inner, s)) return rc;
        if (pl.segments > kJoinSelf) {
            join_segments_kernel<<<grid_of(runs * most, a.roles), 256, 0, s>>>(a);
            if (int rc = check_launch("join_segments_kernel")) return rc;
        }
        v.state_only = false;
    }
    if (int rc = launch_kernel(a, v, p.sample_type, blocks, s)) return rc;
    if (!a.in_place) return DSP_GPU_OK;
    copy_states_kernel<<<grid_of(runs * most), 256, 0, s>>>(a);
    return check_launch("copy_states_kernel");
}

void set_strides(long long *to, const long long *from) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

// Rows of whole packs of `ve` elements, aligned, and a chunk's 64 rows within 2^29 bytes of one another
bool packs(const void *p, const long long *stride, int dim, long long ve, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % (ve * size) == 0 && dim % ve == 0 && stride[0] % ve == 0 && stride[1] % ve == 0 &&
           stride[2] % ve == 0 && stride[1] < (1ll << 21);
}

struct Tensor {
    const void *p;
    const long long *stride;
    int heads, dim;
};

void fill_role(Role &r, const Shape &p, const Tensor &q, const Tensor &k, const Tensor &v, void *o, const long long *o_stride, bool partial) {
    r.q = q.p, r.k = k.p, r.v = v.p, r.o = o;
    set_strides(r.qs, q.stride), set_strides(r.ks, k.stride), set_strides(r.vs, v.stride), set_strides(r.os, o_stride);
    r.q_group = p.heads / q.heads, r.k_group = p.heads / k.heads, r.v_group = p.heads / v.heads;
    r.d1 = q.dim, r.d2 = v.dim;
    r.o_partial = partial;
    const size_t size = sample_bytes(p.sample_type);
    const long long ve = p.sample_type == DSP_GPU_BF16 ? 8 : 4;
    r.vec = packs(q.p, q.stride, q.dim, ve, size) && packs(k.p, k.stride, k.dim, ve, size) && packs(v.p, v.stride, v.dim, ve, size) &&
            packs(o, o_stride, v.dim, 4, partial ? 4 : size);
}

struct BackwardPlan {
    Plan pl[3];     // of dq, dk, dv
    int launches;   // 1: the three in one launch (pl[0]); 2: dq and dk in one, dv in another
    size_t seg, part[3], total;
};

BackwardPlan backward_plan(const Shape &p) {
    BackwardPlan bp{};
    auto pad = [](int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; };
    const int d2[3] = {p.dim_k, p.dim_k, p.dim_v};
    // One launch of all three where their first dimensions are padded alike -- or where there is so little to do that a
    // launch more costs more than the wider padding (2 x 1000 tokens of 12 heads of 48 x 80: 55 us, in two launches 67 us;
    // 2 x 2048 of 16 of 64 x 128: 83 and 93 us; twice that: 126 and 124 us).
    const int wide = std::max(pad(p.dim_k), pad(p.dim_v));
    if (pad(p.dim_k) == pad(p.dim_v) || (wide <= 128 && total_rows(p) * p.heads <= 65536)) {
        bp.launches = 1;
        bp.pl[0] = make_plan(p, wide, d2, 3);
        bp.seg = 3 * segment_bytes(p, bp.pl[0]);
    } else {  // the launches follow one another: the segments of the second take the place of the first's
        bp.launches = 2;
        bp.pl[0] = make_plan(p, p.dim_v, d2, 2);
        bp.pl[2] = make_plan(p, p.dim_k, d2 + 2, 1);
        bp.seg = std::max(2 * segment_bytes(p, bp.pl[0]), segment_bytes(p, bp.pl[2]));
    }
    bp.part[0] = part_bytes(p, p.heads_q, p.dim_k);
    bp.part[1] = part_bytes(p, p.heads_k, p.dim_k);
    bp.part[2] = part_bytes(p, p.heads_v, p.dim_v);
    bp.total = bp.seg + bp.part[0] + bp.part[1] + bp.part[2];
    return bp;
}

int take_workspace(const char *who, size_t need, void *given, size_t given_bytes, const Buffers &used, hipStream_t s, char **out) {
    *out = nullptr;
    if (need == 0) return DSP_GPU_OK;
    if (given) {
        if (given_bytes < need) return fail(DSP_GPU_EINVAL, "%s: a workspace of %zu bytes, %zu are needed", who, given_bytes, need);
        if (reinterpret_cast<uintptr_t>(given) % 16) return fail(DSP_GPU_EINVAL, "%s: workspace not aligned to 16 bytes", who);
        if (used.meet(given, need)) return fail(DSP_GPU_EINVAL, "%s: the workspace overlaps a buffer", who);
        *out = static_cast<char *>(given);
        return DSP_GPU_OK;
    }
    void *p = nullptr;
    if (int rc = workspace(WS_ATTENTION, need, &p, s)) return rc;
    *out = static_cast<char *>(p);
    return DSP_GPU_OK;
}

template <typename T>
int add_heads(const Args &a, const Shape &p, const Shared &g, int count, hipStream_t s) {
    add_heads_kernel<T><<<grid_of(total_rows(p), count), 256, 0, s>>>(a, g);
    return check_launch("add_heads_kernel");
}

size_t state_bytes(const Shape &p) { return sizeof(float) * p.batch * p.heads * p.dim_k * p.dim_v; }

}  // namespace
}  // namespace la
}  // namespace dspgpu

using namespace dspgpu;
using namespace dspgpu::la;

extern "C" {

int dsp_gpu_linear_attention_workspace(const dsp_gpu_linear_attention_shape *shape, int backward, size_t *bytes) {
    static const char *who = "dsp_gpu_linear_attention_workspace";
    if (!shape || !bytes) return fail(DSP_GPU_EINVAL, "%s: null argument", who);
    if (int rc = check_shape(who, *shape)) return rc;
    *bytes = 0;
    if (shape->batch == 0 || total_rows(*shape) == 0) return DSP_GPU_OK;
    if (backward) {
        *bytes = backward_plan(*shape).total;
    } else {
        const Plan pl = make_plan(*shape, shape->dim_k, &shape->dim_v, 1);
        *bytes = segment_bytes(*shape, pl);
    }
    return DSP_GPU_OK;
}

int dsp_gpu_linear_attention(const void *q, const void *k, const void *v, void *o, const dsp_gpu_linear_attention_shape *shape,
                             const double *log_decay, double scale, const float *state_in, float *state_out, void *workspace,
                             size_t workspace_bytes, void *stream) {
    static const char *who = "dsp_gpu_linear_attention";
    if (!shape || !log_decay) return fail(DSP_GPU_EINVAL, "%s: null argument", who);
    const Shape &p = *shape;
    if (int rc = check_shape(who, p)) return rc;
    Args a{};
    if (int rc = check_decay(who, log_decay, p.heads, scale, a.log2_decay)) return rc;
    const size_t rows = total_rows(p);
    if (p.batch == 0 && !(p.zero_rest && rows)) return DSP_GPU_OK;
    if (rows && (!q || !k || !v || !o)) return fail(DSP_GPU_EINVAL, "%s: null buffer", who);
    const size_t size = sample_bytes(p.sample_type), sb = state_bytes(p);
    const size_t batch = p.offsets ? 1 : p.batch, n = p.offsets ? p.rows : p.n, ob = extent(p.o_stride, batch, n, p.heads, p.dim_v, size);
    if (rows && !rows_distinct(p.o_stride, batch, n, p.heads, p.dim_v)) return fail(DSP_GPU_EINVAL, "%s: rows of o overlap one another", who);
    Buffers used = inputs(p, q, k, v);
    if (state_in != state_out) used.add(state_in, sb);
    if (used.meet(o, ob)) return fail(DSP_GPU_EINVAL, "%s: o overlaps an input", who);
    used.add(o, ob);
    if (used.meet(state_out, sb)) return fail(DSP_GPU_EINVAL, "%s: state_out overlaps something else", who);
    used.add(state_out, sb);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Plan pl = make_plan(p, p.dim_k, &p.dim_v, 1);
    char *ws = nullptr;
    if (int rc = take_workspace(who, rows ? segment_bytes(p, pl) : 0, workspace, workspace_bytes, used, s, &ws)) return rc;
    a.roles = 1;
    Role &r = a.role[0];
    fill_role(r, p, {q, p.q_stride, p.heads_q, p.dim_k}, {k, p.k_stride, p.heads_k, p.dim_k}, {v, p.v_stride, p.heads_v, p.dim_v}, o, p.o_stride, false);
    r.read = r.pscale = static_cast<float>(scale);
    r.write = 1.0f;
    r.s_in = state_in;
    r.s_in_d = p.dim_v;
    r.s_in_n = 1;
    r.s_out = state_out;
    a.in_place = pl.segments > 1 && state_in && state_in == state_out;
    if (int rc = run(p, a, pl, ws, s)) return rc;
    if (!p.zero_rest || !(p.offsets || p.lengths) || !rows) return DSP_GPU_OK;
    Rest z{};
    z.p[0] = o;
    set_strides(z.stride[0], p.o_stride);
    z.heads[0] = p.heads;
    z.dim[0] = p.dim_v;
    z.wide = size == 4;
    z.rows = static_cast<long long>(rows);
    return zero_rest(a, z, 1, s);
}

int dsp_gpu_linear_attention_backward(const void *q, const void *k, const void *v, const void *dout, void *dq, void *dk, void *dv,
                                      const dsp_gpu_linear_attention_shape *shape, const double *log_decay, double scale,
                                      const float *state_in, const float *dstate_out, float *dstate_in, void *workspace,
                                      size_t workspace_bytes, void *stream) {
    static const char *who = "dsp_gpu_linear_attention_backward";
    if (!shape || !log_decay) return fail(DSP_GPU_EINVAL, "%s: null argument", who);
    const Shape &p = *shape;
    if (int rc = check_shape(who, p)) return rc;
    Args a{};
    if (int rc = check_decay(who, log_decay, p.heads, scale, a.log2_decay)) return rc;
    const size_t rows = total_rows(p), size = sample_bytes(p.sample_type), sb = state_bytes(p);
    if (p.batch == 0 && !(p.zero_rest && rows)) return DSP_GPU_OK;
    if (rows && (!q || !k || !v || !dout || !dq || !dk || !dv)) return fail(DSP_GPU_EINVAL, "%s: null buffer", who);
    if (rows > 0x7fffffffu) return fail(DSP_GPU_EINVAL, "%s: %zu rows", who, rows);
    const size_t batch = p.offsets ? 1 : p.batch, n = p.offsets ? p.rows : p.n;
    Buffers used = inputs(p, q, k, v);
    used.add(dout, extent(p.o_stride, batch, n, p.heads, p.dim_v, size));
    used.add(state_in, sb);
    used.add(dstate_out, sb);  // dk reads it while dv writes dstate_in: not in place
    const struct {
        const void *p;
        size_t bytes;
    } written[4] = {{dq, rows * p.heads_q * p.dim_k * size}, {dk, rows * p.heads_k * p.dim_k * size}, {dv, rows * p.heads_v * p.dim_v * size}, {dstate_in, sb}};
    for (const auto &x : written) {
        if (used.meet(x.p, x.bytes)) return fail(DSP_GPU_EINVAL, "%s: a gradient overlaps an input or another gradient", who);
        used.add(x.p, x.bytes);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const BackwardPlan bp = backward_plan(p);
    char *ws = nullptr;
    if (int rc = take_workspace(who, rows ? bp.total : 0, workspace, workspace_bytes, used, s, &ws)) return rc;

    const Tensor tq{q, p.q_stride, p.heads_q, p.dim_k}, tk{k, p.k_stride, p.heads_k, p.dim_k}, tv{v, p.v_stride, p.heads_v, p.dim_v},
        tdo{dout, p.o_stride, p.heads, p.dim_v};
    void *grad[3] = {dq, dk, dv};
    const int heads_x[3] = {p.heads_q, p.heads_k, p.heads_v}, dim[3] = {p.dim_k, p.dim_k, p.dim_v};
    float *part[3];
    Role role[3] = {};
    char *at = ws + bp.seg;
    for (int i = 0; i < 3; ++i) {
        part[i] = bp.part[i] ? reinterpret_cast<float *>(at) : nullptr;
        at += bp.part[i];
        const long long h = part[i] ? p.heads : heads_x[i];
        const long long st[3] = {static_cast<long long>(p.n) * h * dim[i], h * dim[i], dim[i]};
        const Tensor &x = i == 0 ? tdo : i == 1 ? tv : tk, &y = i == 0 ? tv : i == 1 ? tdo : tq, &z = i == 0 ? tk : i == 1 ? tq : tdo;
        fill_role(role[i], p, x, y, z, part[i] ? part[i] : grad[i], st, part[i] != nullptr);
        const float sc = static_cast<float>(scale);
        role[i].pscale = sc;
        role[i].read = i == 0 ? sc : 1.0f;
        role[i].write = i == 0 ? 1.0f : sc;
        role[i].late = i != 0;
        role[i].s_in = i == 0 ? state_in : dstate_out;
        role[i].s_in_d = i == 2 ? p.dim_v : 1;  // the states of dq and dk are S^T and dS^T
        role[i].s_in_n = i == 2 ? 1 : p.dim_v;
        role[i].s_out = i == 2 ? dstate_in : nullptr;
    }
    if (bp.launches == 1) {
        a.roles = 3;
        for (int i = 0; i < 3; ++i) a.role[i] = role[i];
        if (int rc = run(p, a, bp.pl[0], ws, s)) return rc;
    } else {
        a.roles = 2;
        a.role[0] = role[0];
        a.role[1] = role[1];
        if (int rc = run(p, a, bp.pl[0], ws, s)) return rc;
        a.roles = 1;
        a.role[0] = role[2];
        if (int rc = run(p, a, bp.pl[2], ws, s)) return rc;
    }
    Shared g{};
    g.rows = static_cast<long long>(rows);
    int count = 0;
    for (int i = 0; i < 3; ++i) {
        if (!part[i] || !rows) continue;
        g.part[count] = part[i];
        g.out[count] = grad[i];
        g.group[count] = p.heads / heads_x[i];
        g.dim[count++] = dim[i];
    }
    if (count) {
        const int rc = p.sample_type == DSP_GPU_BF16 ? add_heads<__bf16>(a, p, g, count, s)
                       : p.sample_type == DSP_GPU_F16 ? add_heads<_Float16>(a, p, g, count, s)
                                                      : add_heads<float>(a, p, g, count, s);
        if (rc) return rc;
    }
    if (!p.zero_rest || !(p.offsets || p.lengths) || !rows) return DSP_GPU_OK;
    Rest z{};
    for (int i = 0; i < 3; ++i) {
        z.p[i] = grad[i];
        z.heads[i] = heads_x[i];
        z.dim[i] = dim[i];
        z.stride[i][2] = dim[i];
        z.stride[i][1] = z.stride[i][2] * heads_x[i];
        z.stride[i][0] = z.stride[i][1] * static_cast<long long>(p.n);
    }
    z.wide = size == 4;
    z.rows = static_cast<long long>(rows);
    return zero_rest(a, z, 3, s);
}

int dsp_gpu_linear_attention_step(const void *q, const void *k, const void *v, void *o, const dsp_gpu_linear_attention_shape *shape,
                                  const double *log_decay, double scale, float *state, const long long *slots, size_t n_slots,
                                  void *stream) {
    static const char *who = "dsp_gpu_linear_attention_step";
    if (!shape || !log_decay) return fail(DSP_GPU_EINVAL, "%s: null argument", who);
    const Shape &p = *shape;
    if (int rc = check_shape(who, p)) return rc;
    StepArgs a{};
    if (int rc = check_decay(who, log_decay, p.heads, scale, a.decay_hi)) return rc;
    for (int h = 0; h < p.heads; ++h) {
        const Decay w = two_parts(std::exp(log_decay[h]));
        a.decay_hi[h] = w.hi;
        a.decay_lo[h] = w.lo;
    }
    if (p.n != 1 || p.offsets || p.lengths) return fail(DSP_GPU_EINVAL, "%s: one token a row (n = 1), no offsets or lengths", who);
    if (p.batch == 0) return DSP_GPU_OK;
    if (!q || !k || !v || !o || !state) return fail(DSP_GPU_EINVAL, "%s: null buffer", who);
    const size_t states = slots ? n_slots : p.batch, size = sample_bytes(p.sample_type);
    if (states == 0 || states > (1ull << 31)) return fail(DSP_GPU_EINVAL, "%s: %zu slots", who, states);
    if (!rows_distinct(p.o_stride, p.batch, 1, p.heads, p.dim_v)) return fail(DSP_GPU_EINVAL, "%s: rows of o overlap one another", who);
    const Range rs{reinterpret_cast<const char *>(state), sizeof(float) * states * p.heads * p.dim_k * p.dim_v};
    const Range ro{static_cast<const char *>(o), extent(p.o_stride, p.batch, 1, p.heads, p.dim_v, size)};
    for (const Range &x : {Range{static_cast<const char *>(q), extent(p.q_stride, p.batch, 1, p.heads_q, p.dim_k, size)},
                           Range{static_cast<const char *>(k), extent(p.k_stride, p.batch, 1, p.heads_k, p.dim_k, size)},
                           Range{static_cast<const char *>(v), extent(p.v_stride, p.batch, 1, p.heads_v, p.dim_v, size)},
                           Range{reinterpret_cast<const char *>(slots), slots ? sizeof(long long) * p.batch : 0}})
        if (meet(x, ro) || meet(x, rs)) return fail(DSP_GPU_EINVAL, "%s: o or the state overlaps an input", who);
    if (meet(ro, rs)) return fail(DSP_GPU_EINVAL, "%s: o overlaps the state", who);
    const size_t blocks = p.batch * p.heads * ((p.dim_v + kStepCols - 1) / kStepCols);
    if (blocks > 0x7fffffffu) return fail(DSP_GPU_EINVAL, "%s: %zu workgroups", who, blocks);
    a.q = q, a.k = k, a.v = v, a.o = o;
    a.qs[0] = p.q_stride[0], a.qs[1] = p.q_stride[2];
    a.ks[0] = p.k_stride[0], a.ks[1] = p.k_stride[2];
    a.vs[0] = p.v_stride[0], a.vs[1] = p.v_stride[2];
    a.os[0] = p.o_stride[0], a.os[1] = p.o_stride[2];
    a.q_group = p.heads / p.heads_q, a.k_group = p.heads / p.heads_k, a.v_group = p.heads / p.heads_v;
    a.heads = p.heads, a.d1 = p.dim_k, a.d2 = p.dim_v;
    a.batch = static_cast<int>(p.batch);
    a.scale = static_cast<float>(scale);
    a.vec = p.dim_v % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
    a.state = state;
    a.slots = slots;
    a.n_slots = static_cast<long long>(n_slots);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.sample_type == DSP_GPU_BF16) return launch_step<__bf16>(a, s);
    if (p.sample_type == DSP_GPU_F16) return launch_step<_Float16>(a, s);
    return launch_step<float>(a, s);
}

}  // extern "C"
