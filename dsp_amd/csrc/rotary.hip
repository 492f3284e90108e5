// rotary.hip -- rotary positions: pairs of each head turned by pos * inv_freq (dsp_gpu_rotary).
//
// Bound by the tensor's traffic, read once and written once.  The angle of a pair is the same for every head of a token, and
// forming it costs more than turning a pair (a double product reduced to turns, then cos and sin in fp32): a thread keeps
// the angles of its 16 bytes of pairs and turns them in up to kReuse heads.  65,536 tokens of 40 heads of 128 bf16: 248 us
// for 1.34 GB, 5.4 TB/s (a copy of 1 GiB: 5.1); 64 tokens of 20 heads: 4.3 us, a launch and two latencies.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.h"

namespace dspgpu {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kReuse = 8;

struct RotaryArgs {
    const void *x;
    void *y;
    long long xs[3], ys[3];
    const long long *positions;
    long long ps[2], position;
    unsigned n;               // tokens of a sequence
    int heads, head_lanes;    // a thread takes heads l, l + head_lanes, ...
    int rot, dim, chunks;     // chunks: threads of a row, the rotated ones first, then the copied ones
    int turned;               // of these, threads that turn pairs
    float gain, sign;
    unsigned long long threads;
    double turns[kMaxPairs];  // inv_freq / 2 pi
};

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
    T e[VE];
};

// VE elements a load; HALF: VE pairs a thread (two loads), else VE / 2 pairs (one load).  WIDE: rows are aligned to a load.
template <typename T, int VE, bool HALF, bool WIDE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    const unsigned long long id = static_cast<unsigned long long>(block_index()) * 256 + threadIdx.x;
    if (id >= a.threads) return;
    unsigned long long token;
    int chunk, lane;
    if (a.threads < (1ull << 32)) {
        const unsigned u = static_cast<unsigned>(id), v = u / a.chunks;
        chunk = u % a.chunks;
        lane = v % a.head_lanes;
        token = v / a.head_lanes;
    } else {
        const unsigned long long v = id / a.chunks;
        chunk = static_cast<int>(id % a.chunks);
        lane = static_cast<int>(v % a.head_lanes);
        token = v / a.head_lanes;
    }
    const long long b = token / a.n, t = token % a.n;
    const T *x = static_cast<const T *>(a.x) + b * a.xs[0] + t * a.xs[1];
    T *y = static_cast<T *>(a.y) + b * a.ys[0] + t * a.ys[1];
    auto load = [&](const T *p) {
        Vec<T, VE> v;
        if (WIDE) v = *reinterpret_cast<const Vec<T, VE> *>(p);
        else {
#pragma unroll
            for (int e = 0; e < VE; ++e) v.e[e] = p[e];
        }
        return v;
    };
    auto store = [&](T *p, const Vec<T, VE> &v) {
        if (WIDE) *reinterpret_cast<Vec<T, VE> *>(p) = v;
        else {
#pragma unroll
            for (int e = 0; e < VE; ++e) p[e] = v.e[e];
        }
    };
    if (chunk >= a.turned) {  // behind the rotated part
        const int at = a.rot + (chunk - a.turned) * VE;
        for (int h = lane; h < a.heads; h += a.head_lanes) {
            if (WIDE || at + VE <= a.dim) store(y + h * a.ys[2] + at, load(x + h * a.xs[2] + at));
            else
                for (int e = at; e < a.dim; ++e) y[h * a.ys[2] + e] = x[h * a.xs[2] + e];
        }
        return;
    }
    const double pos = static_cast<double>(a.positions ? a.positions[b * a.ps[0] + t * a.ps[1]] : a.position + t);
    constexpr int PAIRS = HALF ? VE : VE / 2;
    float c[PAIRS], s[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const double turn = pos * a.turns[chunk * PAIRS + i];
        const float part = static_cast<float>(turn - rint(turn));  // in [-1/2, 1/2] turns
        sincospif(2.0f * part, &s[i], &c[i]);
        s[i] *= a.gain * a.sign;
        c[i] *= a.gain;
    }
    const int at = chunk * VE, half = a.rot / 2;
#pragma unroll 2
    for (int h = lane; h < a.heads; h += a.head_lanes) {
        const T *xr = x + h * a.xs[2] + at;
        T *yr = y + h * a.ys[2] + at;
        if (HALF) {
            const Vec<T, VE> u = load(xr), v = load(xr + half);
            Vec<T, VE> p, q;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float x0 = static_cast<float>(u.e[i]), x1 = static_cast<float>(v.e[i]);
                p.e[i] = static_cast<T>(x0 * c[i] - x1 * s[i]);
                q.e[i] = static_cast<T>(x0 * s[i] + x1 * c[i]);
            }
            store(yr, p);
            store(yr + half, q);
        } else {
            const Vec<T, VE> u = load(xr);
            Vec<T, VE> p;
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const float x0 = static_cast<float>(u.e[2 * i]), x1 = static_cast<float>(u.e[2 * i + 1]);
                p.e[2 * i] = static_cast<T>(x0 * c[i] - x1 * s[i]);
                p.e[2 * i + 1] = static_cast<T>(x0 * s[i] + x1 * c[i]);
            }
            store(yr, p);
        }
    }
}

template <typename T, int VE, bool HALF, bool WIDE>
int launch(RotaryArgs &a, size_t rows, bool copy, hipStream_t s) {
    a.turned = HALF ? a.rot / 2 / VE : a.rot / VE;
    a.chunks = a.turned + (copy ? (a.dim - a.rot + VE - 1) / VE : 0);
    // Heads share a thread's angles, but the card is filled first: 2^19 threads are all it holds at once.
    const size_t most = rows * static_cast<size_t>(a.chunks) * a.heads;
    const int reuse = static_cast<int>(std::min<size_t>(kReuse, std::max<size_t>(1, most >> 19)));
    a.head_lanes = (a.heads + reuse - 1) / reuse;
    a.threads = static_cast<unsigned long long>(rows) * a.chunks * a.head_lanes;
    const unsigned long long blocks = (a.threads + 255) / 256;
    if (blocks > kMostBlocks) return fail(DSP_GPU_EINVAL, "dsp_gpu_rotary: %llu workgroups", blocks);
    rotary_kernel<T, VE, HALF, WIDE><<<grid_of(blocks), 256, 0, s>>>(a);
    return check_launch("rotary_kernel");
}

bool whole(const RotaryArgs &a, int ve, bool half, size_t size) {
    const uintptr_t mask = ve * size - 1;
    if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) & mask) return false;
    for (int i = 0; i < 3; ++i)
        if (a.xs[i] % ve || a.ys[i] % ve) return false;
    return (half ? a.rot / 2 : a.rot) % ve == 0 && a.dim % ve == 0;
}

// 16 bytes an access where rows allow it, else 8, else single elements
template <typename T>
int launch_type(RotaryArgs &a, size_t rows, bool half, bool copy, hipStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (whole(a, W, half, sizeof(T))) return half ? launch<T, W, true, true>(a, rows, copy, s) : launch<T, W, false, true>(a, rows, copy, s);
    if (whole(a, W / 2, half, sizeof(T))) return half ? launch<T, W / 2, true, true>(a, rows, copy, s) : launch<T, W / 2, false, true>(a, rows, copy, s);
    return half ? launch<T, 1, true, false>(a, rows, copy, s) : launch<T, 2, false, false>(a, rows, copy, s);
}

}  // namespace
}  // namespace dspgpu

using namespace dspgpu;

extern "C" int dsp_gpu_rotary(const void *x, void *y, int sample_type, size_t batch, size_t n, int heads, int dim,
                              const long long x_stride[3], const long long y_stride[3], const double *inv_freq, int rot_dim,
                              int layout, const long long *positions, const long long position_stride[2], long long position,
                              double gain, int direction, void *stream) {
    static const char *who = "dsp_gpu_rotary";
    if (sample_type != DSP_GPU_F32 && sample_type != DSP_GPU_F16 && sample_type != DSP_GPU_BF16)
        return fail(DSP_GPU_EINVAL, "%s: sample type %d (F32, F16 or BF16)", who, sample_type);
    if (!x_stride || !y_stride || !inv_freq || (positions && !position_stride)) return fail(DSP_GPU_EINVAL, "%s: null argument", who);
    if (heads < 1 || heads > 65536 || dim < 2 || dim > 1024) return fail(DSP_GPU_EINVAL, "%s: %d heads of %d elements", who, heads, dim);
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > dim || rot_dim > 2 * kMaxPairs)
        return fail(DSP_GPU_EINVAL, "%s: rot_dim %d (even, 2 ... min(dim, %d))", who, rot_dim, 2 * kMaxPairs);
    if (layout != DSP_GPU_ROTARY_HALF && layout != DSP_GPU_ROTARY_INTERLEAVED) return fail(DSP_GPU_EINVAL, "%s: layout %d", who, layout);
    if (direction != DSP_GPU_FORWARD && direction != DSP_GPU_INVERSE) return fail(DSP_GPU_EINVAL, "%s: direction %d", who, direction);
    if (!std::isfinite(gain)) return fail(DSP_GPU_EINVAL, "%s: non-finite gain", who);
    if (batch > (1ull << 31) || n > (1ull << 31)) return fail(DSP_GPU_EINVAL, "%s: too many tokens", who);
    RotaryArgs a{};
    for (int i = 0; i < rot_dim / 2; ++i) {
        if (!std::isfinite(inv_freq[i])) return fail(DSP_GPU_EINVAL, "%s: non-finite inv_freq[%d]", who, i);
        a.turns[i] = inv_freq[i] / 6.283185307179586476925286766559;
    }
    for (int i = 0; i < 3; ++i) {
        if (x_stride[i] < 0 || y_stride[i] < 0 || x_stride[i] > (1ll << 40) || y_stride[i] > (1ll << 40))
            return fail(DSP_GPU_EINVAL, "%s: stride %lld / %lld", who, x_stride[i], y_stride[i]);
        a.xs[i] = x_stride[i];
        a.ys[i] = y_stride[i];
    }
    if (positions && (position_stride[0] < 0 || position_stride[1] < 0)) return fail(DSP_GPU_EINVAL, "%s: negative position stride", who);
    if (batch == 0 || n == 0) return DSP_GPU_OK;
    if (!x || !y) return fail(DSP_GPU_EINVAL, "%s: null buffer", who);
    if (!extent_fits(x_stride, batch, n, heads, dim) || !extent_fits(y_stride, batch, n, heads, dim))
        return fail(DSP_GPU_EINVAL, "%s: x or y is larger than any memory", who);
    if (positions) {
        const long long st[3] = {position_stride[0], position_stride[1], 0};
        if (!extent_fits(st, batch, n, 1, 1)) return fail(DSP_GPU_EINVAL, "%s: positions are larger than any memory", who);
    }
    if (!rows_distinct(y_stride, batch, n, heads, dim)) return fail(DSP_GPU_EINVAL, "%s: rows of y overlap one another", who);
    const size_t size = sample_type == DSP_GPU_F32 ? 4 : 2;
    auto bytes = [&](const long long *st) { return ((batch - 1) * st[0] + (n - 1) * st[1] + (heads - 1) * st[2] + dim) * size; };
    const char *x0 = static_cast<const char *>(x), *y0 = static_cast<const char *>(y);
    bool in_place = x0 == y0;  // the same elements: every axis that has more than one step takes the same stride
    const size_t count[3] = {batch, n, static_cast<size_t>(heads)};
    for (int i = 0; i < 3; ++i) in_place = in_place && (count[i] <= 1 || x_stride[i] == y_stride[i]);
    if (!in_place && x0 < y0 + bytes(y_stride) && y0 < x0 + bytes(x_stride)) return fail(DSP_GPU_EINVAL, "%s: x and y overlap", who);
    if (positions) {
        const char *p0 = reinterpret_cast<const char *>(positions);
        const size_t pb = ((batch - 1) * position_stride[0] + (n - 1) * position_stride[1] + 1) * sizeof(long long);
        if (p0 < y0 + bytes(y_stride) && y0 < p0 + pb) return fail(DSP_GPU_EINVAL, "%s: positions and y overlap", who);
        a.ps[0] = position_stride[0];
        a.ps[1] = position_stride[1];
    }
    a.x = x;
    a.y = y;
    a.positions = positions;
    a.position = position;
    a.n = static_cast<unsigned>(n);
    a.heads = heads;
    a.dim = dim;
    a.rot = rot_dim;
    a.gain = static_cast<float>(gain);
    a.sign = direction == DSP_GPU_INVERSE ? -1.0f : 1.0f;
    const bool half = layout == DSP_GPU_ROTARY_HALF, copy = !in_place && rot_dim < dim;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t rows = batch * n;
    if (sample_type == DSP_GPU_BF16) return launch_type<__bf16>(a, rows, half, copy, s);
    if (sample_type == DSP_GPU_F16) return launch_type<_Float16>(a, rows, half, copy, s);
    return launch_type<float>(a, rows, half, copy, s);
}
