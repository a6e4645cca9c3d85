// Short causal convolution over the steps of many sequences, a few taps a channel, with or without a silu, and its backward pass.
//
// With the inputs before the first step (state) in front, z[t] = bias + sum_j w[j] x[t - (W - 1) + j] and y = z or z sigmoid(z).  Bound by
// memory: a thread takes 16 bytes of neighbouring channels and a stretch of steps, and keeps the W - 1 rows before the present one in
// registers, so that each row is read once, and W - 1 again at the start of a stretch.  65,536 x 1,000 fp32, three taps: 112 us, 4.8 TB/s.  4,096 x 8 x 2,048 bf16, ragged, four taps and a silu:
// forward 51 us, 4.1 TB/s; back 88, 3.6, since a thread's 250 registers leave two wavefronts a SIMD, and an entry takes some 35 vector instructions.
#include "readout.hpp"

namespace bmtk {
namespace {

constexpr int kAhead = 4;   // rows of x (and dy) that a thread asks for at once

struct ConvArgs {
    const void *x, *w, *bias, *state;
    const int32_t *lengths;
    const void *dy, *d_last;
    void *y, *last, *dx, *d_state;
    float *part;                // [stretches * batch][dim * (width + 1)]: sums of a stretch, the weights' and then the bias's
    int64_t n_steps, x_t, x_b, dy_t, dy_b, batch;
    int32_t dim, vectors, width, stretch, silu;
    FastDiv by_vectors;
};

// neighbouring numbers wherever they begin, as they lie in memory: loads of 16 or 8 bytes where their size allows
template <typename T, int V>
struct Raw {
    static constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : (int)sizeof(T), kLoads = kBytes / kWord;
    typedef uint32_t Words __attribute__((ext_vector_type(kWord >= 8 ? kWord / 4 : 1)));
    typedef Words Loose __attribute__((aligned(2)));
    union {
        Words w[kLoads];
        T v[V];
    };
    __device__ __forceinline__ Raw() {}
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if constexpr (kWord >= 8) w[i] = reinterpret_cast<const Loose *>(p)[i];
            else v[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T *p) const
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if constexpr (kWord >= 8) reinterpret_cast<Loose *>(p)[i] = w[i];
            else p[i] = v[i];
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ void get(const T *p, float (&v)[V])
{
    Raw<T, V> q;
    q.load(p);
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = (float)q.v[c];
}

template <typename T, int V>
__device__ __forceinline__ void put(T *p, const float (&v)[V])
{
    Raw<T, V> q;
#pragma unroll
    for (int c = 0; c < V; ++c) q.v[c] = (T)v[c];
    q.store(p);
}

// 1 / (1 + e^-z)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }

// What a thread works on: V channels from c on of sequence b, steps t0 <= t < t1.  Of a number of channels that V does not divide the last
// vector begins earlier, so that some channels are computed twice, to the same bits.
template <int V>
struct Place {
    int64_t t0, t1, end;
    int32_t b, c;
    bool there;
    __device__ __forceinline__ Place(const ConvArgs &a)
    {
        const uint32_t q = blockIdx.x * 256u + threadIdx.x;
        b = (int32_t)div_by(q, a.by_vectors);
        c = min((int32_t)(q - (uint32_t)b * a.vectors) * V, a.dim - V);
        there = b < a.batch;
        t0 = (int64_t)blockIdx.y * a.stretch;
        t1 = min(t0 + a.stretch, a.n_steps);
        end = a.n_steps;
        if (there && a.lengths) end = min(max((int64_t)a.lengths[b], (int64_t)0), a.n_steps);
    }
};

// Taps of a thread's channels; W is the width or, where that is 5 to 8, 8 with the taps in front of it left out everywhere
template <typename TW, int W, int V>
struct Taps {
    float w[W][V], bias[V];
    __device__ __forceinline__ Taps(const ConvArgs &a, int32_t c)
    {
        const TW *p = static_cast<const TW *>(a.w) + (int64_t)c * a.width;
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) w[j][k] = 0.0f;
        if constexpr (W < 8) {
            float flat[W * V];
            get<TW, W * V>(p, flat);
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) w[j][k] = flat[k * W + j];
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (j >= W - a.width)
#pragma unroll
                    for (int k = 0; k < V; ++k) w[j][k] = (float)p[k * a.width + j - (W - a.width)];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) bias[k] = 0.0f;
        if (a.bias) get<TW, V>(static_cast<const TW *>(a.bias) + c, bias);
    }
};

// x of step t, of the state where t < 0, 0 behind the sequence's end and in front of what the taps reach
template <typename T, int V>
__device__ __forceinline__ void input(const ConvArgs &a, const Place<V> &at, int64_t t, float (&v)[V])
{
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
    if (t >= 0) {
        if (t < at.end) get<T, V>(static_cast<const T *>(a.x) + t * a.x_t + at.b * a.x_b + at.c, v);
    } else if (a.state && t >= 1 - a.width) {
        get<T, V>(static_cast<const T *>(a.state) + ((t + a.width - 1) * a.batch + at.b) * a.dim + at.c, v);
    }
}

// Rows t .. t + kAhead - 1 as they lie in memory; of a step behind the sequence's end the last one that it has, or the first: nothing
// outside is read and there are no branches, so that the loads are all under way at once
template <typename T, int V>
__device__ __forceinline__ void ask(const T *p, int64_t stride, int64_t t, int64_t end, Raw<T, V> (&raw)[kAhead])
{
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u].load(p + max(min(t + u, end - 1), (int64_t)0) * stride);
}

template <typename T, int V>
__device__ __forceinline__ void take(const Raw<T, V> &raw, bool there, float (&v)[V])
{
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = there ? (float)raw.v[k] : 0.0f;
}

template <typename T, typename TW, int W, int V>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs a)
{
    const Place<V> at(a);
    if (!at.there) return;
    const Taps<TW, W, V> taps(a, at.c);
    const int first = W - a.width;   // (tap of a width of 5 to 7)
    float x[W - 1 + kAhead][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) input<T, V>(a, at, at.t0 - (W - 1) + j, x[j]);
    T *y = static_cast<T *>(a.y) + (at.t0 * a.batch + at.b) * a.dim + at.c;
    const T *from = static_cast<const T *>(a.x) + at.b * a.x_b + at.c;
    Raw<T, V> raw[kAhead];
    ask<T, V>(from, a.x_t, at.t0, at.end, raw);
    for (int64_t t = at.t0; t < at.t1; t += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) take<T, V>(raw[u], t + u < at.end, x[W - 1 + u]);
        if (t + kAhead < at.t1) ask<T, V>(from, a.x_t, t + kAhead, at.end, raw);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (t + u >= at.t1) break;
            float z[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                z[k] = taps.bias[k];
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (W < 8 || j >= first) z[k] = fmaf(taps.w[j][k], x[u + j][k], z[k]);
            }
            if (a.silu) {
#pragma unroll
                for (int k = 0; k < V; ++k) z[k] *= sigmoid(z[k]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) z[k] = t + u < at.end ? z[k] : 0.0f;
            put<T, V>(y, z);
            y += a.batch * a.dim;
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) x[j][k] = x[j + kAhead][k];
    }
    if (blockIdx.y == 0) {
        T *last = static_cast<T *>(a.last) + (int64_t)at.b * a.dim + at.c;
        for (int j = 0; j < a.width - 1; ++j) {
            float v[V];
            input<T, V>(a, at, at.end - (a.width - 1) + j, v);
            put<T, V>(last + j * a.batch * a.dim, v);
        }
    }
}

// dz[t] = dy[t] dy/dz, dx[t'] = sum_j w[j] dz[t' + (W - 1) - j], the same for the state at t' < 0.  A thread makes z again from x, goes W - 1 steps
// further than its stretch for dz, and adds up its own steps' parts of the weights' gradient.
template <typename T, typename TW, int W, int V>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs a)
{
    const Place<V> at(a);
    if (!at.there) return;
    const Taps<TW, W, V> taps(a, at.c);
    const int first = W - a.width;
    float x[W - 1 + kAhead][V], dz[W - 1 + kAhead][V], dw[W][V], db[V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        input<T, V>(a, at, at.t0 - (W - 1) + j, x[j]);
#pragma unroll
        for (int k = 0; k < V; ++k) dz[j][k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        db[k] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][k] = 0.0f;
    }
    // (the first stretch has the state's gradient in front of it)
    const int64_t from = blockIdx.y == 0 ? 1 - (int64_t)a.width : at.t0;
    const T *x_from = static_cast<const T *>(a.x) + at.b * a.x_b + at.c, *dy_from = static_cast<const T *>(a.dy) + at.b * a.dy_b + at.c;
    Raw<T, V> x_raw[kAhead], dy_raw[kAhead];
    ask<T, V>(x_from, a.x_t, at.t0, at.end, x_raw);
    ask<T, V>(dy_from, a.dy_t, at.t0, at.end, dy_raw);
    for (int64_t t = at.t0; t < at.t1 + W - 1; t += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            take<T, V>(x_raw[u], t + u < at.end, x[W - 1 + u]);
            take<T, V>(dy_raw[u], t + u < at.end, dz[W - 1 + u]);
        }
        if (t + kAhead < at.t1 + W - 1) {
            ask<T, V>(x_from, a.x_t, t + kAhead, at.end, x_raw);
            ask<T, V>(dy_from, a.dy_t, t + kAhead, at.end, dy_raw);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (a.silu) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float z = taps.bias[k];
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (W < 8 || j >= first) z = fmaf(taps.w[j][k], x[u + j][k], z);
                    const float p = sigmoid(z);
                    // (behind the end dy is 0, and z may be anything)
                    dz[W - 1 + u][k] = t + u < at.end ? dz[W - 1 + u][k] * fmaf(z * p, 1.0f - p, p) : 0.0f;
                }
            }
            // (x before the sequence's end may be infinite where dz behind it is 0)
            if (t + u < min(at.t1, at.end)) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    db[k] += dz[W - 1 + u][k];
#pragma unroll
                    for (int j = 0; j < W; ++j) dw[j][k] = fmaf(dz[W - 1 + u][k], x[u + j][k], dw[j][k]);
                }
            }
            const int64_t to = t + u - (W - 1);
            if (to < from || to >= at.t1) continue;
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[k] = 0.0f;
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (W < 8 || j >= first) v[k] = fmaf(taps.w[j][k], dz[W - 1 + u - j][k], v[k]);
            }
            const int64_t j = to - at.end + a.width - 1;   // which of the last inputs this is
            if (a.d_last && j >= 0 && to < at.end) {
                float d[V];
                get<T, V>(static_cast<const T *>(a.d_last) + (j * a.batch + at.b) * a.dim + at.c, d);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] += d[k];
            }
            if (to >= at.end) {   // (dz is 0 there; said so, since a weight may be infinite)
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = 0.0f;
            }
            if (to >= 0) put<T, V>(static_cast<T *>(a.dx) + (to * a.batch + at.b) * a.dim + at.c, v);
            else if (a.d_state) put<T, V>(static_cast<T *>(a.d_state) + ((to + a.width - 1) * a.batch + at.b) * a.dim + at.c, v);
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) x[j][k] = x[j + kAhead][k], dz[j][k] = dz[j + kAhead][k];
    }
    float *part = a.part + ((int64_t)blockIdx.y * a.batch + at.b) * a.dim * (a.width + 1);
    if constexpr (W < 8) {
        float flat[W * V];
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) flat[k * W + j] = dw[j][k];
        put<float, W * V>(part + (int64_t)at.c * W, flat);
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (j >= first)
#pragma unroll
                for (int k = 0; k < V; ++k) part[(int64_t)(at.c + k) * a.width + j - first] = dw[j][k];
    }
    put<float, V>(part + (int64_t)a.dim * a.width + at.c, db);
}

// sums of `parts` rows of `columns` numbers: a workgroup takes 64 columns, each of its 16 wavefronts every sixteenth row
template <typename TW>
__global__ __launch_bounds__(1024) void conv_join_kernel(const float *part, int64_t parts, int32_t columns, int32_t weights, TW *d_w, TW *d_bias)
{
    __shared__ float sums[16][64];
    const int wave = threadIdx.x / 64, lane = lane_id(), col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < columns) {
        const float *p = part + col;
        int64_t k = wave;
        for (; k + 7 * 16 < parts; k += 8 * 16) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[(k + i * 16) * columns];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; k < parts; k += 16) s += p[k * columns];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= columns) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sums[i][lane];
    if (col < weights) d_w[col] = (TW)s;
    else if (d_bias) d_bias[col - weights] = (TW)s;
}

// Steps of a thread.  Long stretches read fewer rows twice and leave fewer sums to join; the chip wants some 2,048 wavefronts.
int32_t stretch_of(int64_t n_steps, int64_t batch, int32_t dim, int32_t v)
{
    const int64_t threads = batch * div_up(dim, v), wanted = div_up((int64_t)2048 * 64, threads);
    int64_t s = div_up(n_steps, wanted);
    s = s < 8 ? 8 : s > 64 ? 64 : s;
    // (a launch has up to 65,535 rows of workgroups)
    while (div_up(n_steps, s) > 65535) s *= 2;
    return (int32_t)s;
}

// Channels of a thread.  Back, where a thread has twice as much to keep, eight of 16 bits only with four taps or fewer (eight taps are 250 registers with eight channels), rows that begin
// at whole 16 bytes, and enough of them: us of eight and four, 4,096 x 8 x 2,048 88/103; 3,000 x 16 x 641 fp16, two taps 91/79; 30,000 x 1 x 100 75/50.
int32_t vector_of(int64_t n_steps, int64_t batch, int32_t dim, int32_t dtype, int32_t width, bool backward, bool whole)
{
    const bool eight = dtype != BMTK_F32 && (!backward || (width <= 4 && whole && div_up(n_steps, 8) * batch * (dim / 8) >= 2048 * 64));
    return dim >= 8 && eight ? 8 : dim >= 4 ? 4 : 1;
}

template <typename T, typename TW, int W, int V>
void launch(const ConvArgs &a, dim3 grid, bool backward, hipStream_t s)
{
    if constexpr (W < 8 || V < 8)   // (see vector_of)
        if (backward) return conv_bwd_kernel<T, TW, W, V><<<grid, 256, 0, s>>>(a);
    conv_fwd_kernel<T, TW, W, V><<<grid, 256, 0, s>>>(a);
}

template <typename T, typename TW, int V>
void launch_width(const ConvArgs &a, dim3 grid, bool backward, hipStream_t s)
{
    switch (a.width) {
        case 2: return launch<T, TW, 2, V>(a, grid, backward, s);
        case 3: return launch<T, TW, 3, V>(a, grid, backward, s);
        case 4: return launch<T, TW, 4, V>(a, grid, backward, s);
        default: return launch<T, TW, 8, V>(a, grid, backward, s);
    }
}

template <typename T, typename TW>
void launch_vector(const ConvArgs &a, int32_t v, dim3 grid, bool backward, hipStream_t s)
{
    if (v == 1) return launch_width<T, TW, 1>(a, grid, backward, s);
    if (v == 4) return launch_width<T, TW, 4>(a, grid, backward, s);
    if constexpr (sizeof(T) == 2) return launch_width<T, TW, 8>(a, grid, backward, s);
}

int run(const char *name, int32_t dtype, int32_t weight_dtype, ConvArgs &a, bool backward, void *d_weight, void *d_bias, void *stream)
{
    BMTK_REQUIRE(a.n_steps > 0 && a.batch > 0 && a.dim > 0, "%s: sizes must be positive", name);
    BMTK_REQUIRE(a.width >= 2 && a.width <= BMTK_CONV_MAX_WIDTH, "%s: width must lie in 2..%d, got %d", name, BMTK_CONV_MAX_WIDTH, a.width);
    BMTK_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown type %d", name, dtype);
    BMTK_REQUIRE(weight_dtype == BMTK_F32 || weight_dtype == dtype, "%s: weights must be float32 or of the type of x", name);
    BMTK_REQUIRE(a.n_steps < (int64_t{1} << 31) - 4096 && a.batch < (int64_t{1} << 31) && a.batch * a.dim < (int64_t{1} << 31), "%s: too many steps or columns", name);
    const auto whole = [](const void *p, int64_t t, int64_t b) { return t % 8 == 0 && b % 8 == 0 && aligned(p, 16); };
    const int32_t v = vector_of(a.n_steps, a.batch, a.dim, dtype, a.width, backward, a.dim % 8 == 0 && whole(a.x, a.x_t, a.x_b) && whole(a.dy, a.dy_t, a.dy_b) && aligned(a.dx, 16));
    a.vectors = (int32_t)div_up(a.dim, v);
    a.by_vectors = fast_div((uint32_t)a.vectors);
    a.stretch = stretch_of(a.n_steps, a.batch, a.dim, v);
    const int64_t across = div_up(a.batch * a.vectors, 256), down = div_up(a.n_steps, a.stretch);
    BMTK_REQUIRE(across * 256 < (int64_t{1} << 31), "%s: too many columns", name);
    // (sixteen threads of the sums' launch for each weight and bias)
    BMTK_REQUIRE(!backward || (int64_t)a.dim * (a.width + 1) < (int64_t{1} << 28), "%s: too many weights for a launch", name);
    // (stretches are a launch's second size, so that 2^32 threads are never asked for in one)
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)across, (uint32_t)down);
    BMTK_BY_TYPE(dtype, T, {
        if (weight_dtype == BMTK_F32) launch_vector<T, float>(a, v, grid, backward, s);
        else launch_vector<T, T>(a, v, grid, backward, s);
    });
    BMTK_CHECK_LAUNCH(name);
    if (!backward) return 0;
    const int32_t columns = a.dim * (a.width + 1);
    BMTK_BY_TYPE(weight_dtype, TW, {
        conv_join_kernel<TW><<<(uint32_t)div_up(columns, 64), 1024, 0, s>>>(a.part, down * a.batch, columns, a.dim * a.width, static_cast<TW *>(d_weight), static_cast<TW *>(d_bias));
    });
    BMTK_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_short_conv_workspace_bytes(int64_t n_steps, int64_t batch, int32_t dim, int32_t width, int32_t dtype)
{
    if (n_steps <= 0 || batch <= 0 || dim <= 0 || width < 2 || width > BMTK_CONV_MAX_WIDTH || dtype < 0 || dtype > 2 || batch >= (int64_t{1} << 31) ||
        batch * dim >= (int64_t{1} << 31) || n_steps >= (int64_t{1} << 31) - 4096)
        return 0;
    int64_t stretches = 0;   // (of the call's strides, which decide, nothing is known here)
    for (const bool whole : {false, true}) {
        const int64_t n = div_up(n_steps, stretch_of(n_steps, batch, dim, vector_of(n_steps, batch, dim, dtype, width, true, whole)));
        stretches = n > stretches ? n : stretches;
    }
    return stretches * batch * dim * (width + 1) * 4;
}

extern "C" int bmtk_short_conv_fwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t silu, const void *x, int64_t x_t,
                                   int64_t x_b, const void *weight, const void *bias, const void *state, const int32_t *lengths, void *y, void *last, void *stream)
{
    BMTK_REQUIRE(x && weight && y && last, "short_conv_fwd: null pointer");
    ConvArgs a{};
    a.x = x, a.w = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.y = y, a.last = last;
    a.n_steps = n_steps, a.x_t = x_t, a.x_b = x_b, a.batch = batch, a.dim = dim, a.width = width, a.silu = silu != 0;
    return run("short_conv_fwd", dtype, weight_dtype, a, false, nullptr, nullptr, stream);
}

extern "C" int bmtk_short_conv_bwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t silu, const void *x, int64_t x_t,
                                   int64_t x_b, const void *weight, const void *bias, const void *state, const int32_t *lengths, const void *dy, int64_t dy_t, int64_t dy_b,
                                   const void *d_last, void *dx, void *d_weight, void *d_bias, void *d_state, float *workspace, void *stream)
{
    BMTK_REQUIRE(x && weight && dy && dx && d_weight, "short_conv_bwd: null pointer");
    BMTK_REQUIRE(workspace, "short_conv_bwd: needs a workspace");
    ConvArgs a{};
    a.x = x, a.w = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.dy = dy, a.d_last = d_last, a.dx = dx, a.d_state = d_state, a.part = workspace;
    a.n_steps = n_steps, a.x_t = x_t, a.x_b = x_b, a.dy_t = dy_t, a.dy_b = dy_b, a.batch = batch, a.dim = dim, a.width = width, a.silu = silu != 0;
    return run("short_conv_bwd", dtype, weight_dtype, a, true, d_weight, d_bias, stream);
}
