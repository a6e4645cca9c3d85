// Selective state space scan: a memory of N numbers a channel,
//     h[t][c][n] = e^(delta[t][c] rate[c][n]) h[t-1][c][n] + delta[t][c] x[t][c] write[t][n],   y[t][c] = sum_n read[t][n] h[t][c][n] + skip[c] x[t][c],
// and its backward pass.
//
// What bounds it: of a step, channel and state, an exponential (four issue slots of a vector unit) and four more operations; memory is a third of
// that.  A lane is a channel, so that write and read are the same for all lanes of a wavefront and come through scalar loads, and sums over the
// states need no exchange between lanes; a wavefront holds four states of 64 channels, a workgroup all states of them, and its wavefronts add up their
// parts of y through LDS, sixteen steps at a time.  Where sequences and channels do not fill the chip, time is cut into stretches: their end
// states from zero first (sums), what enters each of them then (join), and the stretches again from there.  A stretch's decay needs no
// product: it is e^(rate times the sum of its deltas).
//
// 65,536 x 1 x 1,024 x 16 bf16 forward: sums 232 us, join 32, the stretches again 345; seven and eight issue slots a state and step are 190 and 220 us of that at 2.4 GHz, staging a fifth.  4,096 x 4 x 2,048 x 16
// bf16 both ways 1.04 ms: back some 27 slots, of which five are sums over the lanes.  64 x 2,048 x 16, one step: 7.4 us, 2.4 TB/s.
#include <type_traits>

#include "readout.hpp"

namespace bmtk {
namespace {

constexpr int kSteps = BMTK_SCAN_MARK;   // steps of a block: what a workgroup stages at once, and of which a state is kept
constexpr int kOwn = 4;                  // states of a wavefront
constexpr int64_t kFewSteps = 8;         // up to which the steps are taken one by one
constexpr float kLog2e = 1.44269504f;
constexpr float kLeast = 1.17549435e-38f;   // a stretch's decay is at least this, so that an infinite state stays infinite

struct SelArgs {
    const void *x, *dt, *write, *read, *dy;
    const float *rate, *skip, *dt_bias, *state, *d_last;
    const int32_t *lengths;
    void *y, *dx, *d_dt, *d_write, *d_read;
    float *last, *marks, *d_rate, *d_skip, *d_dt_bias, *d_state;
    float *spread;            // [batch][groups][waves][padded_steps][2][kOwn]: write and read in 32 bits, 0 behind a sequence's end
    float *ends;              // [stretches][batch][dim][padded]: a stretch's end from zero, then what enters it
    float *deltas;            // [stretches][batch][dim]: sum of a stretch's deltas
    float *part_write, *part_read;   // [tiles][batch][groups][waves][n_steps][kOwn]: sums over a tile's channels
    float *part_rate;         // [stretches][batch][dim][padded]
    float *part_skip, *part_bias;    // [stretches][batch][dim]
    int64_t n_steps, batch, x_t, x_b, dt_t, dt_b, write_t, write_b, read_t, read_b, dy_t, dy_b;
    int64_t padded_steps;     // n_steps, to whole blocks
    int64_t stretch_steps;    // a multiple of kSteps
    int32_t dim, groups, n_states, waves, padded, channels, tiles, stretches, softplus;   // padded: waves * kOwn; channels, tiles: of a group
};

// write and read as the main kernels see them: of the constant address space, so that they come through scalar loads (an earlier kernel has written them)
typedef __attribute__((address_space(4))) const float Shared;

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

// log(1 + e^v) and its derivative.  With e = e^-|v| it is max(v, 0) + log(1 + e), and log(1 + e) = 2 artanh(e / (2 + e)), whose argument is at most 1/3:
// the series to the 15th power leaves 2^-27 of it, and nothing cancels where e is small.
__device__ __forceinline__ float softplus_of(float v)
{
    const float e = exp2_of(-kLog2e * fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = 1.0f / 15;
    p = fmaf(p, q, 1.0f / 13);
    p = fmaf(p, q, 1.0f / 11);
    p = fmaf(p, q, 1.0f / 9);
    p = fmaf(p, q, 1.0f / 7);
    p = fmaf(p, q, 1.0f / 5);
    p = fmaf(p, q, 1.0f / 3);
    p = fmaf(p, q, 1.0f);
    return fmaf(2.0f * s, p, v > 0.0f ? v : v != v ? v : 0.0f);
}
__device__ __forceinline__ float softplus_slope(float v)
{
    const float e = exp2_of(-kLog2e * fabsf(v));
    return (v >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e);
}

// ---------------------------------------------------------------------------------------------------------------------
// write and read in 32 bits, a wavefront's four states of both next to one another and step behind step, for scalar loads

template <typename T>
__global__ __launch_bounds__(256) void spread_kernel(SelArgs a, int64_t rows)
{
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k >= rows * a.padded) return;
    const int64_t row = k / a.padded;                  // (t * batch + b) * groups + g
    const int32_t n = (int32_t)(k - row * a.padded);
    const int64_t tb = row / a.groups;
    const int32_t g = (int32_t)(row - tb * a.groups);
    const int64_t t = tb / a.batch, b = tb - t * a.batch;
    const bool there = n < a.n_states && t < (a.lengths ? min((int64_t)a.lengths[b], a.n_steps) : a.n_steps);
    float w = 0.0f, r = 0.0f;
    if (there) {
        w = (float)static_cast<const T *>(a.write)[t * a.write_t + b * a.write_b + (int64_t)g * a.n_states + n];
        r = (float)static_cast<const T *>(a.read)[t * a.read_t + b * a.read_b + (int64_t)g * a.n_states + n];
    }
    float *to = a.spread + ((((b * a.groups + g) * a.waves + n / kOwn) * a.padded_steps + t) * 2) * kOwn + n % kOwn;
    to[0] = w;
    to[kOwn] = r;
}

// ---------------------------------------------------------------------------------------------------------------------

// what a workgroup works on: 64 channels of a group (fewer in its last tile), a sequence, a stretch of steps
struct Tile {
    int32_t lane, wave, g, c;      // c: this lane's channel, or the group's last one for lanes without
    int64_t b, t0, t1, end;        // steps t0 <= t < t1 of the stretch; end: the sequence's length
    bool there;
    __device__ __forceinline__ Tile(const SelArgs &a)
    {
        lane = lane_id();
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        const int32_t tile = blockIdx.x % a.tiles;
        const int32_t gb = blockIdx.x / a.tiles;
        g = gb % a.groups;
        // (the sequences in another order in every stretch: workgroups whose numbers are some power of two apart share a compute unit, and sequences end early)
        b = gb / a.groups + blockIdx.y % a.batch;
        b -= b >= a.batch ? a.batch : 0;
        const int32_t in_group = tile * kWave + lane;
        there = in_group < a.channels;
        c = g * a.channels + min(in_group, a.channels - 1);
        t0 = (int64_t)blockIdx.y * a.stretch_steps;
        t1 = min(t0 + a.stretch_steps, a.n_steps);
        end = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.n_steps) : a.n_steps;
    }
    __device__ __forceinline__ int64_t column(const SelArgs &a) const { return b * a.dim + c; }
};

// rates of the wavefront's four states, times log2 e, and other numbers of [..][padded] or [..][n_states] (the ones behind the last state are 0)
__device__ __forceinline__ void get_states(const float *p, int32_t n0, int32_t n, bool whole, float (&v)[kOwn])
{
    if (whole) {
        const Pack<float, kOwn> q = *reinterpret_cast<const Pack<float, kOwn> *>(p + n0);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) v[i] = q.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) v[i] = n0 + i < n ? p[n0 + i] : 0.0f;
    }
}
__device__ __forceinline__ void put_states(float *p, int32_t n0, int32_t n, bool whole, const float (&v)[kOwn])
{
    if (whole) {
        Pack<float, kOwn> q;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) q.v[i] = v[i];
        *reinterpret_cast<Pack<float, kOwn> *>(p + n0) = q;
    } else {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (n0 + i < n) p[n0 + i] = v[i];
    }
}

// whether rows of n_states numbers from p on can be read four at a time
__device__ __forceinline__ bool whole_states(const SelArgs &a, const void *p) { return a.n_states % kOwn == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Inputs of a block of steps on their way from memory: a wavefront takes the rows wave, wave + waves, ...
template <typename T, typename TD, int Rows, bool Backward>
struct Inputs {
    T x[Rows], dy[Backward ? Rows : 1];
    TD dt[Rows];
    __device__ __forceinline__ void ask(const SelArgs &a, const Tile &at, int64_t t)
    {
        const T *x_from = static_cast<const T *>(a.x) + at.b * a.x_b + at.c;
        const TD *dt_from = static_cast<const TD *>(a.dt) + at.b * a.dt_b + at.c;
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            // (a step that is there: what lies behind the end is cut when it is used)
            const int64_t step = max(min(t + at.wave + r * a.waves, at.end - 1), (int64_t)0);
            x[r] = x_from[step * a.x_t];
            dt[r] = dt_from[step * a.dt_t];
            if constexpr (Backward) dy[r] = (static_cast<const T *>(a.dy) + at.b * a.dy_b + at.c)[step * a.dy_t];
        }
    }
};

__device__ __forceinline__ float delta_of(const SelArgs &a, float v) { return a.softplus ? softplus_of(v) : v; }

// ---------------------------------------------------------------------------------------------------------------------
// forward, for up to Waves wavefronts, of which each stages and finishes up to Rows rows of a block.  Sums: only the ends of the stretches, from zero.

template <typename T, typename TD, int Waves, int Rows, bool Sums>
__global__ __launch_bounds__(Waves * kWave) void selective_fwd_kernel(SelArgs a)
{
    extern __shared__ float lds[];
    float2 *staged = reinterpret_cast<float2 *>(lds);                 // [kSteps][kWave]: delta, delta x
    float *parts = lds + 2 * kSteps * kWave;                          // [waves][kSteps][kWave]: y's sum over a wavefront's states
    const Tile at(a);
    const int32_t n0 = at.wave * kOwn;
    const int64_t column = at.column(a);
    float rate[kOwn], h[kOwn];
    get_states(a.rate + (int64_t)at.c * a.n_states, n0, a.n_states, whole_states(a, a.rate), rate);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) rate[i] *= kLog2e, h[i] = 0.0f;
    if (!Sums) {
        if (a.stretches > 1) get_states(a.ends + ((int64_t)blockIdx.y * a.batch * a.dim + column) * a.padded, n0, a.n_states, true, h);
        else if (a.state) get_states(a.state + column * a.n_states, n0, a.n_states, whole_states(a, a.state), h);
    }
    const float bias = a.dt_bias ? a.dt_bias[at.c] : 0.0f, skip = a.skip ? a.skip[at.c] : 0.0f;
    const Shared *spread = (const Shared *)(a.spread + ((at.b * a.groups + at.g) * a.waves + at.wave) * a.padded_steps * 2 * kOwn);
    Inputs<T, TD, Rows, false> in;
    in.ask(a, at, at.t0);
    float total = 0.0f;
    for (int64_t t = at.t0; t < at.t1; t += kSteps) {
        float x[Rows];
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const int row = at.wave + r * a.waves;
            const bool there = at.there && t + row < at.end && t + row < at.t1;
            x[r] = there ? (float)in.x[r] : 0.0f;
            const float delta = there ? delta_of(a, (float)in.dt[r] + bias) : 0.0f;
            if (row < kSteps) staged[row * kWave + at.lane] = make_float2(delta, there ? delta * x[r] : 0.0f);
            if (Sums) total += row < kSteps ? delta : 0.0f;
        }
        __syncthreads();
        if (t + kSteps < at.t1) in.ask(a, at, t + kSteps);
        if (!Sums && a.marks && at.there) put_states(a.marks + (t / kSteps * a.batch * a.dim + column) * a.n_states, n0, a.n_states, whole_states(a, a.marks), h);
        if (t < at.end) {
            const Shared *wr = spread + t * 2 * kOwn;
            // (a step behind the stretch's last one has delta and delta x 0, and changes nothing)
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const float2 d = staged[k * kWave + at.lane];
                float y = 0.0f;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    h[i] = fmaf(exp2_of(d.x * rate[i]), h[i], d.y * wr[k * 2 * kOwn + i]);
                    if (!Sums) y = fmaf(wr[k * 2 * kOwn + kOwn + i], h[i], y);
                }
                if (!Sums) parts[(at.wave * kSteps + k) * kWave + at.lane] = y;
            }
        }
        __syncthreads();
        if (!Sums) {
            T *y_to = static_cast<T *>(a.y) + (t * a.batch + at.b) * a.dim + at.c;
#pragma unroll
            for (int r = 0; r < Rows; ++r) {
                const int row = at.wave + r * a.waves;
                if (row >= kSteps || t + row >= at.t1 || !at.there) continue;
                float y = 0.0f;
                if (t + row < at.end) {
                    y = skip * x[r];
                    for (int w = 0; w < a.waves; ++w) y += parts[(w * kSteps + row) * kWave + at.lane];
                }
                y_to[row * a.batch * a.dim] = (T)y;
            }
        }
    }
    if (Sums) {
        if (at.there) put_states(a.ends + ((int64_t)blockIdx.y * a.batch * a.dim + column) * a.padded, n0, a.padded, true, h);
        // (the last barrier is behind what was read of it)
        lds[at.wave * kWave + at.lane] = total;
        __syncthreads();
        if (at.wave == 0 && at.there) {
            for (int w = 1; w < a.waves; ++w) total += lds[w * kWave + at.lane];
            a.deltas[(int64_t)blockIdx.y * a.batch * a.dim + column] = total;
        }
    } else if (at.there && (int32_t)blockIdx.y == a.stretches - 1) {
        put_states(a.last + column * a.n_states, n0, a.n_states, whole_states(a, a.last), h);
    }
}

// A few steps, with the states as they lie in memory: a lane has four of a channel's, Lanes neighbouring lanes the channel's all, and y is summed over those.  Bound
// by the states, read and written.
template <typename T, typename TD, int Lanes>
__global__ __launch_bounds__(256) void selective_step_kernel(SelArgs a, FastDiv by_dim, FastDiv by_channels)
{
    const uint32_t q = blockIdx.x * 256u + threadIdx.x, column = q / Lanes;
    const int32_t n0 = (int32_t)(q % Lanes) * kOwn;
    if (column >= (uint32_t)(a.batch * a.dim)) return;   // (Lanes divides a wavefront: a channel's lanes leave together)
    const uint32_t b = div_by(column, by_dim), c = column - b * (uint32_t)a.dim, g = div_by(c, by_channels);
    const bool whole = whole_states(a, a.rate) && whole_states(a, a.last) && (!a.state || whole_states(a, a.state)) && n0 < a.n_states;
    const int64_t end = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.n_steps) : a.n_steps;
    float rate[kOwn], h[kOwn];
    get_states(a.rate + (int64_t)c * a.n_states, n0, a.n_states, whole, rate);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) rate[i] *= kLog2e, h[i] = 0.0f;
    if (a.state) get_states(a.state + (int64_t)column * a.n_states, n0, a.n_states, whole, h);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.skip ? a.skip[c] : 0.0f;
    for (int64_t t = 0; t < a.n_steps; ++t) {
        if (t % kSteps == 0 && a.marks) put_states(a.marks + (t / kSteps * a.batch * a.dim + column) * a.n_states, n0, a.n_states, false, h);
        float y = 0.0f;
        if (t < end) {
            const float x = (float)static_cast<const T *>(a.x)[t * a.x_t + b * a.x_b + c];
            const float delta = delta_of(a, (float)static_cast<const TD *>(a.dt)[t * a.dt_t + b * a.dt_b + c] + bias), u = delta * x;
            const T *write = static_cast<const T *>(a.write) + t * a.write_t + b * a.write_b + (int64_t)g * a.n_states;
            const T *read = static_cast<const T *>(a.read) + t * a.read_t + b * a.read_b + (int64_t)g * a.n_states;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                if (n0 + i >= a.n_states) continue;
                h[i] = fmaf(exp2_of(delta * rate[i]), h[i], u * (float)write[n0 + i]);
                y = fmaf((float)read[n0 + i], h[i], y);
            }
#pragma unroll
            for (int k = 1; k < Lanes; k *= 2) y += __shfl_xor(y, k);
            y = fmaf(skip, x, y);
        }
        if (n0 == 0) static_cast<T *>(a.y)[(t * a.batch + b) * a.dim + c] = (T)y;
    }
    put_states(a.last + (int64_t)column * a.n_states, n0, a.n_states, whole, h);
}

// What enters each stretch, from its neighbour's: in the order of time from the state, or (Back) against it from the last state's gradient
template <bool Back>
__global__ __launch_bounds__(256) void selective_join_kernel(SelArgs a, int64_t columns)
{
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, column = k / a.padded;
    const int32_t n = (int32_t)(k - column * a.padded);
    if (column >= columns) return;
    const int32_t c = (int32_t)(column % a.dim);
    const bool there = n < a.n_states;
    const float *given = Back ? a.d_last : a.state;
    const float rate = there ? a.rate[(int64_t)c * a.n_states + n] * kLog2e : 0.0f;
    float s = there && given ? given[column * a.n_states + n] : 0.0f;
    const int64_t step = columns * a.padded;
    constexpr int kAhead = 8;
    for (int32_t j = 0; j < a.stretches; j += kAhead) {
        float end[kAhead], delta[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int32_t at = min(j + i, a.stretches - 1), q = Back ? a.stretches - 1 - at : at;
            end[i] = a.ends[q * step + k];
            delta[i] = a.deltas[q * columns + column];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (j + i >= a.stretches) break;
            const int32_t q = Back ? a.stretches - 1 - j - i : j + i;
            a.ends[q * step + k] = s;
            const float decay = exp2_of(delta[i] * rate);
            s = fmaf(decay < kLeast ? kLeast : decay, s, end[i]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// backward.  g[t] = dy read + e[t+1] g[t+1] is the gradient by h[t]; with q = g e[t] h[t-1]
//     d_read = sum_c dy h,  d_write = sum_c g delta x,  s1 = sum_n g write,  s2 = sum_n q rate,  d_rate = sum_t q delta,
//     dx = delta s1 + skip dy,  d_delta = x s1 + s2.
// Of a block of steps a wavefront first makes its states again from the one that was kept, then goes through the block from its end.

// Sums of two registers over pairs of lanes 32 (16) apart: a's in the lower lanes of a pair, b's in the upper ones
__device__ __forceinline__ float add_halves(float x, float y)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_rows(float x, float y)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the same within rows of 16 lanes, for pairs `1 << Bit` apart
template <int Bit>
__device__ __forceinline__ float add_pairs(float x, float y, int lane)
{
    constexpr int kCtrl = Bit == 3 ? 0x128 /* row_ror:8 */ : Bit == 2 ? 0x124 : Bit == 1 ? 0x4E /* quad_perm 2,3,0,1 */ : 0xB1 /* quad_perm 1,0,3,2 */;
    const bool upper = lane >> Bit & 1;
    const float keep = upper ? y : x, send = upper ? x : y;
    return keep + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(send), kCtrl, 0xF, 0xF, true));
}

// v[k], k < 16: a row of 16 lanes holds 16 numbers each; lane l of it gets the sum over the row of number l
__device__ __forceinline__ float sum_rows(float (&v)[kSteps], int lane)
{
    // (lanes 4 apart within 8: a rotation by 4 goes beyond them, so that the halves of 8 are exchanged by a mirror first)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = add_pairs<3>(v[k], v[k + 8], lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool upper = lane >> 2 & 1;
        const float keep = upper ? v[k + 4] : v[k], send = upper ? v[k] : v[k + 4];
        // lane ^ 7 (row_half_mirror), then ^ 3 (quad_perm 3,2,1,0)
        const int m = __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(send), 0x141, 0xF, 0xF, true);
        v[k] = keep + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, m, 0x1B, 0xF, 0xF, true));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = add_pairs<1>(v[k], v[k + 2], lane);
    return add_pairs<0>(v[0], v[1], lane);
}

// (two wavefronts a SIMD, where a workgroup has no more: of a few states, whose wavefronts stage many rows, the compiler would take more registers than that leaves)
template <typename T, typename TD, int Waves, int Rows, bool Sums>
__global__ __launch_bounds__(Waves * kWave, Waves == 16 ? 4 : 2) void selective_bwd_kernel(SelArgs a)
{
    // A block's decays and states are kept in registers, 128 of them; of 16 wavefronts, which have no more, by halves, the first half made twice
    constexpr int kParts = Waves == 16 ? 2 : 1, kEach = kSteps / kParts;
    extern __shared__ float lds[];
    float4 *staged = reinterpret_cast<float4 *>(lds);                        // [kSteps][kWave]: delta, x, dy, slope of delta
    float2 *parts = reinterpret_cast<float2 *>(lds + 4 * kSteps * kWave);    // [waves][kSteps][kWave]: s1, s2 of a wavefront's states
    const Tile at(a);
    const int32_t n0 = at.wave * kOwn;
    const int64_t column = at.column(a);
    float rate[kOwn], rate2[kOwn], back[kOwn], d_rate[kOwn];   // back: e[t+1] g[t+1]
    get_states(a.rate + (int64_t)at.c * a.n_states, n0, a.n_states, whole_states(a, a.rate), rate);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) rate2[i] = rate[i] * kLog2e, back[i] = d_rate[i] = 0.0f;
    if (!Sums) {
        if (a.stretches > 1) get_states(a.ends + ((int64_t)blockIdx.y * a.batch * a.dim + column) * a.padded, n0, a.n_states, true, back);
        else if (a.d_last) get_states(a.d_last + column * a.n_states, n0, a.n_states, whole_states(a, a.d_last), back);
    }
    const float bias = a.dt_bias ? a.dt_bias[at.c] : 0.0f, skip = a.skip ? a.skip[at.c] : 0.0f;
    const Shared *spread = (const Shared *)(a.spread + ((at.b * a.groups + at.g) * a.waves + at.wave) * a.padded_steps * 2 * kOwn);
    const int64_t part_row = (((int64_t)(blockIdx.x % a.tiles) * a.batch + at.b) * a.groups + at.g) * a.waves + at.wave;
    Inputs<T, TD, Rows, true> in;
    const int64_t t_last = at.t0 + (at.t1 - at.t0 - 1) / kSteps * kSteps;
    in.ask(a, at, t_last);
    float total = 0.0f, d_skip = 0.0f, d_bias = 0.0f;
    for (int64_t t = t_last; t >= at.t0; t -= kSteps) {
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const int row = at.wave + r * a.waves;
            const bool there = at.there && t + row < at.end && t + row < at.t1 && row < kSteps;
            const float v = (float)in.dt[r] + bias, delta = there ? delta_of(a, v) : 0.0f, slope = Sums || !there ? 0.0f : a.softplus ? softplus_slope(v) : 1.0f;
            if (row < kSteps) staged[row * kWave + at.lane] = make_float4(delta, there ? (float)in.x[r] : 0.0f, there ? (float)in.dy[r] : 0.0f, slope);
            if (Sums) total += delta;
        }
        __syncthreads();
        if (t > at.t0) in.ask(a, at, t - kSteps);
        // (steps behind the stretch's last one have delta, x and dy 0)
        if (t < at.end) {
            const Shared *wr = spread + t * 2 * kOwn;
            if constexpr (Sums) {
#pragma unroll
                for (int k = kSteps - 1; k >= 0; --k) {
                    const float d = staged[k * kWave + at.lane].x, dy_k = staged[k * kWave + at.lane].z;
                    const Shared *w = wr + k * 2 * kOwn;
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) back[i] = exp2_of(d * rate2[i]) * fmaf(dy_k, w[kOwn + i], back[i]);
                }
            } else {
                float first[kOwn], middle[kOwn];
                get_states(a.marks + (t / kSteps * a.batch * a.dim + column) * a.n_states, n0, a.n_states, whole_states(a, a.marks), first);
                if (!at.there)   // (a neighbour's may be infinite, and is not this lane's to add up)
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) first[i] = 0.0f;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) middle[i] = first[i];
                if constexpr (kParts == 2) {
#pragma unroll
                    for (int k = 0; k < kEach; ++k) {
                        if (k % 4 == 0) asm volatile("" : "+s"(wr), "+v"(middle[0]));
                        const float4 d = staged[k * kWave + at.lane];
                        const float u = d.x * d.y;
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) middle[i] = fmaf(u, wr[k * 2 * kOwn + i], exp2_of(d.x * rate2[i]) * middle[i]);
                    }
                }
                float sum_read[kSteps], sum_write[kSteps];
#pragma unroll
                for (int part = kParts - 1; part >= 0; --part) {
                    float e[kEach][kOwn], eh[kEach][kOwn], h[kOwn];
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) h[i] = part ? middle[i] : first[i];
#pragma unroll
                    for (int k = 0; k < kEach; ++k) {
                        if (k % 4 == 0) asm volatile("" : "+s"(wr), "+v"(h[0]));
                        const float4 d = staged[(part * kEach + k) * kWave + at.lane];
                        const float u = d.x * d.y;
                        const Shared *w = wr + (part * kEach + k) * 2 * kOwn;
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) {
                            e[k][i] = exp2_of(d.x * rate2[i]);
                            eh[k][i] = e[k][i] * h[i];
                            h[i] = fmaf(u, w[i], eh[k][i]);
                        }
                    }
#pragma unroll
                    for (int q = kEach - 1; q >= 0; --q) {
                        const int k = part * kEach + q;
                        // (write and read are asked for again, four steps at a time: there are no scalar registers to keep those of the block in)
                        if (k % 4 == 3) asm volatile("" : "+s"(wr), "+v"(back[0]));
                        const float4 d = staged[k * kWave + at.lane];
                        const float u = d.x * d.y, dy_k = d.z;
                        const Shared *w = wr + k * 2 * kOwn;
                        float s1 = 0.0f, s2 = 0.0f, by_read[kOwn], by_write[kOwn];
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) {
                            const float g = fmaf(dy_k, w[kOwn + i], back[i]);
                            by_read[i] = dy_k * fmaf(u, w[i], eh[q][i]);
                            by_write[i] = g * u;
                            s1 = fmaf(g, w[i], s1);
                            const float by_decay = g * eh[q][i];
                            s2 = fmaf(by_decay, rate[i], s2);
                            d_rate[i] = fmaf(by_decay, d.x, d_rate[i]);
                            back[i] = e[q][i] * g;
                        }
                        parts[(at.wave * kSteps + k) * kWave + at.lane] = make_float2(s1, s2);
                        // states 0 and 2, 1 and 3 share a register, in halves; then all four, in rows of 16 lanes: 0, 1, 2, 3
                        sum_read[k] = add_rows(add_halves(by_read[0], by_read[2]), add_halves(by_read[1], by_read[3]));
                        sum_write[k] = add_rows(add_halves(by_write[0], by_write[2]), add_halves(by_write[1], by_write[3]));
                    }
                }
                const float r = sum_rows(sum_read, at.lane), w = sum_rows(sum_write, at.lane);
                // lane l of a row of 16: the step whose bits were told apart in the order 8, 4, 2, 1
                const int k = at.lane & 15, i = at.lane >> 4;
                if (t + k < at.t1) {
                    const int64_t to = (part_row * a.n_steps + t + k) * kOwn + i;
                    a.part_read[to] = t + k < at.end ? r : 0.0f;
                    a.part_write[to] = t + k < at.end ? w : 0.0f;
                }
            }
        } else if (!Sums) {
            const int k = at.lane & 15, i = at.lane >> 4;
            if (t + k < at.t1) {
                const int64_t to = (part_row * a.n_steps + t + k) * kOwn + i;
                a.part_read[to] = a.part_write[to] = 0.0f;
            }
        }
        __syncthreads();
        if (!Sums) {
#pragma unroll
            for (int r = 0; r < Rows; ++r) {
                const int row = at.wave + r * a.waves;
                if (row >= kSteps || t + row >= at.t1 || !at.there) continue;
                float s1 = 0.0f, s2 = 0.0f;
                if (t + row < at.end)
                    for (int w = 0; w < a.waves; ++w) {
                        const float2 p = parts[(w * kSteps + row) * kWave + at.lane];
                        s1 += p.x;
                        s2 += p.y;
                    }
                const bool there = t + row < at.end;
                const float4 d = staged[row * kWave + at.lane];   // (this wavefront's own)
                const float dx = there ? fmaf(d.x, s1, skip * d.z) : 0.0f, d_dt = there ? fmaf(d.y, s1, s2) * d.w : 0.0f;
                const int64_t to = ((t + row) * a.batch + at.b) * a.dim + at.c;
                static_cast<T *>(a.dx)[to] = (T)dx;
                static_cast<TD *>(a.d_dt)[to] = (TD)d_dt;
                d_skip = fmaf(d.z, d.y, d_skip);
                d_bias += d_dt;
            }
        }
    }
    const int64_t stretch_column = (int64_t)blockIdx.y * a.batch * a.dim + column;
    if (Sums) {
        if (at.there) put_states(a.ends + stretch_column * a.padded, n0, a.padded, true, back);
        lds[at.wave * kWave + at.lane] = total;
        __syncthreads();
        if (at.wave == 0 && at.there) {
            for (int w = 1; w < a.waves; ++w) total += lds[w * kWave + at.lane];
            a.deltas[stretch_column] = total;
        }
        return;
    }
    if (at.there) {
        put_states(a.part_rate + stretch_column * a.padded, n0, a.padded, true, d_rate);
        if (blockIdx.y == 0 && a.d_state) put_states(a.d_state + column * a.n_states, n0, a.n_states, whole_states(a, a.d_state), back);
    }
    float2 *sums = reinterpret_cast<float2 *>(lds);
    __syncthreads();
    sums[at.wave * kWave + at.lane] = make_float2(d_skip, d_bias);
    __syncthreads();
    if (at.wave == 0 && at.there) {
        for (int w = 1; w < a.waves; ++w) {
            const float2 p = sums[w * kWave + at.lane];
            d_skip += p.x;
            d_bias += p.y;
        }
        a.part_skip[stretch_column] = d_skip;
        a.part_bias[stretch_column] = d_bias;
    }
}

// d_write and d_read from their sums over each tile's channels
template <typename T>
__global__ __launch_bounds__(256) void selective_join_shared_kernel(SelArgs a, int64_t total)
{
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;   // [batch][groups][waves][n_steps][kOwn]
    if (k >= total) return;
    float r = 0.0f, w = 0.0f;
    for (int j = 0; j < a.tiles; ++j) {
        r += a.part_read[j * total + k];
        w += a.part_write[j * total + k];
    }
    const int32_t i = (int32_t)(k % kOwn);
    int64_t row = k / kOwn;
    const int64_t t = row % a.n_steps;
    row /= a.n_steps;
    const int32_t wave = (int32_t)(row % a.waves);
    row /= a.waves;
    const int64_t g = row % a.groups, b = row / a.groups;
    const int32_t n = wave * kOwn + i;
    if (n >= a.n_states) return;
    const int64_t to = ((t * a.batch + b) * a.groups + g) * a.n_states + n;
    static_cast<T *>(a.d_read)[to] = (T)r;
    static_cast<T *>(a.d_write)[to] = (T)w;
}

// sums of `parts` rows: of [parts][dim * padded] (d_rate), [parts][dim] (d_skip, d_dt_bias).  A workgroup takes 64 numbers, each wavefront every sixteenth row.
__global__ __launch_bounds__(1024) void selective_join_channels_kernel(SelArgs a, int64_t parts, int64_t rate_blocks, int64_t dim_blocks)
{
    __shared__ float sums[16][64];
    const int wave = threadIdx.x / 64, lane = lane_id();
    int64_t block = blockIdx.x;
    const float *from = a.part_rate;
    int64_t width = (int64_t)a.dim * a.padded;
    int which = 0;
    if (block >= rate_blocks) {
        block -= rate_blocks;
        which = block >= dim_blocks ? 2 : 1;
        if (which == 2) block -= dim_blocks;
        from = which == 1 ? a.part_skip : a.part_bias;
        width = a.dim;
    }
    const int64_t col = block * 64 + lane;
    float s = 0.0f;
    if (col < width) {
        const float *p = from + col;
        int64_t k = wave;
        for (; k + 7 * 16 < parts; k += 8 * 16) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[(k + i * 16) * width];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; k < parts; k += 16) s += p[k * width];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= width) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sums[i][lane];
    if (which == 0) {
        const int64_t c = col / a.padded;
        const int32_t n = (int32_t)(col - c * a.padded);
        if (n < a.n_states) a.d_rate[c * a.n_states + n] = s;
    } else {
        float *to = which == 1 ? a.d_skip : a.d_dt_bias;
        if (to) to[col] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------------

struct Plan {
    int32_t waves, padded, channels, tiles, stretches;
    int64_t stretch_steps, padded_steps, spread, ends, deltas, shared, rate, per_dim;   // sizes in numbers
    Plan(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t n_states, bool backward)
    {
        waves = (int32_t)div_up(n_states, kOwn);
        padded = waves * kOwn;
        channels = dim / groups;
        tiles = (int32_t)div_up(channels, kWave);
        // Stretches cost their sums beforehand, which are about as much again, but a workgroup waits for its own wavefronts twice a block: from some 4,096 wavefronts on
        // (back, where a block is three times as long, 2,048) one stretch does.  us of 2,000 x 8 x 4,096 x 16, 2,048 wavefronts: forward 624 in one stretch, 490 in eight;
        // back 1,240 and 1,430.  Otherwise as many as make 16,384, down to a block each: 65,536 x 1 x 1,024 x 16 forward 688 with 4,096, 580 with 12,288, 562 with 16,384;
        // 600 x 32 x 64 x 8 fp32 both ways 153 with stretches of four blocks, 113 of two, 98 of one.
        const int64_t across = batch * groups * tiles * waves, blocks = div_up(n_steps, kSteps);
        int64_t s = across >= (backward ? 2048 : 4096) ? 1 : div_up(16384, across);
        // What enters the stretches is found one after the other, eight of them in the time of 20 steps or so: not more than the root of three times the steps, either.  us with as many as above, with
        // the root of once and of three times the steps: 65,536 x 1 x 5 x 16 both ways 1,004, 413, 336; 30,000 x 1 x 100 x 16 582, 326, 312; 5,000 x 1 x 300 x 1 161, 220, 164.
        int64_t root = 64;
        while (root * root < 3 * n_steps) root += 8;
        if (s > root) s = root;
        if (s > blocks) s = blocks;
        if (s > 65535) s = 65535;   // (a launch's rows of workgroups)
        const int64_t each = div_up(blocks, s);
        stretch_steps = each * kSteps;
        stretches = (int32_t)div_up(blocks, each);
        padded_steps = blocks * kSteps;
        spread = batch * groups * waves * padded_steps * 2 * kOwn;
        ends = stretches > 1 ? stretches * batch * dim * padded : 0;
        deltas = stretches > 1 ? stretches * batch * dim : 0;
        shared = backward ? (int64_t)tiles * batch * groups * waves * n_steps * kOwn : 0;
        rate = backward ? stretches * batch * dim * padded : 0;
        per_dim = backward ? stretches * batch * dim : 0;
    }
    static int64_t room(int64_t n) { return div_up(n, 64) * 64; }
    int64_t numbers() const { return room(spread) + room(ends) + room(deltas) + 2 * room(shared) + room(rate) + 2 * room(per_dim); }
    void place(SelArgs &a, float *ws) const
    {
        const auto next = [&](int64_t n) {
            float *p = ws;
            ws += room(n);
            return p;
        };
        a.spread = next(spread), a.ends = next(ends), a.deltas = next(deltas), a.part_write = next(shared), a.part_read = next(shared), a.part_rate = next(rate);
        a.part_skip = next(per_dim), a.part_bias = next(per_dim);
        a.waves = waves, a.padded = padded, a.channels = channels, a.tiles = tiles, a.stretches = stretches, a.stretch_steps = stretch_steps, a.padded_steps = padded_steps;
    }
};

bool sizes_fit(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t n_states)
{
    if (!(n_steps > 0 && batch > 0 && dim > 0 && groups > 0 && dim % groups == 0 && n_states > 0 && n_states <= BMTK_SELECTIVE_MAX_STATES && n_steps < (int64_t{1} << 31) - 4096 &&
          batch < (int64_t{1} << 31) && batch * dim < (int64_t{1} << 31)))
        return false;
    // 2^32 threads a launch, whole workgroups: one for each state of a step, of a channel; sixteen where a channel's sums are put together, which are P and two, lanes without a channel with the
    // others
    const int64_t most = (int64_t{1} << 32) - 256, padded = div_up(n_states, kOwn) * kOwn, rows = div_up(n_steps, kSteps) * kSteps * batch * groups;
    const int64_t lanes = batch * groups * div_up(dim / groups, kWave) * kWave, sums = (div_up(dim * padded, 64) + 2 * div_up(dim, 64)) * 1024;
    return rows < most && rows * padded < most && batch * dim * padded < most && sums < most && lanes < most && lanes * (padded / kOwn) < most;
}

template <typename T, typename TD, int Waves, int Rows>
int launch(const char *name, const SelArgs &a, dim3 grid, bool backward, hipStream_t s)
{
    const uint32_t threads = (uint32_t)a.waves * kWave;
    const int64_t columns = a.batch * a.dim;
    const uint32_t joins = (uint32_t)div_up(columns * a.padded, 256);
    const int32_t unit = kSteps * kWave * 4, lds = (backward ? 4 + 2 * a.waves : 2 + a.waves) * unit;
    if constexpr (Waves > 4) {
        // more than 64 KB of LDS (of 160) has to be asked for, once per kernel and device
        static bool asked[2][64];
        int dev = 0;
        hipError_t err = hipGetDevice(&dev);
        if (err == hipSuccess && !(dev >= 0 && dev < 64 && asked[backward][dev])) {
            const void *kernel = backward ? reinterpret_cast<const void *>(selective_bwd_kernel<T, TD, Waves, Rows, false>)
                                          : reinterpret_cast<const void *>(selective_fwd_kernel<T, TD, Waves, Rows, false>);
            err = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (backward ? 4 + 2 * Waves : 2 + Waves) * unit);
            if (err == hipSuccess && dev >= 0 && dev < 64) asked[backward][dev] = true;
        }
        if (err != hipSuccess) {
            set_error("%s: cannot reserve LDS: %s", name, hipGetErrorString(err));
            return BMTK_E_LAUNCH;
        }
    }
    // (the sums over wavefronts of a stretch's delta and of d_skip and d_bias need two times kWave numbers for up to 16 wavefronts: what is staged)
    if (!backward) {
        if (a.stretches > 1) {
            selective_fwd_kernel<T, TD, Waves, Rows, true><<<grid, threads, 2 * unit, s>>>(a);
            selective_join_kernel<false><<<joins, 256, 0, s>>>(a, columns);
        }
        selective_fwd_kernel<T, TD, Waves, Rows, false><<<grid, threads, lds, s>>>(a);
    } else {
        if (a.stretches > 1) {
            selective_bwd_kernel<T, TD, Waves, Rows, true><<<grid, threads, 4 * unit, s>>>(a);
            selective_join_kernel<true><<<joins, 256, 0, s>>>(a, columns);
        }
        selective_bwd_kernel<T, TD, Waves, Rows, false><<<grid, threads, lds, s>>>(a);
    }
    BMTK_CHECK_LAUNCH(name);
    return 0;
}

template <typename T, typename TD>
int launch_rows(const char *name, const SelArgs &a, dim3 grid, bool backward, hipStream_t s)
{
    if (a.waves == 1) return launch<T, TD, 1, 16>(name, a, grid, backward, s);
    if (a.waves <= 3) return launch<T, TD, 3, 8>(name, a, grid, backward, s);
    if (a.waves == 4) return launch<T, TD, 4, 4>(name, a, grid, backward, s);
    if (a.waves <= 8) return launch<T, TD, 8, 4>(name, a, grid, backward, s);
    return launch<T, TD, 16, 2>(name, a, grid, backward, s);
}

template <typename T, typename TD>
int launch_step(const char *name, const SelArgs &a, hipStream_t s)
{
    int lanes = 1;
    while (lanes * kOwn < a.n_states) lanes *= 2;
    const int64_t threads = a.batch * a.dim * lanes;
    const uint32_t blocks = (uint32_t)div_up(threads, 256);
    const FastDiv by_dim = fast_div((uint32_t)a.dim), by_channels = fast_div((uint32_t)(a.dim / a.groups));
    switch (lanes) {
        case 1: selective_step_kernel<T, TD, 1><<<blocks, 256, 0, s>>>(a, by_dim, by_channels); break;
        case 2: selective_step_kernel<T, TD, 2><<<blocks, 256, 0, s>>>(a, by_dim, by_channels); break;
        case 4: selective_step_kernel<T, TD, 4><<<blocks, 256, 0, s>>>(a, by_dim, by_channels); break;
        case 8: selective_step_kernel<T, TD, 8><<<blocks, 256, 0, s>>>(a, by_dim, by_channels); break;
        default: selective_step_kernel<T, TD, 16><<<blocks, 256, 0, s>>>(a, by_dim, by_channels);
    }
    BMTK_CHECK_LAUNCH(name);
    return 0;
}

// Whether the steps are few enough for the kernel that takes them one by one: it has one launch instead of two
bool few_steps(int64_t n_steps, int64_t batch, int32_t dim) { return n_steps <= kFewSteps && batch * dim < (int64_t{1} << 27); }

int run(const char *name, SelArgs &a, int32_t dtype, int32_t dt_dtype, bool backward, float *workspace, hipStream_t s)
{
    BMTK_REQUIRE(a.n_steps > 0 && a.batch > 0 && a.dim > 0 && a.groups > 0 && a.n_states > 0, "%s: sizes must be positive", name);
    BMTK_REQUIRE(a.dim % a.groups == 0, "%s: %d channels are not divided evenly by %d groups", name, a.dim, a.groups);
    BMTK_REQUIRE(a.n_states <= BMTK_SELECTIVE_MAX_STATES, "%s: up to %d states, got %d", name, BMTK_SELECTIVE_MAX_STATES, a.n_states);
    BMTK_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown type %d", name, dtype);
    BMTK_REQUIRE(dt_dtype == BMTK_F32 || dt_dtype == dtype, "%s: dt must be float32 or of the type of x", name);
    BMTK_REQUIRE(sizes_fit(a.n_steps, a.batch, a.dim, a.groups, a.n_states), "%s: too many steps, columns or states", name);
    if (!backward && few_steps(a.n_steps, a.batch, a.dim)) {
        BMTK_BY_TYPE(dtype, T, { return dt_dtype == BMTK_F32 ? launch_step<T, float>(name, a, s) : launch_step<T, T>(name, a, s); });
    }
    const Plan plan(a.n_steps, a.batch, a.dim, a.groups, a.n_states, backward);
    const int64_t across = a.batch * a.groups * plan.tiles, rows = plan.padded_steps * a.batch * a.groups;
    BMTK_REQUIRE(workspace, "%s: needs a workspace", name);
    plan.place(a, workspace);
    BMTK_BY_TYPE(dtype, T, { spread_kernel<T><<<(uint32_t)div_up(rows * plan.padded, 256), 256, 0, s>>>(a, rows); });
    BMTK_CHECK_LAUNCH(name);
    const dim3 grid((uint32_t)across, (uint32_t)plan.stretches);
    BMTK_BY_TYPE(dtype, T, {
        const int failed = dt_dtype == BMTK_F32 ? launch_rows<T, float>(name, a, grid, backward, s) : launch_rows<T, T>(name, a, grid, backward, s);
        if (failed) return failed;
    });
    if (!backward) return 0;
    const int64_t shared = plan.shared / plan.tiles;
    BMTK_BY_TYPE(dtype, T, { selective_join_shared_kernel<T><<<(uint32_t)div_up(shared, 256), 256, 0, s>>>(a, shared); });
    const int64_t rate_blocks = div_up((int64_t)a.dim * plan.padded, 64), dim_blocks = div_up(a.dim, 64);
    selective_join_channels_kernel<<<(uint32_t)(rate_blocks + 2 * dim_blocks), 1024, 0, s>>>(a, (int64_t)plan.stretches * a.batch, rate_blocks, dim_blocks);
    BMTK_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_selective_scan_workspace_bytes(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t n_states, int32_t backward)
{
    if (!sizes_fit(n_steps, batch, dim, groups, n_states) || (!backward && few_steps(n_steps, batch, dim))) return 0;
    return Plan(n_steps, batch, dim, groups, n_states, backward != 0).numbers() * 4;
}

extern "C" int bmtk_selective_scan_fwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t n_states, int32_t dtype, int32_t dt_dtype, int32_t softplus,
                                       const void *x, int64_t x_t, int64_t x_b, const void *dt, int64_t dt_t, int64_t dt_b, const void *write, int64_t write_t,
                                       int64_t write_b, const void *read, int64_t read_t, int64_t read_b, const float *rate, const float *skip, const float *dt_bias,
                                       const float *state, const int32_t *lengths, void *y, float *last, float *marks, float *workspace, void *stream)
{
    BMTK_REQUIRE(x && dt && write && read && rate && y && last, "selective_scan_fwd: null pointer");
    SelArgs a{};
    a.x = x, a.dt = dt, a.write = write, a.read = read, a.rate = rate, a.skip = skip, a.dt_bias = dt_bias, a.state = state, a.lengths = lengths, a.y = y, a.last = last, a.marks = marks;
    a.n_steps = n_steps, a.batch = batch, a.dim = dim, a.groups = groups, a.n_states = n_states, a.softplus = softplus != 0;
    a.x_t = x_t, a.x_b = x_b, a.dt_t = dt_t, a.dt_b = dt_b, a.write_t = write_t, a.write_b = write_b, a.read_t = read_t, a.read_b = read_b;
    return run("selective_scan_fwd", a, dtype, dt_dtype, false, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int bmtk_selective_scan_bwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t n_states, int32_t dtype, int32_t dt_dtype, int32_t softplus,
                                       const void *x, int64_t x_t, int64_t x_b, const void *dt, int64_t dt_t, int64_t dt_b, const void *write, int64_t write_t,
                                       int64_t write_b, const void *read, int64_t read_t, int64_t read_b, const float *rate, const float *skip, const float *dt_bias,
                                       const float *marks, const int32_t *lengths, const void *dy, int64_t dy_t, int64_t dy_b, const float *d_last, void *dx, void *d_dt,
                                       void *d_write, void *d_read, float *d_rate, float *d_skip, float *d_dt_bias, float *d_state, float *workspace, void *stream)
{
    BMTK_REQUIRE(x && dt && write && read && rate && marks && dy && dx && d_dt && d_write && d_read && d_rate, "selective_scan_bwd: null pointer");
    SelArgs a{};
    a.x = x, a.dt = dt, a.write = write, a.read = read, a.rate = rate, a.skip = skip, a.dt_bias = dt_bias, a.lengths = lengths, a.dy = dy, a.d_last = d_last;
    a.marks = const_cast<float *>(marks);
    a.dx = dx, a.d_dt = d_dt, a.d_write = d_write, a.d_read = d_read, a.d_rate = d_rate, a.d_skip = d_skip, a.d_dt_bias = d_dt_bias, a.d_state = d_state;
    a.n_steps = n_steps, a.batch = batch, a.dim = dim, a.groups = groups, a.n_states = n_states, a.softplus = softplus != 0;
    a.x_t = x_t, a.x_b = x_b, a.dt_t = dt_t, a.dt_b = dt_b, a.write_t = write_t, a.write_b = write_b, a.read_t = read_t, a.read_b = read_b, a.dy_t = dy_t, a.dy_b = dy_b;
    return run("selective_scan_bwd", a, dtype, dt_dtype, true, workspace, static_cast<hipStream_t>(stream));
}
