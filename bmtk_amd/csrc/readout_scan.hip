// Gated linear recurrence over the steps of many sequences, h[t] = a[t] h[t - 1] + x[t], and its backward pass.
#include <type_traits>

#include "readout.hpp"

namespace bmtk {
namespace {

constexpr int kSteps = BMTK_SCAN_MARK;  // steps that a wavefront holds in registers; the state before each such block is kept
constexpr int kMaxWaves = 8, kRoundWaves = 16;   // of a workgroup that takes rounds; of one that takes a single one

// One column is one channel of one sequence: column q = sequence q / dim, channel q % dim.  A lane takes V neighbouring columns.
struct ScanArgs {
    const void *x, *a;
    const float *state;
    const int32_t *lengths;
    void *h;
    float *last, *marks;
    const void *dh;
    const float *d_last;
    void *dx, *da;
    float *d_state, *da_part;   // da_part: partial sums of the gates' gradient
    float *sums;                // [splits][2][columns]: product of the gates and end state of a stretch, see scan_sums
    int64_t n_steps, columns, split_steps;
    int64_t x_t, x_b, a_t, a_b, dh_t, dh_b;   // strides of what is read, in elements; what is written is contiguous
    int32_t dim, channels;      // channels of a gate
    int32_t seg_lanes;          // lanes whose part of a gate's gradient is summed at once
    int32_t parts;              // such sums of a step and sequence
    int64_t sequences;
};

template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, bool there, float other, float (&v)[V])
{
    if (there) {
        const Pack<T, V> q = *reinterpret_cast<const Pack<T, V> *>(p);
#pragma unroll
        for (int c = 0; c < V; ++c) v[c] = (float)q.v[c];
    } else {
#pragma unroll
        for (int c = 0; c < V; ++c) v[c] = other;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, const float (&v)[V])
{
    Pack<T, V> q;
#pragma unroll
    for (int c = 0; c < V; ++c) q.v[c] = (T)v[c];
    *reinterpret_cast<Pack<T, V> *>(p) = q;
}

// Gates: one per channel for all steps, one per channel and step, or one per step for several neighbouring channels (a lane's are of one gate)
enum { kConst = 0, kEach = 1, kShared = 2 };

// A lane's part of a block of steps as it lies in memory, in whole registers: two 16-bit numbers stay in one until they are computed with
template <typename T, int V>
struct Block {
    static constexpr int kBytes = V * (int)sizeof(T), kRegs = (kBytes + 3) / 4;
    uint32_t w[kSteps][kRegs];
    // `last`: the last step that one of the wavefront's sequences has (or step 0); behind it that one again: nothing outside is read, there are no
    // branches, and those steps are cut
    __device__ __forceinline__ void load(const T *p, int64_t stride, int64_t t0, int64_t last)
    {
        int64_t at = min(t0, last);
        const T *row = p + at * stride;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            if constexpr (kBytes == 2) {
                w[k][0] = *reinterpret_cast<const uint16_t *>(row);
            } else {
                const Pack<uint32_t, kRegs> q = *reinterpret_cast<const Pack<uint32_t, kRegs> *>(row);
#pragma unroll
                for (int r = 0; r < kRegs; ++r) w[k][r] = q.v[r];
            }
            row += at < last ? stride : 0;
            ++at;
        }
    }
    // steps from `there` on are as if they were `other`
    __device__ __forceinline__ void cut(int there, float other)
    {
        uint32_t o;
        if constexpr (sizeof(T) == 4) {
            o = __float_as_uint(other);
        } else {
            const T h = (T)other;
            uint16_t bits;
            __builtin_memcpy(&bits, &h, 2);
            o = bits * 0x10001u;
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int r = 0; r < kRegs; ++r) w[k][r] = k < there ? w[k][r] : o;
    }
    // (of a single number, that one whatever c is)
    __device__ __forceinline__ float get(int k, int c) const
    {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[k][V == 1 ? 0 : c]);
        } else if constexpr (std::is_same<T, bf16>::value) {
            return __uint_as_float(V == 1 || c == 0 ? w[k][0] << 16 : w[k][0] & 0xffff0000u);
        } else {
            const uint16_t bits = (uint16_t)(V == 1 || c == 0 ? w[k][0] : w[k][0] >> 16);
            f16 h;
            __builtin_memcpy(&h, &bits, 2);
            return (float)h;
        }
    }
    // What follows makes its 32-bit numbers of the block again: kept from before they would be twice the registers.
    __device__ __forceinline__ void again()
    {
        if (sizeof(T) == 4) return;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) asm volatile("" : "+v"(w[k][0]));
    }
};

// What a lane knows of its columns
template <int V>
struct Lane {
    int64_t col;
    bool in;
    int32_t b, ch, len, longest;   // longest: of the wavefront's sequences
    int gate;
};
template <int V, int G>
__device__ __forceinline__ Lane<V> lane_of(const ScanArgs &s, int64_t tile)
{
    Lane<V> l;
    l.col = (tile * kWave + lane_id()) * V;
    l.in = l.col < s.columns;
    const int64_t q = l.in ? l.col : 0;   // (a lane without columns reads those of the first one and writes nothing)
    l.b = (int32_t)(q / s.dim);
    l.ch = (int32_t)(q - (int64_t)l.b * s.dim);
    l.len = s.lengths ? min(max(s.lengths[l.b], 0), (int32_t)s.n_steps) : (int32_t)s.n_steps;
    l.longest = l.len;
    if (s.lengths) {
#pragma unroll
        for (int m = kWave / 2; m > 0; m /= 2) l.longest = max(l.longest, __shfl_xor(l.longest, m));
    }
    l.longest = __builtin_amdgcn_readfirstlane(l.longest);
    l.gate = G == kShared ? l.ch / s.channels : l.ch;
    return l;
}

// What is left of a state behind several steps.  (Decays above 1 may have a product that 32 bits do not hold: it leaves nothing nothing.)
__device__ __forceinline__ float passed(float product, float state) { return state == 0.0f ? 0.0f : product * state; }

// A product of decays that 32 bits do not hold, though none of them is 0 (0.4 over 128 steps), is their smallest number: an infinite state stays infinite behind
// it, as it does step by step, and of any other there is 2^-149 left at most.
__device__ __forceinline__ float times(float p, float q)
{
    const float r = p * q;
    return r == 0.0f && p != 0.0f && q != 0.0f ? __builtin_copysignf(0x1p-149f, r) : r;
}
// The same of a block's decays, `p` being their plain product: looked at again only where that is 0
template <int V, typename Gate>
__device__ __forceinline__ void keep_products(float (&p)[V], const Gate &gate)
{
#pragma unroll
    for (int c = 0; c < V; ++c)
        if (p[c] == 0.0f) {
            p[c] = 1.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) p[c] = times(p[c], gate(k, c));
        }
}

// State that a stretch begins with: the stretches before it, in order.  sums[k][0]: product of the gates of stretch k, [1]: where it ends from zero.
template <int V>
__device__ __forceinline__ void fold(const float *sums, int64_t columns, const Lane<V> &l, int first, int last, int by, float (&h)[V])
{
    if (!l.in) return;
    for (int k = first; k != last; k += by) {
        float p[V], e[V];
        load_v<float, V>(sums + (int64_t)(2 * k) * columns + l.col, true, 0.0f, p);
        load_v<float, V>(sums + (int64_t)(2 * k + 1) * columns + l.col, true, 0.0f, e);
#pragma unroll
        for (int c = 0; c < V; ++c) h[c] = passed(p[c], h[c]) + e[c];
    }
}

// One pass over the steps of a stretch in rounds: each wavefront takes kSteps steps into registers, finds what they do to a state
// that enters them, (product of the gates, end from zero), the wavefronts tell each other, and each then computes its steps from the
// state that really enters.  Everything is read once, a round ahead.
// Short sequences are bound by the launches and by a round's way from load over exchange to store: 600 x 32 x 64 fp32 (4.9 MB each way) 8.3 us forward in
// two launches, 11.9 back in three.
template <int V, int kWaves>
struct Tell {
    float v[2][kWaves][2][V][kWave];   // [round in turn][wavefront][product, end]
};

// A round's exchange: `enter` is the state before the round and becomes the one behind it; returns in `mine` the one before the wavefront's block
template <int V, int kWaves>
__device__ __forceinline__ void exchange(Tell<V, kWaves> &tell, int turn, int wave, int waves, const float (&p)[V], const float (&e)[V], float (&enter)[V], float (&mine)[V])
{
    const int lane = lane_id();
#pragma unroll
    for (int c = 0; c < V; ++c) {
        tell.v[turn][wave][0][c][lane] = p[c];
        tell.v[turn][wave][1][c][lane] = e[c];
    }
    // (two sets of places in turn: whoever writes the one of a round has passed the barrier behind the round before)
    __syncthreads();
    for (int w = 0; w < waves; ++w) {
        if (w == wave)
#pragma unroll
            for (int c = 0; c < V; ++c) mine[c] = enter[c];
#pragma unroll
        for (int c = 0; c < V; ++c) enter[c] = passed(tell.v[turn][w][0][c][lane], enter[c]) + tell.v[turn][w][1][c][lane];
    }
}

// (kOne: a single round, of which none has to be read ahead: stretches of 128 steps, 600 x 32 x 64 fp32, 8.3 us
// against 9.3)
template <typename TX, typename TA, int V, int G, bool kOne>
__global__ void __launch_bounds__((kOne ? kRoundWaves : kMaxWaves) * kWave) scan_fwd_kernel(const ScanArgs s)
{
    constexpr int kWaves = kOne ? kRoundWaves : kMaxWaves;
    constexpr int VA = G == kEach ? V : 1;
    __shared__ Tell<V, kWaves> tell;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), waves = blockDim.x / kWave;
    const Lane<V> l = lane_of<V, G>(s, blockIdx.x);
    const int64_t t_lo = (int64_t)blockIdx.y * s.split_steps, t_hi = min(s.n_steps, t_lo + s.split_steps);
    const TX *x = static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch;
    const TA *a = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    TX *h = static_cast<TX *>(s.h) + l.col;
    float a_const[V];
    if (G == kConst) load_v<TA, V>(a, true, 0.0f, a_const);
    float enter[V];
#pragma unroll
    for (int c = 0; c < V; ++c) enter[c] = 0.0f;
    if (s.state && l.in) load_v<float, V>(s.state + l.col, true, 0.0f, enter);
    fold<V>(s.sums, s.columns, l, 0, blockIdx.y, 1, enter);

    const int64_t round_steps = (int64_t)waves * kSteps;
    Block<TX, V> xb[2];
    Block<TA, VA> ab[2];
    const int64_t last = max(min(t_hi, (int64_t)l.longest) - 1, (int64_t)0);
    auto load = [&](int i, int64_t t0) {
        xb[i].load(x, s.x_t, t0, last);
        if (G != kConst) ab[i].load(a, s.a_t, t0, last);
    };
    auto round = [&](int i, int64_t t0) {
        const int there = (int)min(max(min((int64_t)l.len, t_hi) - t0, (int64_t)0), (int64_t)kSteps);
        const bool all = __ballot(there < kSteps) == 0;
        if (!all) {
            xb[i].cut(there, 0.0f);
            if (G != kConst) ab[i].cut(there, 1.0f);
        }
        auto gate = [&](int k, int c) { return G == kConst ? (k < there ? a_const[c] : 1.0f) : ab[i].get(k, c); };
        float p[V], e[V], mine[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            p[c] = 1.0f, e[c] = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) e[c] = __builtin_fmaf(gate(k, c), e[c], xb[i].get(k, c)), p[c] *= gate(k, c);
        }
        keep_products<V>(p, gate);
        exchange(tell, i, wave, waves, p, e, enter, mine);
        if (t0 >= t_hi) return;
        xb[i].again();
        if (G != kConst) ab[i].again();
        if (s.marks && l.in) store_v<float, V>(s.marks + t0 / kSteps * s.columns + l.col, mine);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float out[V];
#pragma unroll
            for (int c = 0; c < V; ++c) {
                mine[c] = __builtin_fmaf(gate(k, c), mine[c], xb[i].get(k, c));
                out[c] = k < there ? mine[c] : 0.0f;
            }
            if (t0 + k < t_hi && l.in) store_v<TX, V>(h + (t0 + k) * s.columns, out);
        }
    };
    int64_t t0 = t_lo + wave * kSteps;
    load(0, t0);
    for (int64_t done = t_lo; done < t_hi; done += 2 * round_steps, t0 += 2 * round_steps) {
        if (!kOne) load(1, t0 + round_steps);
        round(0, t0);
        if (kOne || done + round_steps >= t_hi) break;
        load(0, t0 + 2 * round_steps);
        round(1, t0 + round_steps);
    }
    if (wave == 0 && blockIdx.y == gridDim.y - 1 && l.in) store_v<float, V>(s.last + l.col, enter);
}

// Sum over `lanes` neighbouring lanes (a power of two, the same for all), in each of them.  Moves within the vector unit: a sum over 32 lanes by
// moves through LDS (__shfl_xor) takes 35 of a backward pass's 130 us (4,096 x 8 x 2,048, a gate per 64 channels).
template <int kCtrl>
__device__ __forceinline__ float plus_moved(float v)
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, true));
}
__device__ __forceinline__ float sum_lanes(float v, int lanes)
{
    if (lanes > 1) v = plus_moved<0xB1>(v);    // neighbours of two: quad_perm 1, 0, 3, 2
    if (lanes > 2) v = plus_moved<0x4E>(v);    // pairs of four: quad_perm 2, 3, 0, 1
    if (lanes > 4) v = plus_moved<0x141>(v);   // fours of eight (each holds one value): row_half_mirror
    if (lanes > 8) v = plus_moved<0x140>(v);   // eights of sixteen: row_mirror
    if (lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (lanes > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// The last part of a block on the way back, from the gradient `mine` that enters behind its last step
template <typename TX, typename TA, int V, int G, int VA>
__device__ __forceinline__ void backward_block(const ScanArgs &s, const Lane<V> &l, const Block<TX, V> &gb, const Block<TA, VA> &ab, const float (&a_const)[V],
                                               const float (&before)[kSteps][V], int there, int64_t t0, int64_t t_hi, float (&mine)[V], float (&d_const)[V])
{
    const int lane = lane_id();
    TX *dx = static_cast<TX *>(s.dx) + l.col;
    TA *da = static_cast<TA *>(s.da);
#pragma unroll
    for (int k = kSteps - 1; k >= 0; --k) {
        const int64_t t = t0 + k;
        float g[V], d[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const float all = gb.get(k, c) + mine[c];
            g[c] = k < there ? all : 0.0f;   // (behind a sequence's end the gradient of its last state passes through)
            d[c] = k < there ? all * before[k][c] : 0.0f;
            mine[c] = (G == kConst ? (k < there ? a_const[c] : 1.0f) : ab.get(k, c)) * all;
            if (G == kConst) d_const[c] += d[c];
        }
        const bool write = t < t_hi && l.in;
        if (write) store_v<TX, V>(dx + t * s.columns, g);
        if (G == kEach && write) store_v<TA, V>(da + t * s.columns + l.col, d);
        if (G == kShared) {
            const float sum = sum_lanes(V == 2 ? d[0] + d[V - 1] : d[0], s.seg_lanes);
            if (write && (lane & (s.seg_lanes - 1)) == 0) {
                // a gate's channels within the lanes: its gradient; else parts of it, to be joined
                const int64_t at = (t * s.sequences + l.b) * s.parts;
                if (s.da_part) s.da_part[at + l.ch / (V * s.seg_lanes)] = sum;
                else da[at + l.gate] = (TA)sum;
            }
        }
    }
}

// On the way back the state is c[t] = a[t] (dh[t] + c[t + 1]), what a gradient that enters behind step t becomes before it.
template <typename TX, typename TA, int V, int G>
__global__ void __launch_bounds__(kRoundWaves * kWave) scan_bwd_kernel(const ScanArgs s)
{
    constexpr int VA = G == kEach ? V : 1;
    __shared__ Tell<V, kRoundWaves> tell;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), waves = blockDim.x / kWave;
    const Lane<V> l = lane_of<V, G>(s, blockIdx.x);
    const int64_t t_lo = (int64_t)blockIdx.y * s.split_steps, t_hi = min(s.n_steps, t_lo + s.split_steps);
    const TX *x = static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch;
    const TA *a = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    const TX *dh = static_cast<const TX *>(s.dh) + (int64_t)l.b * s.dh_b + l.ch;
    float a_const[V], d_const[V];
    if (G == kConst) load_v<TA, V>(a, true, 0.0f, a_const);
    float enter[V];
#pragma unroll
    for (int c = 0; c < V; ++c) enter[c] = d_const[c] = 0.0f;
    if (s.d_last && l.in) load_v<float, V>(s.d_last + l.col, true, 0.0f, enter);
    fold<V>(s.sums, s.columns, l, gridDim.y - 1, blockIdx.y, -1, enter);

    const int64_t round_steps = (int64_t)waves * kSteps;
    const int64_t rounds = (t_hi - t_lo + round_steps - 1) / round_steps, last = max(min(t_hi, (int64_t)l.longest) - 1, (int64_t)0);
    Block<TX, V> xb, gb;
    Block<TA, VA> ab;
    float before[kSteps][V];
    for (int64_t round = 0; round < rounds; ++round) {
        // the last block first
        const int64_t t0 = t_lo + (rounds * waves - 1 - (round * waves + wave)) * kSteps;
        gb.load(dh, s.dh_t, t0, last);
        if (G != kConst) ab.load(a, s.a_t, t0, last);
        xb.load(x, s.x_t, t0, last);
        // (columns that are not there: as behind their end)
        const int there = l.in ? (int)min(max(min((int64_t)l.len, t_hi) - t0, (int64_t)0), (int64_t)kSteps) : 0;
        if (__ballot(there < kSteps) != 0) {
            gb.cut(there, 0.0f);
            xb.cut(there, 0.0f);
            if (G != kConst) ab.cut(there, 1.0f);
        }
        auto gate = [&](int k, int c) { return G == kConst ? (k < there ? a_const[c] : 1.0f) : ab.get(k, c); };
        if (l.in && t0 < t_hi) load_v<float, V>(s.marks + t0 / kSteps * s.columns + l.col, true, 0.0f, before[0]);
        else
#pragma unroll
            for (int c = 0; c < V; ++c) before[0][c] = 0.0f;
        float p[V], e[V], mine[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            p[c] = 1.0f, e[c] = 0.0f;
#pragma unroll
            for (int k = kSteps - 1; k >= 0; --k) e[c] = gate(k, c) * (gb.get(k, c) + e[c]), p[c] *= gate(k, c);
        }
        keep_products<V>(p, gate);
        // the states before each step, again from the kept one
#pragma unroll
        for (int k = 1; k < kSteps; ++k)
#pragma unroll
            for (int c = 0; c < V; ++c) before[k][c] = __builtin_fmaf(gate(k - 1, c), before[k - 1][c], xb.get(k - 1, c));
        exchange(tell, (int)(round & 1), wave, waves, p, e, enter, mine);
        gb.again();
        if (G != kConst) ab.again();
        if (t0 < t_hi) backward_block<TX, TA, V, G>(s, l, gb, ab, a_const, before, there, t0, t_hi, mine, d_const);
    }
    if (l.in && wave == 0 && blockIdx.y == 0 && s.d_state) store_v<float, V>(s.d_state + l.col, enter);
    if (G == kConst) {
        // the wavefronts' sums together, in order
        __syncthreads();
#pragma unroll
        for (int c = 0; c < V; ++c) tell.v[0][wave][0][c][lane] = d_const[c];
        __syncthreads();
        if (wave != 0 || !l.in) return;
        for (int w = 1; w < waves; ++w)
#pragma unroll
            for (int c = 0; c < V; ++c) d_const[c] += tell.v[0][w][0][c][lane];
        store_v<float, V>(s.da_part + (int64_t)blockIdx.y * s.columns + l.col, d_const);
    }
}

// What a whole stretch does, for the stretches that are computed from it: the product of its gates and its end from zero, forwards or backwards.  Each
// wavefront takes every waves-th block, from the stretch's other end to where the pass proper begins, so that what that pass reads first was
// read last; the wavefronts' blocks of a round are joined as they come, in the order of time.
template <typename TX, typename TA, int V, int G, bool kBack, bool kOne>
__global__ void __launch_bounds__(kMaxWaves * kWave) scan_sums_kernel(const ScanArgs s)
{
    constexpr int VA = G == kEach ? V : 1;
    __shared__ Tell<V, kMaxWaves> tell;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), waves = blockDim.x / kWave;
    const Lane<V> l = lane_of<V, G>(s, blockIdx.x);
    // (stretch blockIdx.y, on the way back + 1: what the last one to be passed does, nobody asks)
    const int stretch = blockIdx.y + (kBack ? 1 : 0);
    const int64_t t_lo = (int64_t)stretch * s.split_steps, t_hi = min(s.n_steps, t_lo + s.split_steps);
    const TX *x = kBack ? static_cast<const TX *>(s.dh) + (int64_t)l.b * s.dh_b + l.ch : static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch;
    const int64_t x_t = kBack ? s.dh_t : s.x_t;
    const TA *a = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    float a_const[V];
    if (G == kConst) load_v<TA, V>(a, true, 0.0f, a_const);
    const int64_t round_steps = (int64_t)waves * kSteps;
    const int64_t rounds = (t_hi - t_lo + round_steps - 1) / round_steps;
    const int64_t last = max(min(t_hi, (int64_t)l.longest) - 1, (int64_t)0);
    float product[V], end[V];
#pragma unroll
    for (int c = 0; c < V; ++c) product[c] = 1.0f, end[c] = 0.0f;
    Block<TX, V> xb[2];
    Block<TA, VA> ab[2];
    auto block_of = [&](int64_t round) { return t_lo + (kBack ? round : rounds - 1 - round) * round_steps + wave * kSteps; };
    auto load = [&](int i, int64_t round) {
        const int64_t t0 = block_of(round < rounds ? round : rounds - 1);
        xb[i].load(x, x_t, t0, last);
        if (G != kConst) ab[i].load(a, s.a_t, t0, last);
    };
    auto take = [&](int i, int64_t round) {
        const int64_t t0 = block_of(round);
        const int there = (int)min(max(min((int64_t)l.len, t_hi) - t0, (int64_t)0), (int64_t)kSteps);
        if (__ballot(there < kSteps) != 0) {
            xb[i].cut(there, 0.0f);
            if (G != kConst) ab[i].cut(there, 1.0f);
        }
        auto gate = [&](int k, int c) { return G == kConst ? (k < there ? a_const[c] : 1.0f) : ab[i].get(k, c); };
        float p[V], e[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            p[c] = 1.0f, e[c] = 0.0f;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int k = kBack ? kSteps - 1 - j : j;
                e[c] = kBack ? gate(k, c) * (xb[i].get(k, c) + e[c]) : __builtin_fmaf(gate(k, c), e[c], xb[i].get(k, c));
                p[c] *= gate(k, c);
            }
        }
        keep_products<V>(p, gate);
#pragma unroll
        for (int c = 0; c < V; ++c) {
            tell.v[i][wave][0][c][lane] = p[c];
            tell.v[i][wave][1][c][lane] = e[c];
        }
        __syncthreads();
        if (wave != 0) return;
        // the round's blocks, then what was found before, which the state passes afterwards
        float rp[V], re[V];
#pragma unroll
        for (int c = 0; c < V; ++c) rp[c] = 1.0f, re[c] = 0.0f;
        for (int j = 0; j < waves; ++j) {
            const int w = kBack ? waves - 1 - j : j;
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const float pw = tell.v[i][w][0][c][lane];
                re[c] = passed(pw, re[c]) + tell.v[i][w][1][c][lane];
                rp[c] = times(rp[c], pw);
            }
        }
#pragma unroll
        for (int c = 0; c < V; ++c) {
            end[c] = passed(product[c], re[c]) + end[c];
            product[c] = times(product[c], rp[c]);
        }
    };
    load(0, 0);
    for (int64_t round = 0; round < rounds; round += 2) {
        if (!kOne) load(1, round + 1);
        take(0, round);
        if (kOne || round + 1 >= rounds) break;
        load(0, round + 2);
        take(1, round + 1);
    }
    if (wave == 0 && l.in) {
        store_v<float, V>(s.sums + (int64_t)(2 * stretch) * s.columns + l.col, product);
        store_v<float, V>(s.sums + (int64_t)(2 * stretch + 1) * s.columns + l.col, end);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long sequences of few columns in one pass over the data.  A workgroup holds a stretch, one block a wavefront, in registers, and tells
// what it does to a state (product, end from zero) as soon as it knows; what enters it follows from the stretches of its group of kGroup before it and from
// the state that entered the group, which the last workgroup of the group before tells.  So every sum is made in an order that is
// fixed, and the way from one group to the next is all that happens one after the other.
//
// 65,536 x 1,000 bf16, a gate per channel: 114 us forward (393 MB, 3.5 TB/s; two passes 156).  4,096 x 8 x 2,048 bf16, a gate per 64 channels, ragged: 71 us
// forward and 113 back.  Three workgroups on a compute unit in the place of two change nothing: what is left is memory that is read and written by turns.
//
// Workgroups take their stretches by a counter, in the order in which the state passes: what one waits for comes from workgroups that have begun before
// it and wait for earlier ones only, so every wait ends, however few run at once.  Values are told as 64 bits at a time, all ones being none yet.
constexpr int kChainWaves = 8, kGroup = 16, kChainLeast = 20, kChainFew = 8;
constexpr uint64_t kNone = ~0ull;

struct Chain {
    uint64_t *stretch;   // [stretches][columns]: product and end
    uint64_t *group;     // [groups + 1][columns]: the state that enters
    uint32_t *counter;
    int64_t tiles, stretches;
};

constexpr int kClear = 4;   // values of a thread
__global__ void __launch_bounds__(kBlock) chain_clear_kernel(uint64_t *p, int64_t n, uint32_t *counter)
{
    const int64_t first = (int64_t)blockIdx.x * kBlock * kClear + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kClear; ++k)
        if (first + k * kBlock < n) p[first + k * kBlock] = kNone;
    if (first == 0) *counter = 0;
}

template <int V>
__device__ __forceinline__ void say(uint64_t *p, const float (&hi)[V], const float (&lo)[V])
{
#pragma unroll
    for (int c = 0; c < V; ++c) {
        // (a NaN of all ones in both would be taken for none)
        const uint32_t h = hi[c] != hi[c] ? 0x7fc00000u : __float_as_uint(hi[c]);
        __hip_atomic_store(p + c, ((uint64_t)h << 32) | __float_as_uint(lo[c]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
// K values as they are told; the loop's bound is never met (see above), and would show as NaN
template <int V, int K>
__device__ __forceinline__ void hear(const uint64_t *const (&p)[K], const bool (&asked)[K], uint64_t (&v)[K][V])
{
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < V; ++c) v[k][c] = 0;
    for (int tries = 0; tries < (1 << 22); ++tries) {
        bool some = false;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (asked[k])
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    v[k][c] = __hip_atomic_load(p[k] + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    some = some || v[k][c] == kNone;
                }
        if (__ballot(some) == 0) return;
        __builtin_amdgcn_s_sleep(2);
    }
}

// What a stretch's wavefronts know of one another
template <int V>
struct ChainShared {
    float block[kChainWaves][2][V][kWave];    // of the stretch: product, end
    float before[kChainWaves][2][V][kWave];   // of the stretches before it in its group, a part of them each
    float group[V][kWave];                    // the state that entered the group
    uint32_t ticket;
};

// The state that enters this wavefront's block: `mine`.  order: how many stretches come before.  `given`: what enters the first one.  Whoever is last of all
// leaves the end state in `last`.
template <int V>
__device__ __forceinline__ void chain(ChainShared<V> &sh, const Chain &ch, const Lane<V> &l, int64_t columns, int64_t order, int wave, const float (&p)[V],
                                      const float (&e)[V], const float *given, float *last, float (&mine)[V])
{
    const int lane = lane_id();
#pragma unroll
    for (int c = 0; c < V; ++c) sh.block[wave][0][c][lane] = p[c], sh.block[wave][1][c][lane] = e[c];
    __syncthreads();
    // the blocks before this one, and the whole stretch
    float pp[V], pe[V], wp[V], we[V];
    auto join = [&](auto product_of) {
#pragma unroll
        for (int c = 0; c < V; ++c) wp[c] = 1.0f, we[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < kChainWaves; ++w) {
            if (w == wave)
#pragma unroll
                for (int c = 0; c < V; ++c) pp[c] = wp[c], pe[c] = we[c];
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const float bp = sh.block[w][0][c][lane];
                we[c] = passed(bp, we[c]) + sh.block[w][1][c][lane];
                wp[c] = product_of(wp[c], bp);
            }
        }
    };
    // (every stretch waits for this: products are looked at one by one only where they come out as 0, 4,096 x 8 x 2,048 bf16 75 us against 81)
    join([](float p, float q) { return p * q; });
    bool none = false;
#pragma unroll
    for (int c = 0; c < V; ++c) none = none || wp[c] == 0.0f;
    if (__ballot(none) != 0) join([](float p, float q) { return times(p, q); });
    if (wave == 0 && l.in) say<V>(ch.stretch + order * columns + l.col, wp, we);
    // a part of the group's stretches before
    constexpr int kPart = kGroup / kChainWaves;
    const int64_t group = order / kGroup, first = group * kGroup + wave * kPart;
    {
        const uint64_t *from[kPart];
        bool asked[kPart];
        uint64_t v[kPart][V];
#pragma unroll
        for (int k = 0; k < kPart; ++k) {
            asked[k] = l.in && first + k < order;
            from[k] = ch.stretch + (asked[k] ? (first + k) * columns + l.col : 0);
        }
        hear<V, kPart>(from, asked, v);
        float fp[V], fe[V];
#pragma unroll
        for (int c = 0; c < V; ++c) fp[c] = 1.0f, fe[c] = 0.0f;
#pragma unroll
        for (int k = 0; k < kPart; ++k)
            if (asked[k])
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    const float sp = __uint_as_float((uint32_t)(v[k][c] >> 32));
                    fe[c] = passed(sp, fe[c]) + __uint_as_float((uint32_t)v[k][c]);
                    fp[c] = times(fp[c], sp);
                }
#pragma unroll
        for (int c = 0; c < V; ++c) sh.before[wave][0][c][lane] = fp[c], sh.before[wave][1][c][lane] = fe[c];
    }
    if (wave == kChainWaves - 1) {
        float h[V];
#pragma unroll
        for (int c = 0; c < V; ++c) h[c] = 0.0f;
        if (group == 0) {
            if (given && l.in) load_v<float, V>(given + l.col, true, 0.0f, h);
        } else {
            const uint64_t *from[1] = {ch.group + (l.in ? group * columns + l.col : 0)};
            const bool asked[1] = {l.in};
            uint64_t v[1][V];
            hear<V, 1>(from, asked, v);
#pragma unroll
            for (int c = 0; c < V; ++c) h[c] = __uint_as_float((uint32_t)v[0][c]);
        }
#pragma unroll
        for (int c = 0; c < V; ++c) sh.group[c][lane] = h[c];
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
        h[c] = sh.group[c][lane];
#pragma unroll
        for (int w = 0; w < kChainWaves; ++w) h[c] = passed(sh.before[w][0][c][lane], h[c]) + sh.before[w][1][c][lane];
        mine[c] = passed(pp[c], h[c]) + pe[c];
    }
    const bool ends = order == ch.stretches - 1;
    if (wave == 0 && l.in && (ends || order % kGroup == kGroup - 1)) {
        float out[V], zero[V];
#pragma unroll
        for (int c = 0; c < V; ++c) out[c] = passed(wp[c], h[c]) + we[c], zero[c] = 0.0f;
        if (!ends) say<V>(ch.group + (group + 1) * columns + l.col, zero, out);
        else if (last) store_v<float, V>(last + l.col, out);
    }
}

template <typename TX, typename TA, int V, int G>
__global__ void __launch_bounds__(kChainWaves * kWave, 4) scan_fwd_chain_kernel(const ScanArgs s, const Chain ch)
{
    constexpr int VA = G == kEach ? V : 1;
    __shared__ ChainShared<V> sh;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    if (threadIdx.x == 0) sh.ticket = __hip_atomic_fetch_add(ch.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int64_t ticket = __builtin_amdgcn_readfirstlane((int)sh.ticket), order = ticket / ch.tiles;
    const Lane<V> l = lane_of<V, G>(s, ticket - order * ch.tiles);
    const int64_t t0 = (order * kChainWaves + wave) * kSteps, t_hi = s.n_steps;
    const TA *a = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    Block<TX, V> xb;
    Block<TA, VA> ab;
    const int64_t last = max(min(t_hi, (int64_t)l.longest) - 1, (int64_t)0);
    xb.load(static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch, s.x_t, t0, last);
    if (G != kConst) ab.load(a, s.a_t, t0, last);
    float a_const[V];
    if (G == kConst) load_v<TA, V>(a, true, 0.0f, a_const);
    const int there = (int)min(max(min((int64_t)l.len, t_hi) - t0, (int64_t)0), (int64_t)kSteps);
    if (__ballot(there < kSteps) != 0) {
        xb.cut(there, 0.0f);
        if (G != kConst) ab.cut(there, 1.0f);
    }
    auto gate = [&](int k, int c) { return G == kConst ? (k < there ? a_const[c] : 1.0f) : ab.get(k, c); };
    float p[V], e[V], mine[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
        p[c] = 1.0f, e[c] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) e[c] = __builtin_fmaf(gate(k, c), e[c], xb.get(k, c)), p[c] *= gate(k, c);
    }
    keep_products<V>(p, gate);
    chain<V>(sh, ch, l, s.columns, order, wave, p, e, s.state, s.last, mine);
    if (t0 >= t_hi || !l.in) return;
    xb.again();
    if (G != kConst) ab.again();
    if (s.marks) store_v<float, V>(s.marks + t0 / kSteps * s.columns + l.col, mine);
    TX *h = static_cast<TX *>(s.h) + l.col;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        float out[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            mine[c] = __builtin_fmaf(gate(k, c), mine[c], xb.get(k, c));
            out[c] = k < there ? mine[c] : 0.0f;
        }
        if (t0 + k < t_hi) store_v<TX, V>(h + (t0 + k) * s.columns, out);
    }
}

template <typename TX, typename TA, int V, int G>
__global__ void __launch_bounds__(kChainWaves * kWave, 4) scan_bwd_chain_kernel(const ScanArgs s, const Chain ch)
{
    constexpr int VA = G == kEach ? V : 1;
    __shared__ ChainShared<V> sh;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    if (threadIdx.x == 0) sh.ticket = __hip_atomic_fetch_add(ch.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int64_t ticket = __builtin_amdgcn_readfirstlane((int)sh.ticket), order = ticket / ch.tiles;
    const Lane<V> l = lane_of<V, G>(s, ticket - order * ch.tiles);
    // from the last block on
    const int64_t stretch = ch.stretches - 1 - order, t0 = (stretch * kChainWaves + kChainWaves - 1 - wave) * kSteps, t_hi = s.n_steps;
    const TA *a = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    Block<TX, V> xb, gb;
    Block<TA, VA> ab;
    const int64_t last = max(min(t_hi, (int64_t)l.longest) - 1, (int64_t)0);
    gb.load(static_cast<const TX *>(s.dh) + (int64_t)l.b * s.dh_b + l.ch, s.dh_t, t0, last);
    if (G != kConst) ab.load(a, s.a_t, t0, last);
    xb.load(static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch, s.x_t, t0, last);
    float a_const[V], d_const[V];
    if (G == kConst) load_v<TA, V>(a, true, 0.0f, a_const);
    const int there = l.in ? (int)min(max(min((int64_t)l.len, t_hi) - t0, (int64_t)0), (int64_t)kSteps) : 0;
    if (__ballot(there < kSteps) != 0) {
        gb.cut(there, 0.0f);
        xb.cut(there, 0.0f);
        if (G != kConst) ab.cut(there, 1.0f);
    }
    auto gate = [&](int k, int c) { return G == kConst ? (k < there ? a_const[c] : 1.0f) : ab.get(k, c); };
    float p[V], e[V], mine[V], before[kSteps][V];
    if (l.in && t0 < t_hi) load_v<float, V>(s.marks + t0 / kSteps * s.columns + l.col, true, 0.0f, before[0]);
    else
#pragma unroll
        for (int c = 0; c < V; ++c) before[0][c] = 0.0f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        d_const[c] = 0.0f;
        p[c] = 1.0f, e[c] = 0.0f;
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k) e[c] = gate(k, c) * (gb.get(k, c) + e[c]), p[c] *= gate(k, c);
    }
    keep_products<V>(p, gate);
    chain<V>(sh, ch, l, s.columns, order, wave, p, e, s.d_last, s.d_state, mine);
    gb.again();
    if (G != kConst) ab.again();
    // the states before each step, again from the kept one
#pragma unroll
    for (int k = 1; k < kSteps; ++k)
#pragma unroll
        for (int c = 0; c < V; ++c) before[k][c] = __builtin_fmaf(gate(k - 1, c), before[k - 1][c], xb.get(k - 1, c));
    if (t0 < t_hi) backward_block<TX, TA, V, G>(s, l, gb, ab, a_const, before, there, t0, t_hi, mine, d_const);
    if (G == kConst) {
        // the wavefronts' sums together, in order
        __syncthreads();
#pragma unroll
        for (int c = 0; c < V; ++c) sh.block[wave][0][c][lane] = d_const[c];
        __syncthreads();
        if (wave != 0 || !l.in) return;
        for (int w = 1; w < kChainWaves; ++w)
#pragma unroll
            for (int c = 0; c < V; ++c) d_const[c] += sh.block[w][0][c][lane];
        store_v<float, V>(s.da_part + order * s.columns + l.col, d_const);
    }
}

// One step: nothing to join
template <typename TX, typename TA, int V, int G>
__global__ void __launch_bounds__(kBlock) scan_one_kernel(const ScanArgs s)
{
    Lane<V> l;
    l.col = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * V;
    if (l.col >= s.columns) return;
    l.b = (int32_t)(l.col / s.dim);
    l.ch = (int32_t)(l.col - (int64_t)l.b * s.dim);
    l.gate = G == kShared ? l.ch / s.channels : l.ch;
    const bool there = !s.lengths || s.lengths[l.b] > 0;
    float x[V], a[V], h[V], out[V];
    load_v<TX, V>(static_cast<const TX *>(s.x) + (int64_t)l.b * s.x_b + l.ch, there, 0.0f, x);
    const TA *gate = static_cast<const TA *>(s.a) + (G == kConst ? 0 : (int64_t)l.b * s.a_b) + l.gate;
    if (G == kShared) {
        float one[1];
        load_v<TA, 1>(gate, there, 1.0f, one);
#pragma unroll
        for (int c = 0; c < V; ++c) a[c] = one[0];
    } else {
        load_v<TA, V>(gate, there, 1.0f, a);
    }
    load_v<float, V>(s.state + l.col, s.state != nullptr, 0.0f, h);
    if (s.marks) store_v<float, V>(s.marks + l.col, h);
#pragma unroll
    for (int c = 0; c < V; ++c) {
        h[c] = __builtin_fmaf(a[c], h[c], x[c]);
        out[c] = there ? h[c] : 0.0f;
    }
    store_v<TX, V>(static_cast<TX *>(s.h) + l.col, out);
    store_v<float, V>(s.last + l.col, h);
}

// Gradient of one decay per channel: its parts by stretch and sequence, every sixteenth by one wavefront, in order
constexpr int kJoinWaves = 16;
template <typename TA>
__global__ void __launch_bounds__(kJoinWaves * kWave) scan_join_const_kernel(const float *__restrict__ part, int64_t parts, int dim, TA *__restrict__ da)
{
    __shared__ float sum[kJoinWaves][kWave];
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    const int ch = blockIdx.x * kWave + lane;
    const float *p = part + (ch < dim ? ch : 0);
    float v = 0.0f;
    int64_t k = wave;
    for (; k + 3 * kJoinWaves < parts; k += 4 * kJoinWaves) {
        float w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = p[(k + u * kJoinWaves) * dim];
        v += (w[0] + w[1]) + (w[2] + w[3]);
    }
    for (; k < parts; k += kJoinWaves) v += p[k * dim];
    sum[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && ch < dim) {
        for (int w = 1; w < kJoinWaves; ++w) v += sum[w][lane];
        da[ch] = (TA)v;
    }
}

// Gradient of a shared gate: n_part parts next to one another
template <typename TA>
__global__ void __launch_bounds__(kBlock) scan_join_shared_kernel(const float *__restrict__ part, int64_t gates, int n_part, TA *__restrict__ da)
{
    const int64_t g = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (g >= gates) return;
    float v = 0.0f;
    for (int k = 0; k < n_part; ++k) v += part[g * n_part + k];
    da[g] = (TA)v;
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kFillBlocks = 512;   // workgroups that fill the chip
// How a call is laid out.  A lane takes two channels of a 16-bit type where rows and strides allow it (four bytes a lane and load).
struct Plan {
    int v, waves, seg_lanes, parts;
    int64_t tiles, splits, split_steps;
    int64_t chained;   // stretches of a chain; 0: two passes where there are stretches
    bool one_round() const { return split_steps <= (int64_t)waves * kSteps; }   // of a stretch
    int64_t parts_const() const { return chained ? chained : splits; }
    int64_t sums_floats(int64_t columns) const
    {
        return chained ? 2 * (columns * (chained + chained / kGroup + 1) + 1) : splits > 1 ? 2 * splits * columns : 0;
    }
};

Plan plan_of(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t dtype, bool pairs)
{
    Plan p;
    const int channels = groups > 0 ? dim / groups : 1;
    p.v = dtype != BMTK_F32 && dim % 2 == 0 && pairs && (groups == 0 || groups == dim || channels % 2 == 0) ? 2 : 1;
    p.tiles = div_up(batch * dim, kWave * p.v);
    int64_t w = div_up(n_steps, kSteps);
    p.waves = (int)(w < kMaxWaves ? w : kMaxWaves);
    // stretches of time, of whole rounds: as many as fill the chip
    const int64_t round = (int64_t)p.waves * kSteps;
    int64_t s = kFillBlocks / p.tiles, most = div_up(n_steps, round);
    if (s > most) s = most;
    if (s > 64) s = 64;
    if (s < 1) s = 1;
    p.split_steps = div_up(div_up(n_steps, s), round) * round;
    p.splits = div_up(n_steps, p.split_steps);
    // A chain reads everything once, and has its clearing and its waits: for many stretches, or few columns.  Chain / two passes, us, forward and back:
    // 300 x 12 x 17 fp32 7.0 / 7.7, 9.9 / 10.7; 700 x 4 x 64 bf16 8.4 / 9.3, 9.7 / 11.1; 700 x 32 x 64 fp32 9.6 / 8.4, 13.7 / 12.0;
    // 2,000 x 32 x 64 fp32 18.1 / 16.3, 20.4 / 19.8; 4,096 x 256 bf16 10.5 / 16.9 and 65,536 x 1,000 bf16 112 / 156 forward
    p.chained = div_up(n_steps, kChainWaves * kSteps);
    if (p.splits > 1 && (p.chained >= kChainLeast || (w > kRoundWaves && p.tiles <= kChainFew)) && p.tiles * p.chained < (1 << 22)) p.splits = 1;
    else p.chained = 0;
    // One round of more wavefronts in the place of stretches: 150 x 32 x 64 fp32 4.9 / 8.3 us forward, 7.8 / 10.7 back; two such rounds would take 10.1 / 8.0
    // and 13.4 / 11.2 (500 x 32 x 64)
    if (p.splits > 1 && w <= kRoundWaves) p.splits = 1, p.waves = (int)w, p.split_steps = w * kSteps;
    // A shared gate's gradient is summed over neighbouring lanes, a power of two of them that divides the gate's channels; what that leaves is written as
    // partial sums, 4 bytes each, and joined.  Gates of 32, 64 and 128 channels leave one sum or few; an odd number of channels one for every channel and step:
    // 4,096 x 8 x 2,046 bf16, gates of 33, back 1,340 us and 268 MB of workspace; 2,000 channels in gates of 100 238 us; 2,048 in gates of 32 or 64 117 us.
    p.seg_lanes = p.parts = 0;
    if (groups > 0 && groups != dim) {
        const int seg = gcd(channels, kWave * p.v);
        p.seg_lanes = seg / p.v;   // (two channels a lane only where a gate has an even number of them)
        p.parts = dim / seg;
    }
    return p;
}

int check_scan(const char *who, int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t dtype, int32_t gate_dtype)
{
    BMTK_REQUIRE(n_steps > 0 && batch > 0 && dim > 0 && groups >= 0, "%s: sizes must be positive", who);
    BMTK_REQUIRE(groups == 0 || dim % groups == 0, "%s: %d gates do not share %d channels evenly", who, groups, dim);
    BMTK_REQUIRE(dtype == BMTK_F32 || dtype == BMTK_BF16 || dtype == BMTK_F16, "%s: unknown type %d", who, dtype);
    BMTK_REQUIRE(gate_dtype == BMTK_F32 || gate_dtype == dtype, "%s: decays are in 32 bits or of the input's type", who);
    BMTK_REQUIRE(n_steps < (1ll << 31) - 4096 && batch < (1ll << 31) && batch * (int64_t)dim < (1ll << 31), "%s: too many steps or columns", who);
    return BMTK_OK;
}

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_gated_scan_workspace_bytes(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t backward)
{
    if (check_scan("gated_scan_workspace_bytes", n_steps, batch, dim, groups, BMTK_F32, BMTK_F32) != BMTK_OK) return 0;
    int64_t most = 0;
    for (int pairs = 0; pairs < 2; ++pairs) {
        const Plan p = plan_of(n_steps, batch, dim, groups, BMTK_BF16, pairs != 0);
        int64_t floats = p.sums_floats(batch * dim);
        if (backward && groups == 0) floats += p.parts_const() * batch * dim;
        if (backward && groups > 0 && groups != dim && p.parts != groups) floats += n_steps * batch * p.parts;
        most = floats > most ? floats : most;
    }
    return most * (int64_t)sizeof(float);
}

#define BMTK_SCAN_LAUNCH(KERNEL, ...)                                                                                                         \
    do {                                                                                                                                      \
        if (groups == 0) hipLaunchKernelGGL((KERNEL<TX, TA, V, kConst __VA_ARGS__>), grid, dim3(p.waves *kWave), 0, st, s);                    \
        else if (groups == dim) hipLaunchKernelGGL((KERNEL<TX, TA, V, kEach __VA_ARGS__>), grid, dim3(p.waves *kWave), 0, st, s);              \
        else hipLaunchKernelGGL((KERNEL<TX, TA, V, kShared __VA_ARGS__>), grid, dim3(p.waves *kWave), 0, st, s);                               \
    } while (0)
#define BMTK_COMMA ,
#define BMTK_CHAIN_LAUNCH(KERNEL)                                                                                             \
    do {                                                                                                                      \
        const dim3 grid((unsigned)(p.tiles * p.chained)), block(kChainWaves *kWave);                                          \
        if (groups == 0) hipLaunchKernelGGL((KERNEL<TX, TA, V, kConst>), grid, block, 0, st, s, ch);                          \
        else if (groups == dim) hipLaunchKernelGGL((KERNEL<TX, TA, V, kEach>), grid, block, 0, st, s, ch);                    \
        else hipLaunchKernelGGL((KERNEL<TX, TA, V, kShared>), grid, block, 0, st, s, ch);                                     \
    } while (0)

namespace {

// (`sums` is the chain's: its values, and the counter behind them)
Chain chain_of(const ScanArgs &s, const Plan &p, hipStream_t st)
{
    Chain ch;
    ch.tiles = p.tiles, ch.stretches = p.chained;
    ch.stretch = reinterpret_cast<uint64_t *>(s.sums);
    ch.group = ch.stretch + p.chained * s.columns;
    const int64_t values = (p.chained + p.chained / kGroup + 1) * s.columns;
    ch.counter = reinterpret_cast<uint32_t *>(ch.stretch + values);
    hipLaunchKernelGGL(chain_clear_kernel, dim3((unsigned)div_up(values, kBlock * kClear)), dim3(kBlock), 0, st, ch.stretch, values, ch.counter);
    return ch;
}

template <typename TX, typename TA, int V>
void launch_fwd(const ScanArgs &s, const Plan &p, int groups, hipStream_t st)
{
    const int dim = s.dim;
    if (s.n_steps == 1) {
        const dim3 one((unsigned)div_up(s.columns, kBlock * V));
        if (groups == 0) hipLaunchKernelGGL((scan_one_kernel<TX, TA, V, kConst>), one, dim3(kBlock), 0, st, s);
        else if (groups == dim) hipLaunchKernelGGL((scan_one_kernel<TX, TA, V, kEach>), one, dim3(kBlock), 0, st, s);
        else hipLaunchKernelGGL((scan_one_kernel<TX, TA, V, kShared>), one, dim3(kBlock), 0, st, s);
        return;
    }
    if (p.chained) {
        const Chain ch = chain_of(s, p, st);
        BMTK_CHAIN_LAUNCH(scan_fwd_chain_kernel);
        return;
    }
    dim3 grid((unsigned)p.tiles, (unsigned)p.splits);
    if (p.splits > 1) {
        grid.y = (unsigned)p.splits - 1;
        if (p.one_round()) BMTK_SCAN_LAUNCH(scan_sums_kernel, BMTK_COMMA false BMTK_COMMA true);
        else BMTK_SCAN_LAUNCH(scan_sums_kernel, BMTK_COMMA false BMTK_COMMA false);
        grid.y = (unsigned)p.splits;
    }
    if (p.one_round()) BMTK_SCAN_LAUNCH(scan_fwd_kernel, BMTK_COMMA true);
    else BMTK_SCAN_LAUNCH(scan_fwd_kernel, BMTK_COMMA false);
}

template <typename TX, typename TA, int V>
void launch_bwd(ScanArgs s, const Plan &p, int groups, hipStream_t st)
{
    const int dim = s.dim;
    const int64_t batch = s.columns / dim;
    if (p.chained) {
        const Chain ch = chain_of(s, p, st);
        BMTK_CHAIN_LAUNCH(scan_bwd_chain_kernel);
    } else {
        dim3 grid((unsigned)p.tiles, (unsigned)p.splits);
        if (p.splits > 1) {
            grid.y = (unsigned)p.splits - 1;
            if (p.one_round()) BMTK_SCAN_LAUNCH(scan_sums_kernel, BMTK_COMMA true BMTK_COMMA true);
            else BMTK_SCAN_LAUNCH(scan_sums_kernel, BMTK_COMMA true BMTK_COMMA false);
            grid.y = (unsigned)p.splits;
        }
        BMTK_SCAN_LAUNCH(scan_bwd_kernel, );
    }
    if (groups == 0)
        hipLaunchKernelGGL((scan_join_const_kernel<TA>), dim3((unsigned)div_up(dim, kWave)), dim3(kJoinWaves * kWave), 0, st, s.da_part, p.parts_const() * batch, dim,
                           (TA *)s.da);
    else if (s.da_part)
        hipLaunchKernelGGL((scan_join_shared_kernel<TA>), dim3((unsigned)div_up(s.n_steps * batch * groups, kBlock)), dim3(kBlock), 0, st, s.da_part,
                           s.n_steps * batch * groups, p.parts / groups, (TA *)s.da);
}

}  // namespace

// TX, TA and V for the call's types; V = 2 only for 16-bit types
#define BMTK_SCAN_TYPES(DO)                                             \
    do {                                                                \
        if (dtype == BMTK_F32) DO(float, float, 1);                     \
        else if (dtype == BMTK_BF16) {                                  \
            if (gate_dtype == BMTK_F32) {                               \
                if (p.v == 2) DO(bf16, float, 2);                       \
                else DO(bf16, float, 1);                                \
            } else {                                                    \
                if (p.v == 2) DO(bf16, bf16, 2);                        \
                else DO(bf16, bf16, 1);                                 \
            }                                                           \
        } else {                                                        \
            if (gate_dtype == BMTK_F32) {                               \
                if (p.v == 2) DO(f16, float, 2);                        \
                else DO(f16, float, 1);                                 \
            } else {                                                    \
                if (p.v == 2) DO(f16, f16, 2);                          \
                else DO(f16, f16, 1);                                   \
            }                                                           \
        }                                                               \
    } while (0)

// two neighbouring channels in one load
static bool in_pairs(const void *p, int dtype, int64_t stride_t, int64_t stride_b)
{
    return aligned(p, 2 * type_size(dtype)) && stride_t % 2 == 0 && stride_b % 2 == 0;
}

extern "C" int bmtk_gated_scan_fwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t dtype, int32_t gate_dtype, const void *x, int64_t x_t,
                                   int64_t x_b, const void *decay, int64_t a_t, int64_t a_b, const float *state, const int32_t *lengths, void *h, float *last,
                                   float *marks, float *workspace, void *stream)
{
    BMTK_REQUIRE(x && decay && h && last, "gated_scan_fwd: pointers must be non-null");
    const int rc = check_scan("gated_scan_fwd", n_steps, batch, dim, groups, dtype, gate_dtype);
    if (rc != BMTK_OK) return rc;
    bool pairs = in_pairs(x, dtype, x_t, x_b) && in_pairs(h, dtype, 0, 0) && aligned(state, 8) && aligned(last, 8) && aligned(marks, 8);
    if (groups == dim || groups == 0) pairs = pairs && in_pairs(decay, gate_dtype, a_t, a_b);
    const Plan p = plan_of(n_steps, batch, dim, groups, dtype, pairs);
    BMTK_REQUIRE(p.sums_floats(batch * dim) == 0 || n_steps == 1 || (workspace && aligned(workspace, 8)), "gated_scan_fwd: needs its workspace");
    BMTK_REQUIRE(p.tiles * p.waves * kWave < (1ll << 32), "gated_scan_fwd: too many columns");
    ScanArgs s{};
    s.x = x, s.a = decay, s.state = state, s.lengths = lengths, s.h = h, s.last = last, s.marks = marks, s.sums = workspace;
    s.n_steps = n_steps, s.columns = batch * dim, s.split_steps = p.split_steps;
    s.x_t = x_t, s.x_b = x_b, s.a_t = a_t, s.a_b = a_b;
    s.dim = dim, s.channels = groups > 0 ? dim / groups : 1, s.sequences = batch;
    const hipStream_t st = (hipStream_t)stream;
#define BMTK_DO(TX, TA, V) launch_fwd<TX, TA, V>(s, p, groups, st)
    BMTK_SCAN_TYPES(BMTK_DO);
#undef BMTK_DO
    BMTK_CHECK_LAUNCH("gated_scan_fwd");
    return BMTK_OK;
}

extern "C" int bmtk_gated_scan_bwd(int64_t n_steps, int64_t batch, int32_t dim, int32_t groups, int32_t dtype, int32_t gate_dtype, const void *x, int64_t x_t,
                                   int64_t x_b, const void *decay, int64_t a_t, int64_t a_b, const float *marks, const int32_t *lengths, const void *dh,
                                   int64_t dh_t, int64_t dh_b, const float *d_last, void *dx, void *d_decay, float *d_state, float *workspace, void *stream)
{
    BMTK_REQUIRE(x && decay && marks && dh && dx && d_decay, "gated_scan_bwd: pointers must be non-null");
    const int rc = check_scan("gated_scan_bwd", n_steps, batch, dim, groups, dtype, gate_dtype);
    if (rc != BMTK_OK) return rc;
    bool pairs = in_pairs(x, dtype, x_t, x_b) && in_pairs(dh, dtype, dh_t, dh_b) && in_pairs(dx, dtype, 0, 0) && aligned(marks, 8) && aligned(d_last, 8) &&
                 aligned(d_state, 8) && aligned(workspace, 8);
    if (groups == dim || groups == 0) pairs = pairs && in_pairs(decay, gate_dtype, a_t, a_b) && in_pairs(d_decay, gate_dtype, 0, 0);
    const Plan p = plan_of(n_steps, batch, dim, groups, dtype, pairs);
    const bool joined = groups == 0 || (groups != dim && p.parts != groups);
    BMTK_REQUIRE(groups == 0 || !joined || div_up(n_steps * batch * groups, kBlock) * kBlock < (1ll << 32), "gated_scan_bwd: too many gates, n_steps * batch * groups must stay below 2^32");
    BMTK_REQUIRE((p.sums_floats(batch * dim) == 0 && !joined) || (workspace && aligned(workspace, 8)), "gated_scan_bwd: needs its workspace");
    BMTK_REQUIRE(p.tiles * p.waves * kWave < (1ll << 32), "gated_scan_bwd: too many columns");
    ScanArgs s{};
    s.x = x, s.a = decay, s.lengths = lengths, s.marks = const_cast<float *>(marks), s.dh = dh, s.d_last = d_last;
    s.dx = dx, s.da = d_decay, s.d_state = d_state, s.sums = workspace;
    if (joined) s.da_part = workspace + p.sums_floats(batch * dim);
    s.n_steps = n_steps, s.columns = batch * dim, s.split_steps = p.split_steps;
    s.x_t = x_t, s.x_b = x_b, s.a_t = a_t, s.a_b = a_b, s.dh_t = dh_t, s.dh_b = dh_b;
    s.dim = dim, s.channels = groups > 0 ? dim / groups : 1, s.sequences = batch, s.seg_lanes = p.seg_lanes, s.parts = p.parts;
    const hipStream_t st = (hipStream_t)stream;
#define BMTK_DO(TX, TA, V) launch_bwd<TX, TA, V>(s, p, groups, st)
    BMTK_SCAN_TYPES(BMTK_DO);
#undef BMTK_DO
    BMTK_CHECK_LAUNCH("gated_scan_bwd");
    return BMTK_OK;
}
