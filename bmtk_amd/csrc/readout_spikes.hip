// Readout of spikes: y[t, b] = sum of the weight rows of the neurons that fired in step t of trial b, and its gradients.
#include <math.h>
#include <type_traits>

#include "readout.hpp"

namespace bmtk {
namespace {

constexpr int kWaves = 4;
constexpr int kManyWaves = 8, kOneBlockWaves = 16;   // of a workgroup of the forward pass
constexpr int kWordsPerLane = 4;  // spike words that a lane has under way at once
constexpr int kQueue = 512;       // spikes found and not yet added: at most 63 left over and one of each word under way
static_assert(kQueue >= kWave * (kWordsPerLane + 1) && (kQueue & (kQueue - 1)) == 0, "room for what a round finds");
constexpr int kSums = 32;         // sums of a lane, in registers

// A wavefront's own queue is written and read by different lanes of it, in order: what the compiler must keep is that order.
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Sums of a lane, VW channels of each of N trials or neurons.  Which of them a spike adds to is the same for all lanes, so that they stay in registers and
// are picked by number (an LDS addition of 64 floats takes 194 clocks on this chip, these seven instructions a tenth of it).
template <int VW, int N>
struct Accumulators {
    typedef float Vec __attribute__((ext_vector_type(N)));
    Vec sum[VW];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int c = 0; c < VW; ++c) sum[c] = 0.0f;
    }
    __device__ __forceinline__ void add(int which, const float (&v)[VW])
    {
#pragma unroll
        for (int c = 0; c < VW; ++c) sum[c][N == 1 ? 0 : which] += v[c];
    }
    __device__ __forceinline__ float get(int c, int which) const { return sum[c][N == 1 ? 0 : which]; }
};

// Adds the rows of m of a queue's spikes: that of lane k's spike, `row`, to the sums of lane k's `which`.  Rows are asked for sixteen (of
// four channels a lane: eight) at a time; `at` is where the lane's channels begin, within a row.
template <typename T, int VW, int N>
__device__ __forceinline__ void add_rows(Accumulators<VW, N> &acc, const T *__restrict__ rows, int dim, unsigned at, int row, int which, int m)
{
    constexpr int kLoads = VW == 4 ? 8 : 16;
    // (a lane works out its own row's distance, once for all)
    const uint64_t distance = (uint64_t)(uint32_t)row * (uint64_t)((uint32_t)dim * (uint32_t)sizeof(T));
    auto load = [&](Pack<T, VW>(&q)[kLoads], int k, int last) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const T *p = reinterpret_cast<const T *>(reinterpret_cast<const char *>(rows) + bcast_u64(distance, min(k + u, last)));
            q[u] = *reinterpret_cast<const Pack<T, VW> *>(p + at);
        }
    };
    auto add = [&](const Pack<T, VW> &q, int lane) {
        float v[VW];
#pragma unroll
        for (int c = 0; c < VW; ++c) v[c] = (float)q.v[c];
        acc.add(N == 1 ? 0 : bcast_i(which, lane), v);
    };
    int k = 0;
    for (; k + kLoads <= m; k += kLoads) {
        Pack<T, VW> q[kLoads];
        load(q, k, kWave - 1);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) add(q[u], k + u);
    }
    if (k < m) {
        Pack<T, VW> q[kLoads];
        load(q, k, m - 1);
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
            if (k + u < m) add(q[u], k + u);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward.  A workgroup takes one step and a slice of its words of spike bits; a wavefront turns the set bits of 64 kWords words at a
// time into a queue of element numbers, works it off 64 spikes at a time (each lane divides one of them into neuron and trial),
// and reads the weight rows, one per spike, 64 * VW channels by its 64 lanes.  The sums of a trial are the wavefront's own, so their
// order is fixed; the wavefronts' sums are added in order at the end, in the LDS that held the queues.
//
// What bounds it is reading rows at random from the L2s and from behind them: at 0.3 % of the neurons a step, 1,000 steps of 230,924 x 256 bf16 take 55 us
// (355 MB of rows, 6.4 TB/s), 600 steps of 51,978 x 32 x 64 fp32 127 us (766 MB, 6.0 TB/s); one step of the former with 64 channels fp32 6.9 us, most of
// it the launch and three dependent reads.
template <typename T, int VW, int N, int kFwdWaves, int kWords>
__global__ void __launch_bounds__(kFwdWaves * kWave)
spike_fwd_kernel(const uint64_t *__restrict__ bits, int64_t stride, int64_t ne, FastDiv by_batch, int trials, int trial_tiles,
                 const T *__restrict__ weight, int dim, int64_t slice_words, T *__restrict__ y, float *__restrict__ part)
{
    extern __shared__ float lds[];   // the queues, then half of the wavefronts' sums
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int64_t t = blockIdx.x;
    const int batch = (int)by_batch.d;
    const int b0 = (int)(blockIdx.z % trial_tiles) * trials, ch0 = (int)(blockIdx.z / trial_tiles) * kWave * VW;
    uint32_t *queue = reinterpret_cast<uint32_t *>(lds) + wave * kQueue;
    // (a lane without channels of its own reads the first ones and writes nothing)
    const unsigned at_ch = ch0 + lane * VW < dim ? ch0 + lane * VW : 0;
    Accumulators<VW, N> acc;
    acc.clear();
    const int64_t words = (ne + 63) >> 6;
    const int64_t w_begin = (int64_t)blockIdx.y * slice_words;
    const int w_count = (int)min(slice_words, words - w_begin);
    const uint64_t *row = bits + t * stride + w_begin;
    const uint64_t last_mask = (ne & 63) ? (1ull << (ne & 63)) - 1 : ~0ull;
    const int last_word = (int)min(words - 1 - w_begin, (int64_t)INT32_MAX);
    const uint32_t first_element = (uint32_t)(w_begin << 6);
    unsigned head = 0, tail = 0;

    auto load = [&](int c, uint64_t (&w)[kWords]) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = row[min(c + k * kWave + lane, w_count - 1)];
    };

    constexpr int kStep = kWave * kWords;
    uint64_t w[kWords] = {}, next[kWords];
    uint32_t first = 0;
    int c = wave * kStep;
    load(c, next);
    for (;;) {
        bool more = true;
        while (tail - head < kWave) {
            uint64_t any = 0;
#pragma unroll
            for (int k = 0; k < kWords; ++k) any |= w[k];
            if (__ballot(any != 0) == 0) {
                more = c < w_count;
                if (!more) break;
#pragma unroll
                for (int k = 0; k < kWords; ++k) {
                    const int at = c + k * kWave + lane;
                    w[k] = at < w_count ? next[k] & (at == last_word ? last_mask : ~0ull) : 0;
                }
                first = first_element + ((uint32_t)(c + lane) << 6);
                c += kFwdWaves * kStep;
                load(c, next);
            }
            // one spike of every word
#pragma unroll
            for (int k = 0; k < kWords; ++k) {
                // (of a word of nothing the last place, which nobody takes: there is no first one)
                const uint32_t e = first + (uint32_t)(k * kWave * 64) + (uint32_t)__builtin_ctzll(w[k] | (1ull << 63));
                bool mine = w[k] != 0;
                if (trial_tiles > 1) mine = mine && (unsigned)((int)(e - div_by(e, by_batch) * (uint32_t)batch) - b0) < (unsigned)trials;
                w[k] &= w[k] - 1;
                const unsigned long long mask = __ballot(mine);
                if (mine) queue[(tail + lane_prefix(mask)) & (kQueue - 1)] = e;
                tail += (unsigned)__popcll(mask);
            }
        }
        wave_order();
        const int m = (int)min(tail - head, (unsigned)kWave);
        if (m > 0) {
            const uint32_t e = queue[(head + lane) & (kQueue - 1)];
            const int i = (int)div_by(e, by_batch);
            add_rows<T, VW, N>(acc, weight, dim, at_ch, i, (int)e - i * batch - b0, m);
            head += m;
        }
        wave_order();
        if (!more && tail == head) break;
    }
    // the upper half of the wavefronts' sums to the lower half's, then those together
    constexpr int kHalf = kFwdWaves / 2;
    const int cells = trials * kWave * VW;
    float *slot = lds + (wave % kHalf) * cells;
    auto put = [&] {
        for (int b = 0; b < trials; ++b)
#pragma unroll
            for (int c = 0; c < VW; ++c) slot[(b * VW + c) * kWave + lane] = acc.get(c, b);
    };
    __syncthreads();
    if (wave >= kHalf) put();
    __syncthreads();
    if (wave < kHalf) {
        for (int b = 0; b < trials; ++b) {
            float v[VW];
#pragma unroll
            for (int c = 0; c < VW; ++c) v[c] = slot[(b * VW + c) * kWave + lane];
            acc.add(b, v);
        }
        put();   // (its own places)
    }
    __syncthreads();
    const int here = min(trials, batch - b0);
    const int64_t out = (t * batch + b0) * (int64_t)dim + ch0;
    const int64_t plane = (int64_t)gridDim.x * batch * dim;
    for (int c = threadIdx.x; c < here * kWave * VW; c += kFwdWaves * kWave) {
        const int l = c % (kWave * VW), b = c / (kWave * VW);
        if (ch0 + l >= dim) continue;
        const float *a = lds + (b * VW + l % VW) * kWave + l / VW;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < kHalf; ++k) s += a[k * cells];
        if (part)
            part[blockIdx.y * plane + out + (int64_t)b * dim + l] = s;
        else
            y[out + (int64_t)b * dim + l] = (T)s;
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock) spike_join_kernel(const float *__restrict__ part, int slices, int64_t plane, T *__restrict__ y)
{
    const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= plane) return;
    float s = 0.0f;
    for (int k = 0; k < slices; ++k) s += part[k * plane + c];
    y[c] = (T)s;
}

// ---------------------------------------------------------------------------------------------------------------------
// Gradient by the weights: row i is the sum of dy[t, b] over the spikes of neuron i.  A wavefront owns `own` neurons and their
// sums, looks through their bits of all steps and reads the dy rows as the forward pass reads the weights.  Nobody else
// adds to its sums: the order is fixed and nothing has to be joined.  600 steps of 51,978 x 32 x 64 fp32: 147 us (766 MB of dy rows, 5.2 TB/s, more
// than half of them out of the L2s).
template <typename T, int VW, int N>
__global__ void __launch_bounds__(kWaves * kWave)
spike_bwd_weight_kernel(const uint64_t *__restrict__ bits, int64_t stride, int64_t n_steps, int64_t n, FastDiv by_batch, int own,
                        const T *__restrict__ dy, int dim, T *__restrict__ d_weight)
{
    __shared__ uint64_t queues[kWaves][kQueue];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int batch = (int)by_batch.d;
    uint64_t *queue = queues[wave];
    const int ch = blockIdx.y * kWave * VW + lane * VW;
    const bool in = ch < dim;
    const unsigned at_ch = in ? ch : 0;
    const int64_t i0 = ((int64_t)blockIdx.x * kWaves + wave) * own;
    if (i0 >= n) return;
    const int mine = (int)min((int64_t)own, n - i0);
    Accumulators<VW, N> acc;
    acc.clear();
    // bits e0 .. e1 of a step, in words w0 .. w0 + nw
    const int64_t e0 = i0 * batch, e1 = (i0 + mine) * batch, w0 = e0 >> 6;
    const int nw = (int)(((e1 + 63) >> 6) - w0);
    const uint64_t first_mask = ~0ull << (e0 & 63), last_mask = (e1 & 63) ? (1ull << (e1 & 63)) - 1 : ~0ull;
    const uint64_t *own_bits = bits + w0;
    const uint32_t first_element = (uint32_t)((w0 << 6) - e0);   // (perhaps below zero: the first word's bits are looked at from e0 on)
    unsigned head = 0, tail = 0;

    // (step, word) pairs, the word faster: lane l begins with pair l and goes on by 64
    int t = lane / nw, w_at = lane % nw;
    const int dt = kWave / nw, dw = kWave % nw, steps = (int)n_steps;
    uint64_t next[kWordsPerLane];
    uint32_t next_t[kWordsPerLane], next_w[kWordsPerLane];
    auto load = [&] {
#pragma unroll
        for (int k = 0; k < kWordsPerLane; ++k) {
            next[k] = own_bits[min(t, steps - 1) * stride + w_at];
            next_t[k] = (uint32_t)t;
            next_w[k] = (uint32_t)w_at;
            t += dt;
            w_at += dw;
            if (w_at >= nw) {
                w_at -= nw;
                ++t;
            }
        }
    };
    load();
    uint64_t w[kWordsPerLane] = {};
    uint32_t at_t[kWordsPerLane] = {}, at_e[kWordsPerLane] = {};
    for (;;) {
        bool more = true;
        while (tail - head < kWave) {
            uint64_t any = 0;
#pragma unroll
            for (int k = 0; k < kWordsPerLane; ++k) any |= w[k];
            if (__ballot(any != 0) == 0) {
                more = __ballot((int)next_t[0] < steps) != 0;
                if (!more) break;
#pragma unroll
                for (int k = 0; k < kWordsPerLane; ++k) {
                    w[k] = (int)next_t[k] < steps ? next[k] : 0;
                    if (next_w[k] == 0) w[k] &= first_mask;
                    if ((int)next_w[k] == nw - 1) w[k] &= last_mask;
                    at_t[k] = next_t[k];
                    at_e[k] = first_element + (next_w[k] << 6);
                }
                load();
            }
#pragma unroll
            for (int k = 0; k < kWordsPerLane; ++k) {
                const unsigned long long mask = __ballot(w[k] != 0);
                if (w[k] != 0) queue[(tail + lane_prefix(mask)) & (kQueue - 1)] = ((uint64_t)at_t[k] << 32) | (uint32_t)(at_e[k] + (uint32_t)__builtin_ctzll(w[k]));
                w[k] &= w[k] - 1;
                tail += (unsigned)__popcll(mask);
            }
        }
        wave_order();
        const int m = (int)min(tail - head, (unsigned)kWave);
        if (m > 0) {
            const uint64_t q = queue[(head + lane) & (kQueue - 1)];
            const uint32_t e = (uint32_t)q;
            const int i = (int)div_by(e, by_batch);
            add_rows<T, VW, N>(acc, dy, dim, at_ch, (int)((uint32_t)(q >> 32) * (uint32_t)batch + (e - (uint32_t)i * (uint32_t)batch)), i, m);
            head += m;
        }
        wave_order();
        if (!more && tail == head) break;
    }
    if (in)
        for (int i = 0; i < mine; ++i) {
            Pack<T, VW> q;
#pragma unroll
            for (int c = 0; c < VW; ++c) q.v[c] = (T)acc.get(c, i);
            *reinterpret_cast<Pack<T, VW> *>(d_weight + (i0 + i) * dim + ch) = q;
        }
}

// ---------------------------------------------------------------------------------------------------------------------
// Gradient by the spikes: dl_dz[t, i, b] = dy[t, b] . W[i], a matrix product whose result is most of its traffic.  A wavefront keeps
// the weights of 64 neurons in registers, 64 channels of them; the workgroup puts the dy rows of 32 (step, trial) pairs into LDS, in the order in which
// the matrix instructions take them, while those before are multiplied.
//
// fp32: the matrix instructions take 16-bit operands sixteen times as fast as 32-bit ones.  Each operand is the sum of three bf16 numbers of 8 bits each
// (what the one before leaves, rounded), exact to 2^-27 of it, and to 2^-134 of anything, where bf16 ends: below 1e-34 that is more, an operand around 1e-36 is
// off by 3e-5 of itself, one around 1e-39 by 3 %.  Of the nine products the six that are not below 2^-24 of the whole are made and added up in fp32.
// fp16: the matrix instructions lose what a product with an operand below 2^-14 has below about 2^-35 (of operands around 2e-7 4e-6 of the sum).
//
// 600 steps of 51,978 x 32 x 64 fp32: 936 us at the median, 755 at best, for 3.99 GB of results (4.3 to 5.3 TB/s).  Writing them alone, in this order, takes 710 to
// 760 us, a fill of as much memory from front to back 583.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
constexpr int kDzK = 64;          // channels at a time
constexpr int kDzWaves = 4;
constexpr int kDzGroups = 2;      // of 32 neurons, of a wavefront
constexpr int kDzNeurons = 32 * kDzGroups;
constexpr int kDzRows = 32;       // (step, trial) pairs at a time

// Eight channels of a row as operands of a matrix instruction
template <typename T>
struct Operand;
template <>
struct Operand<float> {
    static constexpr int kParts = 3;
    typedef bf16x8 Part;
    // whether all numbers are finite (as bf16, too): only then are they the sum of their parts
    __device__ __forceinline__ static bool split(const float (&v)[8], Part (&part)[3])
    {
        float odd = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            float left = v[s];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const bf16 b = (bf16)left;
                part[p][s] = b;
                if (p == 0) odd += (float)b * 0.0f;
                left -= (float)b;
            }
        }
        return odd == 0.0f;
    }
    __device__ __forceinline__ static f32x16 multiply(const Part &a, const Part &b, const f32x16 &acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0); }
};
// fp32 as it is: for small products, whose time is not the matrix instructions'
struct Whole {};
template <>
struct Operand<Whole> {
    static constexpr int kParts = 1;
    typedef f32x8 Part;
    __device__ __forceinline__ static bool split(const float (&v)[8], Part (&part)[1])
    {
#pragma unroll
        for (int s = 0; s < 8; ++s) part[0][s] = v[s];
        return true;
    }
    __device__ __forceinline__ static f32x16 multiply(const Part &a, const Part &b, f32x16 acc)
    {
#pragma unroll
        for (int s = 0; s < 8; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], acc, 0, 0, 0);
        return acc;
    }
};
template <>
struct Operand<bf16> {
    static constexpr int kParts = 1;
    typedef bf16x8 Part;
    __device__ __forceinline__ static bool split(const bf16 (&v)[8], Part (&part)[1])
    {
#pragma unroll
        for (int s = 0; s < 8; ++s) part[0][s] = v[s];
        return true;
    }
    __device__ __forceinline__ static f32x16 multiply(const Part &a, const Part &b, const f32x16 &acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0); }
};
template <>
struct Operand<f16> {
    static constexpr int kParts = 1;
    typedef f16x8 Part;
    __device__ __forceinline__ static bool split(const f16 (&v)[8], Part (&part)[1])
    {
#pragma unroll
        for (int s = 0; s < 8; ++s) part[0][s] = v[s];
        return true;
    }
    __device__ __forceinline__ static f32x16 multiply(const Part &a, const Part &b, const f32x16 &acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); }
};

// Eight channels of row `row` of those that begin at `base`, of which there are `rows` (at least one) left; zero where there is no such row or channel.
// (No branches: what lies outside is read from elsewhere in the last row, and its bits are cleared.  Offsets of 32 bits from a place that is the
// same for all lanes.)
template <typename T, int VL>
__device__ __forceinline__ void load_eight(const T *__restrict__ base, int row, int rows, int dim, int k0, T (&v)[8])
{
    constexpr int kBytes = VL * sizeof(T);
    typedef typename std::conditional<kBytes % 4 == 0, uint32_t, uint16_t>::type Word;
    const unsigned at = (unsigned)min(row, rows - 1) * (unsigned)dim;
#pragma unroll
    for (int s = 0; s < 8; s += VL) {
        Pack<T, VL> q = *reinterpret_cast<const Pack<T, VL> *>(base + (at + (unsigned)min(k0 + s, dim - VL)));
        Word w[kBytes / sizeof(Word)];
        __builtin_memcpy(w, &q, kBytes);
        const Word keep = (Word)-(int)(row < rows && k0 + s < dim);
#pragma unroll
        for (unsigned c = 0; c < kBytes / sizeof(Word); ++c) w[c] &= keep;
        __builtin_memcpy(&q, w, kBytes);
#pragma unroll
        for (int c = 0; c < VL; ++c) v[s + c] = q.v[c];
    }
}

// The same of rows at any distance, for kAny: 16 bytes a load all the same, which need no other alignment than their numbers'.  What would reach behind a row
// is read from further left and moved there.  (At least 16 bytes a row.)
constexpr int kAny = 0;
template <typename T>
__device__ __forceinline__ void load_eight_any(const T *__restrict__ base, int row, int rows, int dim, int k0, T (&v)[8])
{
    constexpr int N = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Loose {
        uint32_t w[4];
    };
    const unsigned at = (unsigned)min(row, rows - 1) * (unsigned)dim;
#pragma unroll
    for (int s = 0; s < 8; s += N) {
        const int from = min(k0 + s, dim - N), shift = row < rows ? k0 + s - from : N;
        const Loose q = *reinterpret_cast<const Loose *>(base + (at + (unsigned)from));
        uint32_t w0 = q.w[0], w1 = q.w[1], w2 = q.w[2], w3 = q.w[3];
        if constexpr (sizeof(T) == 2) {
            const bool half = shift & 1;
            w0 = half ? (w0 >> 16) | (w1 << 16) : w0, w1 = half ? (w1 >> 16) | (w2 << 16) : w1, w2 = half ? (w2 >> 16) | (w3 << 16) : w2, w3 = half ? w3 >> 16 : w3;
        }
        const int words = shift * (int)sizeof(T) / 4;
        const bool one = words & 1, two = words & 2, none = shift >= N;
        w0 = one ? w1 : w0, w1 = one ? w2 : w1, w2 = one ? w3 : w2, w3 = one ? 0 : w3;
        w0 = two ? w2 : w0, w1 = two ? w3 : w1, w2 = two ? 0 : w2, w3 = two ? 0 : w3;
        const uint32_t w[4] = {none ? 0 : w0, none ? 0 : w1, none ? 0 : w2, none ? 0 : w3};
        __builtin_memcpy(v + s, w, 16);
    }
}
template <typename T, int VL>
__device__ __forceinline__ void load_eight_of(const T *__restrict__ base, int row, int rows, int dim, int k0, T (&v)[8])
{
    if constexpr (VL == kAny) load_eight_any<T>(base, row, rows, dim, k0, v);
    else load_eight<T, VL>(base, row, rows, dim, k0, v);
}

// How the products reach memory.  kPairs: neighbouring lanes hold neighbouring (step, trial) pairs.  kAcross (one trial): neighbouring
// neurons.  kTurned + s (4, 8, 16 or a multiple of 32 trials, 2^s fours of them in a tile, and rows that begin on 128 bytes): through LDS into the
// order of memory, 16 bytes a lane, whole lines past the caches.  (Parts of lines written past the caches take five times as long.)
// kSteps1, kSteps4 (2 to 31 trials, up to 64 channels, no small product): a tile is whole steps, 24 pairs at least, and goes through LDS into the order of
// memory too, 4 or (where that divides the trials) 16 bytes a lane.  600 steps of 20,000, against kPairs: 24 trials, 64 channels bf16 244 / 480 us; 12, 64 fp32
// 242 / 266; 10, 33 bf16 139 / 161.  (More channels: the smaller tiles read the weights more often, 12 trials, 300 fp16 269 / 231.)
enum { kPairs = 0, kAcross = 1, kTurned = 2, kSteps1 = 6, kSteps4 = 7 };

// kOnePass: up to 64 channels.  More: passes over 64 of them at a time, each for kTiles tiles of rows, whose sums wait in registers meanwhile (weights that
// are read again for every tile take 710 us where these take 522, 415 where these take 229: 300 steps of 20,000 x 32, 128 channels fp32, and x 12, 300 fp16).
template <typename T, typename O, int VL, int kOut, bool kOnePass>
__global__ void __launch_bounds__(kDzWaves * kWave, kOnePass && (kOut >= kTurned || sizeof(T) == 2) ? 3 : 2)
spike_bwd_spikes_kernel(const T *__restrict__ weight, const T *__restrict__ dy, int64_t rows, int64_t n, FastDiv by_batch, int dim,
                        int64_t rows_per_block, int32_t *__restrict__ not_finite, float *__restrict__ dl_dz)
{
    typedef Operand<O> Op;
    typedef typename Op::Part Part;
    constexpr int P = Op::kParts, kTiles = kOnePass ? 1 : sizeof(T) == 2 ? 4 : 2;
    static_assert(kDzRows * kDzK / 8 == kDzWaves * kWave, "eight channels of a row for every thread");
    // [part][eighth of the channels][row]: what a wavefront reads at once, rows of two eighths, lies together
    __shared__ Part staged[2][P][kDzK / 8][kDzRows];
    __shared__ f32x4 turn[kOut >= kTurned ? kDzWaves : 1][32 * 8];
    __shared__ int odd;   // some number is not finite
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int half = lane / 32, col = lane % 32;
    const int batch = (int)by_batch.d;
    const int64_t ne = n * batch;
    const int64_t i0 = ((int64_t)blockIdx.x * kDzWaves + wave) * kDzNeurons;
    const int64_t r_begin = (int64_t)blockIdx.y * rows_per_block, r_end = min(rows, r_begin + rows_per_block);
    const int passes = kOnePass ? 1 : (dim + kDzK - 1) / kDzK;
    // a stage: a tile of rows and a pass; the tiles of a pass one after the other, then the next pass
    const int tile_rows = kOut >= kSteps1 ? kDzRows / batch * batch : kDzRows;
    const int all_tiles = (int)((r_end - r_begin + tile_rows - 1) / tile_rows), tiles = kOnePass ? 1 : min(kTiles, all_tiles);
    const int stages = (all_tiles + tiles - 1) / tiles * passes * tiles;
    T next[8];
    auto load_rows = [&](int stage) {
        const int at = min(stage, stages - 1);   // (behind the last one: it again, which nobody looks at)
        const int64_t r = min(r_begin + ((int64_t)(at / tiles / passes) * tiles + at % tiles) * tile_rows, r_end - 1);
        load_eight_of<T, VL>(dy + r * dim, threadIdx.x / 8, (int)min(r_end - r, (int64_t)kDzRows), dim, at / tiles % passes * kDzK + threadIdx.x % 8 * 8, next);
    };
    Part a[kDzGroups][P][kDzK / 16];
    auto load_weights = [&](int pass) {
        bool fine = true;
#pragma unroll
        for (int g = 0; g < kDzGroups; ++g)
#pragma unroll
            for (int q = 0; q < kDzK / 16; ++q) {
                T v[8];
                Part part[P];
                if (pass * kDzK + q * 16 >= dim) break;
                // (a wavefront behind the last neuron multiplies the last one's weights, and writes nothing)
                const int64_t first = min(i0, n - 1);
                load_eight_of<T, VL>(weight + first * dim, g * 32 + col, (int)min(n - first, (int64_t)kDzNeurons), dim, pass * kDzK + (2 * q + half) * 8, v);
                fine = Op::split(v, part) && fine;
#pragma unroll
                for (int p = 0; p < P; ++p) a[g][p][q] = part[p];
            }
        return fine;
    };
    f32x16 sums[kTiles][kDzGroups];
    // register k of a lane: column col, row 8 (k / 4) + 4 half + k % 4.  (Pointers that move on: places kept are as many registers.)
    auto put = [&](int64_t r0, const f32x16(&sums)[kDzGroups]) {
        const bool whole = i0 + kDzNeurons <= n && r0 + kDzRows <= r_end;
#pragma unroll
        for (int g = 0; g < kDzGroups; ++g) {
            const int64_t ig = i0 + g * 32;
            if (kOut >= kTurned) {
                // [neuron][pairs by four], turned by the neuron so that neither side meets itself in a bank
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    turn[wave][col * 8 + ((2 * q + half) ^ (col & 7))] = f32x4{sums[g][4 * q], sums[g][4 * q + 1], sums[g][4 * q + 2], sums[g][4 * q + 3]};
                wave_order();
                if constexpr (kOut >= kSteps1) {
                    // 32 neurons' trials of a step lie together
                    const int rows_here = (int)min((int64_t)tile_rows, r_end - r0), left = (int)min((int64_t)32, n - ig);
                    float *to = dl_dz + (int64_t)div_by((uint32_t)r0, by_batch) * ne + ig * batch;
                    if constexpr (kOut == kSteps4) {
                        // (four trials a lane, of all steps of the tile in turn)
#pragma unroll 1
                        for (int at = 4 * lane; at < rows_here * 32; at += 4 * kWave) {
                            const int all_i = (int)div_by((uint32_t)at, by_batch), i = all_i & 31, step = all_i >> 5, b = at - all_i * batch;
                            if (i < left) *reinterpret_cast<f32x4 *>(to + (step * ne + i * batch + b)) = turn[wave][i * 8 + (((step * batch + b) >> 2) ^ (i & 7))];
                        }
                    } else {
                        const float *from = reinterpret_cast<const float *>(turn[wave]);
                        for (int pair = 0; pair < rows_here; pair += batch, to += ne)
                            for (int at = lane; at < left * batch; at += kWave) {
                                const int i = (int)div_by((uint32_t)at, by_batch), q = pair + at - i * batch;
                                to[at] = from[(i * 8 + ((q >> 2) ^ (i & 7))) * 4 + (q & 3)];
                            }
                    }
                    wave_order();
                    continue;
                }
                // A neuron has 2^kShift fours of trials in a step; up to 32 trials the tile begins with a step, of more it is a part of one.  Four `at`
                // of the tile, in the order of memory: step at >> (kShift + 5), neuron (at >> kShift) & 31; of 64 k + lane the sum of both parts'.
                constexpr int kShift = kOut - kTurned;
                const int64_t t0 = kShift < 3 ? r0 >> (kShift + 2) : (int64_t)div_by((uint32_t)r0, by_batch);
                const int c = lane & ((1 << kShift) - 1), i_lane = (lane >> kShift) & 31, step_lane = lane >> (kShift + 5);
                float *to = dl_dz + (t0 + step_lane) * ne + (ig + i_lane) * batch + (r0 - t0 * batch) + 4 * c;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i_k = ((k * kWave) >> kShift) & 31, step_k = (k * kWave) >> (kShift + 5);
                    const int i = i_lane + i_k, c4 = ((step_lane + step_k) << kShift) + c;
                    const f32x4 v = turn[wave][i * 8 + (c4 ^ (i & 7))];
                    if (whole || (ig + i < n && r0 + 4 * c4 < r_end)) __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(to + (step_k * ne + i_k * batch)));
                }
                wave_order();
            } else if (kOut == kAcross) {
                int64_t r = r0 + 4 * half;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    // (one trial: a pair is a step)
                    if (whole || (r < r_end && ig + col < n)) dl_dz[r * ne + ig + col] = sums[g][k];
                    r += k % 4 == 3 ? 5 : 1;
                }
            } else {
                const uint32_t t = div_by((uint32_t)min(r0 + col, r_end - 1), by_batch);
                int64_t i = ig + 4 * half;
                float *p = dl_dz + t * ne + (r0 + col - (int64_t)t * batch) + i * batch;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (whole || (i < n && r0 + col < r_end)) *p = sums[g][k];
                    const int on = k % 4 == 3 ? 5 : 1;
                    p += (int64_t)on * batch;
                    i += on;
                }
            }
        }
    };

    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    load_rows(0);
    if (!load_weights(0)) odd = 1;
    for (int first = 0; first < stages; first += tiles) {
        const int pass = kOnePass ? 0 : first / tiles % passes;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            if (j > 0 && j >= tiles) continue;
            const int stage = first + j, buffer = stage & 1;
            {
                Part part[P];
                if (!Op::split(next, part)) odd = 1;
#pragma unroll
                for (int p = 0; p < P; ++p) staged[buffer][p][threadIdx.x % 8][threadIdx.x / 8] = part[p];
            }
            load_rows(stage + 1);
            // (two buffers in turn: whoever writes the one of a stage has passed the barrier behind the reads of the stage before the last)
            __syncthreads();
            if (pass == 0)
#pragma unroll
                for (int g = 0; g < kDzGroups; ++g) sums[j][g] = 0.0f;
#pragma unroll
            for (int q = 0; q < kDzK / 16; ++q) {
                if (pass * kDzK + q * 16 >= dim) break;
                Part b[P];
#pragma unroll
                for (int p = 0; p < P; ++p) b[p] = staged[buffer][p][2 * q + half][col];
#pragma unroll
                for (int order = P - 1; order >= 0; --order)   // the small ones first
#pragma unroll
                    for (int p = 0; p <= order; ++p)
#pragma unroll
                        for (int g = 0; g < kDzGroups; ++g)
                            sums[j][g] = kOut == kPairs ? Op::multiply(a[g][p][q], b[order - p], sums[j][g]) : Op::multiply(b[order - p], a[g][p][q], sums[j][g]);
            }
        }
        if (!kOnePass && !load_weights(pass < passes - 1 ? pass + 1 : 0)) odd = 1;
        if (kOnePass || pass == passes - 1)
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
                const int64_t r0 = r_begin + ((int64_t)(first / tiles / passes) * tiles + j) * tile_rows;
                if (j == 0 || (j < tiles && r0 < r_end)) put(r0, sums[j]);
            }
    }
    if (P > 1) {
        __syncthreads();
        if (threadIdx.x == 0) not_finite[blockIdx.y * gridDim.x + blockIdx.x] = odd;
    }
}

// What the product in parts is not right for: results of a row of dy or of the weights that holds an infinity, a NaN or a number that is infinite as bf16.  Those
// once more, product by product in fp32, as it comes; all others stay.  A workgroup looks at a part, a thread at a neuron; rows are looked at 256 at a time.
// 600 steps of 51,978 x 32 x 64 in 1.1 ms: with a NaN in a row of dy as long, with an infinite weight 6.0 (a thread makes 928 results), of NaN alone 5.7.
enum { kFine = 0, kInfinite = 1, kNaN = 2 };
__device__ __forceinline__ int kind_of(const float *__restrict__ row, int dim)
{
    int kind = kFine;
    for (int c = 0; c < dim; ++c) {
        const float v = row[c];
        kind = max(kind, v != v ? kNaN : __builtin_fabsf(v) < 0x1.ffp127f ? kFine : kInfinite);
    }
    return kind;
}
__global__ void __launch_bounds__(kBlock)
spike_bwd_spikes_again_kernel(const float *__restrict__ weight, const float *__restrict__ dy, int64_t rows, int64_t n, FastDiv by_batch, int dim,
                              int64_t rows_per_block, int parts_across, const int32_t *__restrict__ not_finite, float *__restrict__ dl_dz)
{
    static_assert(kDzWaves * kDzNeurons == kBlock, "a thread for each neuron of a part");
    const int part = blockIdx.x;
    if (not_finite[part] == 0) return;
    __shared__ int kinds[kBlock];
    const int64_t r_begin = (int64_t)(part / parts_across) * rows_per_block, r_end = min(rows, r_begin + rows_per_block);
    const int64_t i = (int64_t)(part % parts_across) * kBlock + threadIdx.x;
    const bool in = i < n;
    const int own = in ? kind_of(weight + i * dim, dim) : kFine;
    for (int64_t r0 = r_begin; r0 < r_end; r0 += kBlock) {
        const int here = (int)min((int64_t)kBlock, r_end - r0);
        __syncthreads();
        if ((int)threadIdx.x < here) kinds[threadIdx.x] = kind_of(dy + (r0 + threadIdx.x) * dim, dim);
        __syncthreads();
        for (int k = 0; k < here; ++k) {
            const int kind = max(own, kinds[k]);
            if (!in || kind == kFine) continue;
            const int64_t r = r0 + k;
            const uint32_t t = div_by((uint32_t)r, by_batch);
            float s = kind == kNaN ? NAN : 0.0f;
            for (int c = 0; c < dim && s == s; ++c) s += weight[i * dim + c] * dy[r * dim + c];
            dl_dz[(t * n + i) * by_batch.d + (r - (int64_t)t * by_batch.d)] = s;
        }
    }
}

// channels a lane takes: as many as cover a row, of those that its alignment allows
int lane_channels(int dim, int dtype, const void *p)
{
    int vw = 1;
    while (vw < 4 && vw * kWave < dim && dim % (2 * vw) == 0 && aligned(p, 2 * vw * type_size(dtype))) vw *= 2;
    return vw;
}

// Slices of a step's words: enough workgroups that those left over at the end are few, but no more than one for every two loads of words of its wavefronts
// (begun ones too: 1,025 words are two slices).  600 steps of 51,978 x 32 x 64: one slice 152 us, two 127 and 6 for their sum.  Two loads against
// one: 100 steps of 3,001 x 12 x 17 6.8 / 8.3 us, 1 of 51,978 x 32 x 64 14.9 / 19.1, 200 of 6,000 x 16 x 10 11.2 / 12.2; many spikes would have more
// slices, 50 of 5,000 x 32 x 64 at 2 % 19.3 / 15.0, but nobody knows them here.
int64_t fwd_slices(int64_t n_steps, int64_t words, int64_t tiles)
{
    const int64_t most = div_up(words, 2 * kManyWaves * kWave);
    int64_t s = 1200 / (n_steps * tiles);
    s = s < 1 ? 1 : s;
    return s < most ? s : most;
}

struct FwdPlan {
    int vw, trials, trial_tiles, tiles, waves, words_per_lane;
    int64_t slices, slice_words;
};
FwdPlan fwd_plan(int64_t n_steps, int64_t n, int batch, int dim, int vw)
{
    FwdPlan p;
    p.vw = vw;
    p.trial_tiles = (int)div_up(batch, kSums / vw);
    p.trials = (int)div_up(batch, p.trial_tiles);
    p.tiles = p.trial_tiles * (int)div_up(dim, kWave * vw);
    const int64_t words = (n * batch + 63) / 64;
    p.slices = fwd_slices(n_steps, words, p.tiles);
    p.waves = kManyWaves;
    // one step of one trial, up to four words a lane of one workgroup: no slices to join.  A word a lane at a time, where not all
    // wavefronts have four: four at once take longer.  64 channels fp32 at 0.3 %, in one workgroup / that with four words at once / in the slices
    // from above and their sum: 230,924 neurons 7.0 / 7.5 / 8.7 us, 100,000 4.8 / 5.6 / 8.8, 262,144 8.3 / 8.3 / 8.8.  At 2 %, which nobody knows here, slices
    // would be better, 230,924 neurons 21.1 / 24.2 / 12.8.
    if (batch == 1 && p.slices > 1 && words <= kOneBlockWaves * kWave * kWordsPerLane) p.slices = 1, p.waves = kOneBlockWaves;
    p.slice_words = div_up(div_up(words, p.slices), kWave) * kWave;
    p.slices = div_up(words, p.slice_words);
    // (one where four would leave wavefronts without any)
    p.words_per_lane = p.slice_words < p.waves * kWave * kWordsPerLane ? 1 : kWordsPerLane;
    return p;
}

struct DzPlan {
    int64_t across, per_block, down, parts;
    int tile_rows;   // (step, trial) pairs of a tile
    bool whole;   // fp32: in fp32 instructions.  Up to this many products they take some us at most, less than the launch that looks for infinities
};
constexpr double kWholeProducts = 3e8;
DzPlan dz_plan(int64_t n_steps, int64_t n, int batch, int dim)
{
    DzPlan p;
    p.whole = (double)n_steps * batch * n * dim < kWholeProducts;
    p.across = div_up(n, kDzWaves * kDzNeurons);
    p.tile_rows = batch > 1 && batch < kDzRows ? kDzRows / batch * batch : kDzRows;
    if (p.whole || dim > kDzK || 4 * p.tile_rows < 3 * kDzRows) p.tile_rows = kDzRows;
    const int64_t rows = n_steps * batch, most = div_up(rows, p.tile_rows);
    int64_t blocks = div_up(4096, p.across);
    if (blocks > most) blocks = most;
    p.per_block = div_up(most, blocks) * p.tile_rows;
    p.down = div_up(rows, p.per_block);
    p.parts = p.across * p.down;
    return p;
}

int check_sizes(const char *who, int64_t n_steps, int64_t n, int32_t batch, int32_t dim, int32_t dtype)
{
    BMTK_REQUIRE(n_steps > 0 && n > 0 && batch > 0 && dim > 0, "%s: sizes must be positive", who);
    BMTK_REQUIRE(dtype == BMTK_F32 || dtype == BMTK_BF16 || dtype == BMTK_F16, "%s: unknown type %d", who, dtype);
    BMTK_REQUIRE(n < (1ll << 31) && n * (int64_t)batch < (1ll << 31) - 64, "%s: n_neurons * batch must stay below 2^31 - 64", who);
    BMTK_REQUIRE(n_steps < (1ll << 23) && n_steps * (int64_t)batch < (1ll << 31) - 64, "%s: n_steps must stay below 2^23 and n_steps * batch below 2^31 - 64", who);
    BMTK_REQUIRE(dim <= 65536 && batch <= 65536, "%s: batch and dim are at most 65,536", who);
    return BMTK_OK;
}

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_spike_readout_workspace_bytes(int64_t n_steps, int64_t n_neurons, int32_t batch, int32_t dim, int32_t backward)
{
    if (check_sizes("spike_readout_workspace_bytes", n_steps, n_neurons, batch, dim, BMTK_F32) != BMTK_OK) return 0;
    if (backward) {
        const DzPlan p = dz_plan(n_steps, n_neurons, batch, dim);
        return p.whole ? 0 : p.parts * (int64_t)sizeof(int32_t);
    }
    int64_t slices = 1;   // (as many as any alignment of the weights takes)
    for (int vw = 1; vw <= 4; vw *= 2) {
        const FwdPlan p = fwd_plan(n_steps, n_neurons, batch, dim, vw);
        slices = p.slices > slices ? p.slices : slices;
    }
    return slices > 1 ? slices * n_steps * batch * dim * (int64_t)sizeof(float) : 0;
}

extern "C" int bmtk_spike_readout_fwd(const uint64_t *spike_bits, int64_t stride, int64_t n_steps, int64_t n_neurons, int32_t batch, const void *weight,
                                      int32_t dim, int32_t dtype, void *y, float *workspace, void *stream)
{
    BMTK_REQUIRE(spike_bits && weight && y, "spike_readout_fwd: pointers must be non-null");
    int rc = check_sizes("spike_readout_fwd", n_steps, n_neurons, batch, dim, dtype);
    if (rc != BMTK_OK) return rc;
    BMTK_REQUIRE(stride >= (n_neurons * batch + 63) / 64, "spike_readout_fwd: stride is shorter than a step's words");
    const FwdPlan p = fwd_plan(n_steps, n_neurons, batch, dim, lane_channels(dim, dtype, weight));
    BMTK_REQUIRE(p.tiles < 65536 && p.slices < 65536, "spike_readout_fwd: too many trials and channels");
    BMTK_REQUIRE(p.slices == 1 || workspace, "spike_readout_fwd: needs its workspace");
    float *part = p.slices > 1 ? workspace : nullptr;
    const int64_t plane = n_steps * batch * (int64_t)dim;
    BMTK_REQUIRE(plane < (1ll << 31), "spike_readout_fwd: the result is too large");
    const dim3 grid((unsigned)n_steps, (unsigned)p.slices, (unsigned)p.tiles);
    const size_t queues = (size_t)p.waves * kQueue * sizeof(uint32_t), sums = (size_t)p.waves / 2 * p.trials * kWave * p.vw * sizeof(float);
    const size_t lds = queues > sums ? queues : sums;   // (at most 32 KB)
    const hipStream_t st = (hipStream_t)stream;
    const FastDiv by_batch = fast_div((uint32_t)batch);
#define BMTK_FWD_W(VW, N, WAVES, WORDS)                                                                                                                      \
    hipLaunchKernelGGL((spike_fwd_kernel<T, VW, N, WAVES, WORDS>), grid, dim3(WAVES *kWave), lds, st, spike_bits, stride, n_neurons *batch, by_batch, p.trials, \
                       p.trial_tiles, (const T *)weight, dim, p.slice_words, (T *)y, part)
#define BMTK_FWD(VW, N, WAVES)                                                   \
    do {                                                                         \
        if (p.words_per_lane == 1) BMTK_FWD_W(VW, N, WAVES, 1);                  \
        else BMTK_FWD_W(VW, N, WAVES, kWordsPerLane);                            \
    } while (0)
    BMTK_BY_TYPE(dtype, T, {
        if (p.waves == kOneBlockWaves) {
            if (p.vw == 1) BMTK_FWD(1, 1, kOneBlockWaves);
            else if (p.vw == 2) BMTK_FWD(2, 1, kOneBlockWaves);
            else BMTK_FWD(4, 1, kOneBlockWaves);
        } else if (batch == 1) {
            if (p.vw == 1) BMTK_FWD(1, 1, kManyWaves);
            else if (p.vw == 2) BMTK_FWD(2, 1, kManyWaves);
            else BMTK_FWD(4, 1, kManyWaves);
        } else {
            if (p.vw == 1) BMTK_FWD(1, 32, kManyWaves);
            else if (p.vw == 2) BMTK_FWD(2, 16, kManyWaves);
            else BMTK_FWD(4, 8, kManyWaves);
        }
        if (part)
            hipLaunchKernelGGL((spike_join_kernel<T>), dim3((unsigned)div_up(plane, kBlock)), dim3(kBlock), 0, st, part, (int)p.slices, plane, (T *)y);
    });
#undef BMTK_FWD
#undef BMTK_FWD_W
    BMTK_CHECK_LAUNCH("spike_readout_fwd");
    return BMTK_OK;
}

extern "C" int bmtk_spike_readout_bwd_weight(const uint64_t *spike_bits, int64_t stride, int64_t n_steps, int64_t n_neurons, int32_t batch, const void *dy,
                                             int32_t dim, int32_t dtype, void *d_weight, void *stream)
{
    BMTK_REQUIRE(spike_bits && dy && d_weight, "spike_readout_bwd_weight: pointers must be non-null");
    int rc = check_sizes("spike_readout_bwd_weight", n_steps, n_neurons, batch, dim, dtype);
    if (rc != BMTK_OK) return rc;
    BMTK_REQUIRE(stride >= (n_neurons * batch + 63) / 64, "spike_readout_bwd_weight: stride is shorter than a step's words");
    int vw = lane_channels(dim, dtype, dy);
    while (vw > 1 && !aligned(d_weight, vw * type_size(dtype))) vw /= 2;
    // neurons of a wavefront: 256 bits of a step where there are enough of them to fill the chip
    int64_t own = div_up(256, batch);
    const int64_t fill = n_neurons / 2048 < 1 ? 1 : n_neurons / 2048;
    if (own > fill) own = fill;
    if (own > kSums / vw) own = kSums / vw;
    BMTK_REQUIRE(div_up(n_neurons, kWaves * own) * kWaves * kWave < (1ll << 32), "spike_readout_bwd_weight: too many neurons");
    const dim3 grid((unsigned)div_up(n_neurons, kWaves * own), (unsigned)div_up(dim, kWave * vw));
    const hipStream_t st = (hipStream_t)stream;
    const FastDiv by_batch = fast_div((uint32_t)batch);
#define BMTK_BWD(VW, N)                                                                                                                       \
    hipLaunchKernelGGL((spike_bwd_weight_kernel<T, VW, N>), grid, dim3(kWaves *kWave), 0, st, spike_bits, stride, n_steps, n_neurons, by_batch, \
                       (int)own, (const T *)dy, dim, (T *)d_weight)
    BMTK_BY_TYPE(dtype, T, {
        if (own == 1) {
            if (vw == 1) BMTK_BWD(1, 1);
            else if (vw == 2) BMTK_BWD(2, 1);
            else BMTK_BWD(4, 1);
        } else {
            if (vw == 1) BMTK_BWD(1, 32);
            else if (vw == 2) BMTK_BWD(2, 16);
            else BMTK_BWD(4, 8);
        }
    });
#undef BMTK_BWD
    BMTK_CHECK_LAUNCH("spike_readout_bwd_weight");
    return BMTK_OK;
}

extern "C" int bmtk_spike_readout_bwd_spikes(const void *weight, const void *dy, int64_t n_steps, int64_t n_neurons, int32_t batch, int32_t dim, int32_t dtype,
                                             float *dl_dz, int32_t *workspace, void *stream)
{
    BMTK_REQUIRE(weight && dy && dl_dz, "spike_readout_bwd_spikes: pointers must be non-null");
    int rc = check_sizes("spike_readout_bwd_spikes", n_steps, n_neurons, batch, dim, dtype);
    if (rc != BMTK_OK) return rc;
    const DzPlan p = dz_plan(n_steps, n_neurons, batch, dim);
    BMTK_REQUIRE(dtype != BMTK_F32 || p.whole || workspace, "spike_readout_bwd_spikes: needs its workspace");
    const int64_t rows = n_steps * batch;
    const dim3 grid((unsigned)p.across, (unsigned)p.down);
    const int vl = 16 / (int)type_size(dtype);   // 16 bytes a load
    const bool wide = dim % vl == 0 && aligned(weight, 16) && aligned(dy, 16), any = dim >= vl;
    const hipStream_t st = (hipStream_t)stream;
    const FastDiv by_batch = fast_div((uint32_t)batch);
    // (a tile's pairs are whole steps, or 32 trials of one)
    const bool turned = (batch % 32 == 0 || batch == 4 || batch == 8 || batch == 16) && aligned(dl_dz, 128) && n_neurons * batch % 32 == 0;
    const bool steps = batch < kDzRows && !p.whole && dim <= kDzK && p.tile_rows % batch == 0, four = batch % 4 == 0 && aligned(dl_dz, 16);
#define BMTK_DZ(O, VL, OUT, ONE)                                                                                                                       \
    hipLaunchKernelGGL((spike_bwd_spikes_kernel<T, O, VL, OUT, ONE>), grid, dim3(kDzWaves *kWave), 0, st, (const T *)weight, (const T *)dy, rows, n_neurons, \
                       by_batch, dim, p.per_block, workspace, dl_dz)
#define BMTK_DZ_OUT(O, VL, ONE)                                 \
    do {                                                     \
        if (batch == 1) BMTK_DZ(O, VL, kAcross, ONE);           \
        else if (!turned) BMTK_DZ(O, VL, kPairs, ONE);          \
        else if (batch == 4) BMTK_DZ(O, VL, kTurned, ONE);      \
        else if (batch == 8) BMTK_DZ(O, VL, kTurned + 1, ONE);  \
        else if (batch == 16) BMTK_DZ(O, VL, kTurned + 2, ONE); \
        else BMTK_DZ(O, VL, kTurned + 3, ONE);                  \
    } while (0)
#define BMTK_DZ_BY(O, VL)                            \
    do {                                             \
        if (dim <= kDzK) BMTK_DZ_OUT(O, VL, true);   \
        else BMTK_DZ_OUT(O, VL, false);              \
    } while (0)
#define BMTK_DZ_STEPS(O, VL)                                          \
    do {                                                              \
        if (turned || !steps || batch == 1) BMTK_DZ_BY(O, VL);        \
        else if (four) BMTK_DZ(O, VL, kSteps4, true);                 \
        else BMTK_DZ(O, VL, kSteps1, true);                           \
    } while (0)
    if (dtype == BMTK_F32 && p.whole) {
        typedef float T;
        if (wide) BMTK_DZ_BY(Whole, 4);
        else if (any) BMTK_DZ_BY(Whole, kAny);
        else BMTK_DZ_BY(Whole, 1);
    } else {
        BMTK_BY_TYPE(dtype, T, {
            if (wide) BMTK_DZ_STEPS(T, 16 / sizeof(T));
            else if (any) BMTK_DZ_STEPS(T, kAny);
            else BMTK_DZ_STEPS(T, 1);
        });
    }
    if (dtype == BMTK_F32 && !p.whole)
        hipLaunchKernelGGL(spike_bwd_spikes_again_kernel, dim3((unsigned)p.parts), dim3(kBlock), 0, st, (const float *)weight, (const float *)dy, rows, n_neurons,
                           by_batch, dim, p.per_block, (int)p.across, workspace, dl_dz);
#undef BMTK_DZ_STEPS
#undef BMTK_DZ_BY
#undef BMTK_DZ_OUT
#undef BMTK_DZ
    BMTK_CHECK_LAUNCH("spike_readout_bwd_spikes");
    return BMTK_OK;
}
