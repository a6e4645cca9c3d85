// Log probabilities of given tokens, the entropy and the most probable alternatives of each row, and the gradient by the logits.
#include <math.h>

#include "readout.hpp"

namespace bmtk {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// Sums over a part of a row: maximum m (NaN where there is one), s = sum of e^(x - m), u = sum of (x - m) e^(x - m).  Then the logarithm of the
// whole sum is m + log s and the entropy log s - u / s: no term of it is below zero, so nothing cancels.
struct Sums {
    float m, s, u;
};

// maximum with NaN as the largest value
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// x - m, at least -200: e^-200 is 0 in fp32 and a product with it too, also where the difference is -inf, or none (-inf less -inf, or anything less NaN).
// The difference first, then the factor of the exponent, so that logits at the end of the type's range stay in it.
__device__ __forceinline__ float below(float x, float m) { return __builtin_fmaxf(x - m, -200.0f); }
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// a part's sums under the maximum m of several
__device__ __forceinline__ void raise_to(Sums &q, float m)
{
    const float d = below(q.m, m), e = exp_of(d);
    q.u = __builtin_fmaf(d, q.s, q.u) * e;
    q.s *= e;
    q.m = m;
}
// what two parts are together
__device__ __forceinline__ Sums join(Sums a, Sums b)
{
    const float m = max_nan(a.m, b.m);
    raise_to(a, m);
    raise_to(b, m);
    return Sums{m, a.s + b.s, a.u + b.u};
}
// log probability of a logit.  (A row with NaN or +inf has none.)
__device__ __forceinline__ float logp_of(const Sums &q, float x)
{
    if (!(q.m < INFINITY)) return NAN;
    return x == -INFINITY ? -INFINITY : (x - q.m) - logf(q.s);
}

// Order of the alternatives: the larger logit first (NaN before all), of equal ones the lower index.  One whole number for both;
// 0 is below every real one.
__device__ __forceinline__ uint64_t rank_of(float x, uint32_t index)
{
    uint32_t b = __float_as_uint(x + 0.0f);   // (-0 is 0)
    if (x != x) b = 0x7fffffffu;
    b = (int32_t)b < 0 ? ~b : b | 0x80000000u;
    return ((uint64_t)b << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t index_of(uint64_t rank) { return ~(uint32_t)rank; }
__device__ __forceinline__ float logit_of(uint64_t rank)
{
    const uint32_t b = (uint32_t)(rank >> 32);
    return __uint_as_float((int32_t)b < 0 ? b & 0x7fffffffu : ~b);
}

// The value of lane (lane ^ M), by moves within the vector unit: through LDS a sort of 64 lanes waits for 21 round trips (2.5 against 0.5 us).
// All lanes have to be active.
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v)
{
#define BMTK_MOVED(x, ctrl) ((uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x), (ctrl), 0xF, 0xF, true))
    if (M == 1) return BMTK_MOVED(v, 0xB1);                       // quad_perm 1, 0, 3, 2
    if (M == 2) return BMTK_MOVED(v, 0x4E);                       // quad_perm 2, 3, 0, 1
    if (M == 4) return BMTK_MOVED(BMTK_MOVED(v, 0x141), 0x1B);    // row_half_mirror (^ 7), then quad_perm 3, 2, 1, 0 (^ 3)
    if (M == 8) return BMTK_MOVED(v, 0x128);                      // row_ror 8
    if (M == 15) return BMTK_MOVED(v, 0x140);                     // row_mirror
    const auto r = M == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (lane_id() & M) ? r[0] : r[1];
#undef BMTK_MOVED
}
template <int M>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v)
{
    return ((uint64_t)lane_xor<M>((uint32_t)(v >> 32)) << 32) | lane_xor<M>((uint32_t)v);
}
template <int M>
__device__ __forceinline__ float lane_xor(float v)
{
    return __uint_as_float(lane_xor<M>(__float_as_uint(v)));
}

// one comparison of a sorting network over lanes: the lane keeps the larger of its own and its partner's, or the smaller
template <int M>
__device__ __forceinline__ uint64_t exchange(uint64_t v, bool larger)
{
    const uint64_t o = lane_xor<M>(v);
    return (o > v) == larger ? o : v;
}
// lanes of each group of 2 M, bitonic, the largest first where `falling`
template <int M>
__device__ __forceinline__ uint64_t settle(uint64_t v, bool falling)
{
    v = exchange<M>(v, ((lane_id() & M) == 0) == falling);
    if constexpr (M > 1) v = settle<M / 2>(v, falling);
    return v;
}
// lanes of each group of W sorted, the largest first
template <int W, int K = 2>
__device__ __forceinline__ uint64_t sort_lanes(uint64_t v)
{
    v = settle<K / 2>(v, K == W || (lane_id() & K) == 0);
    if constexpr (K < W) v = sort_lanes<W, K * 2>(v);
    return v;
}
// the 64 largest of two sorted lists, sorted: the larger of each pair (l, 63 - l) are those, and are bitonic
__device__ __forceinline__ uint64_t merge_lanes(uint64_t a, uint64_t b)
{
    const uint64_t o = lane_xor<32>(lane_xor<16>(lane_xor<15>(b)));
    return settle<kWave / 2>(a > o ? a : o, true);
}

template <int M>
__device__ __forceinline__ float max_lanes(float v)
{
    v = max_nan(v, lane_xor<M>(v));
    if constexpr (M > 1) v = max_lanes<M / 2>(v);
    return v;
}
template <int M>
__device__ __forceinline__ float sum_lanes(float v)
{
    v += lane_xor<M>(v);
    if constexpr (M > 1) v = sum_lanes<M / 2>(v);
    return v;
}
// the lanes of each group of W together
template <int W>
__device__ __forceinline__ Sums join_lanes(Sums a)
{
    raise_to(a, max_lanes<W / 2>(a.m));
    return Sums{a.m, sum_lanes<W / 2>(a.s), sum_lanes<W / 2>(a.u)};
}

struct Row {
    const void *logits;
    const int64_t *tokens;
    int64_t rows, row_stride;
    int32_t vocab, top;
    int64_t ignore;
    float *logp, *entropy, *lse, *top_logp;
    int64_t *top_index;
};

// what is written of a row, by one lane: its token's logit is read again
template <typename T>
__device__ __forceinline__ void write_row(const Row &a, int64_t r, const Sums &q)
{
    const int64_t token = a.tokens[r];
    float lp = 0.0f;
    if (token != a.ignore) {
        lp = NAN;   // a token outside the vocabulary
        if (token >= 0 && token < a.vocab) lp = logp_of(q, (float)static_cast<const T *>(a.logits)[r * a.row_stride + token]);
    }
    a.logp[r] = lp;
    const bool none = q.m == -INFINITY, odd = !(q.m < INFINITY);
    a.lse[r] = odd ? NAN : none ? -INFINITY : q.m + logf(q.s);
    a.entropy[r] = odd ? NAN : none ? 0.0f : logf(q.s) - q.u / q.s;
}

__device__ __forceinline__ void write_top(const Row &a, int64_t r, const Sums &q, int k, uint64_t rank)
{
    a.top_index[r * a.top + k] = (int64_t)index_of(rank);
    a.top_logp[r * a.top + k] = logp_of(q, logit_of(rank));
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows of up to 64 logits: W lanes each, one logit a lane (19,200 x 10 fp32, top 2: 4.2 us, of which a launch is half)
template <typename T, int W>
__global__ void __launch_bounds__(kBlock) logprobs_short_kernel(const Row a)
{
    const int l = lane_id() & (W - 1);
    const int64_t r = (int64_t)blockIdx.x * (kBlock / W) + threadIdx.x / W;
    const bool in = r < a.rows && l < a.vocab;
    const float x = in ? (float)static_cast<const T *>(a.logits)[r * a.row_stride + l] : -INFINITY;
    Sums q{x, x == -INFINITY ? 0.0f : 1.0f, 0.0f};   // (a row with NaN or +inf: by its maximum)
    q = join_lanes<W>(q);
    if (r < a.rows && l == 0) write_row<T>(a, r, q);
    if (a.top > 0) {
        const uint64_t v = sort_lanes<W>(in ? rank_of(x, l) : 0);
        if (r < a.rows && l < a.top) write_top(a, r, q, l, v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Longer rows: a workgroup takes a row, or a slice of one, in one pass, bound by reading it: 8,192 x 131,072 bf16, top 5, 2.15 GB in 437 us at the median, 399
// at best (4.9 to 5.4 TB/s, what this card reads at).  4,096 x 50,021 bf16 behind a backward pass 113 us, and 106 with all arithmetic left out.

// A wavefront's alternatives: the 64 best so far, sorted, one a lane, and a queue of those that may be among them.  A logit is
// compared with the last that counts; what passes waits until 64 do, which are sorted and merged in at once.
struct Alternatives {
    uint64_t best;
    uint64_t last;       // the last of the best `top`
    float least;         // its logit
    unsigned waiting;
    uint64_t *queue;     // 128 places in LDS

    __device__ __forceinline__ void start(uint64_t *q) { best = last = 0, least = -INFINITY, waiting = 0, queue = q; }
    // What the first N logits of every lane say before any is looked at: the best of each lane are 64 logits, so none below the last that counts of
    // those does.  (Looked at one by one they are all taken, four sorts instead of one.)
    template <int N>
    __device__ __forceinline__ void prime(const float (&x)[N], uint32_t index, int top)
    {
        uint64_t rank = rank_of(x[0], index);
#pragma unroll
        for (int k = 1; k < N; ++k) {
            const uint64_t r = rank_of(x[k], index + k);
            rank = r > rank ? r : rank;
        }
        rank = bcast_u64(sort_lanes<kWave>(rank), top - 1);
        last = rank - 1;   // (which it passes itself)
        least = logit_of(rank);
    }
    __device__ __forceinline__ void take(int top)
    {
        const int l = lane_id();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const unsigned n = waiting < kWave ? waiting : kWave;
        // (the last ones, so that the rest stays where it is)
        const uint64_t v = (unsigned)l < n ? queue[waiting - n + l] : 0;
        waiting -= n;
        best = merge_lanes(best, sort_lanes<kWave>(v));
        const uint64_t now = bcast_u64(best, top - 1);
        if (now > last) last = now, least = logit_of(now);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void look(float x, uint32_t index, bool in, int top)
    {
        const uint64_t rank = rank_of(x, index);
        const bool may = in && rank > last;
        const uint64_t mask = __ballot(may);
        if (mask == 0) return;
        if (may) queue[waiting + lane_prefix(mask)] = rank;
        waiting += (unsigned)__popcll(mask);
        __builtin_amdgcn_wave_barrier();
        if (waiting >= kWave) take(top);
    }
};

template <int N, bool kTop>
__device__ __forceinline__ void take_logits(Sums &q, Alternatives &alt, const float (&x)[N], uint32_t index, bool in, int top)
{
    float m = x[0];
#pragma unroll
    for (int k = 1; k < N; ++k) m = max_nan(m, x[k]);
    if (!(m <= q.m)) raise_to(q, max_nan(q.m, m));
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float d = below(x[k], q.m), e = exp_of(d);
        q.s += e;
        q.u = __builtin_fmaf(d, e, q.u);
    }
    // (equal ones are looked at, and a NaN, which comes before all)
    if (kTop && __ballot(!(m < alt.least)) != 0)
#pragma unroll
        for (int k = 0; k < N; ++k) alt.look(x[k], index + k, in, top);
}

struct Slices {
    int32_t count;
    int32_t length;      // logits of a slice
    float *sums;         // [rows][count][3]
    uint64_t *best;      // [rows][count][top]
};

template <typename T, int kWaves, bool kTop>
__global__ void __launch_bounds__(kWaves * kWave) logprobs_kernel(const Row a, const Slices sl)
{
    constexpr int N = 16 / sizeof(T);
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint64_t queues[kTop ? kWaves : 1][2 * kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int64_t r = blockIdx.x;
    const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
    const int begin = (int)blockIdx.y * sl.length, end = min(a.vocab, begin + sl.length);
    Sums q{-INFINITY, 0.0f, 0.0f};
    Alternatives alt;
    if (kTop) alt.start(queues[wave]);

    // 16 bytes a lane and load from the first address that allows it; what lies before and behind, logit by logit
    const int odd = (int)((reinterpret_cast<uintptr_t>(row + begin) & 15) / sizeof(T));
    const int body = min(end, begin + (odd ? N - odd : 0));
    const int packs = (end - body) / N, tail = body + packs * N;
    // (lanes beyond take -inf, which adds nothing)
    if (wave == 0) {
        const int at = lane < body - begin ? begin + lane : tail + lane - (body - begin);
        const bool in = at < end;
        const float x[1] = {in ? (float)row[at] : -INFINITY};
        take_logits<1, kTop>(q, alt, x, (uint32_t)at, in, a.top);
    }
    // whole loads of the wavefront, the next two on their way while two are worked on; then what is left
    const T *mine = row + body + lane * N;
    auto take = [&](const Pack<T, N> &v, int p, bool in, bool all) {
        float x[N];
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = (float)v.v[k];
        if (!all)
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = in ? x[k] : -INFINITY;
        take_logits<N, kTop>(q, alt, x, (uint32_t)(body + (p + lane) * N), in, a.top);
    };
    constexpr int kStep = kWaves * kWave;
    int p = wave * kWave;
    if (p + kStep + kWave <= packs) {
        Pack<T, N> v[2], w[2];
        auto load = [&](Pack<T, N>(&u)[2], int at) {
#pragma unroll
            for (int k = 0; k < 2; ++k) u[k] = *reinterpret_cast<const Pack<T, N> *>(mine + min(at + k * kStep, packs - kWave) * N);
        };
        load(v, p);
        if (kTop) {
            float x[N];
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = (float)v[0].v[k];
            alt.prime(x, (uint32_t)(body + (p + lane) * N), a.top);
        }
        for (;;) {
            load(w, p + 2 * kStep);
            take(v[0], p, true, true);
            take(v[1], p + kStep, true, true);
            p += 2 * kStep;
            if (p + kStep + kWave > packs) break;
            load(v, p + 2 * kStep);
            take(w[0], p, true, true);
            take(w[1], p + kStep, true, true);
            p += 2 * kStep;
            if (p + kStep + kWave > packs) break;
        }
    }
    for (; p < packs; p += kStep) {
        const bool in = p + lane < packs;
        take(*reinterpret_cast<const Pack<T, N> *>(row + body + min(p + lane, packs - 1) * N), p, in, false);
    }
    if (kTop)
        while (alt.waiting) alt.take(a.top);
    q = join_lanes<kWave>(q);
    if (kWaves > 1) {
        if (lane == 0) wave_sums[wave] = q;
        if (kTop) queues[wave][lane] = alt.best;
        __syncthreads();
        if (wave != 0) return;
        for (int w = 1; w < kWaves; ++w) {
            q = join(q, wave_sums[w]);
            if (kTop) alt.best = merge_lanes(alt.best, queues[w][lane]);
        }
    }
    if (sl.count > 1) {
        const int64_t at = r * sl.count + blockIdx.y;
        if (lane == 0) sl.sums[at * 3] = q.m, sl.sums[at * 3 + 1] = q.s, sl.sums[at * 3 + 2] = q.u;
        if (kTop && lane < a.top) sl.best[at * a.top + lane] = alt.best;
        return;
    }
    if (lane == 0) write_row<T>(a, r, q);
    if (kTop && lane < a.top) write_top(a, r, q, lane, alt.best);
}

// The slices of a row together: a wavefront takes every sixteenth, the sixteen lists are merged pair by pair
constexpr int kJoinWaves = 16;
template <typename T, bool kTop>
__global__ void __launch_bounds__(kJoinWaves * kWave) logprobs_join_kernel(const Row a, const Slices sl)
{
    __shared__ uint64_t lists[kTop ? kJoinWaves : 1][kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), waves = blockDim.x / kWave;
    const int64_t r = blockIdx.x;
    uint64_t best = 0;
    if (kTop) {
        for (int k = wave; k < sl.count; k += waves) best = merge_lanes(best, lane < a.top ? sl.best[(r * sl.count + k) * a.top + lane] : 0);
        for (int half = waves / 2; half > 0; half /= 2) {
            if (wave >= half && wave < 2 * half) lists[wave][lane] = best;
            __syncthreads();
            if (wave < half) best = merge_lanes(best, lists[wave + half][lane]);
        }
    }
    if (wave != 0) return;
    Sums q{-INFINITY, 0.0f, 0.0f};
    for (int k = lane; k < sl.count; k += kWave) {
        const float *p = sl.sums + (r * sl.count + k) * 3;
        q = join(q, Sums{p[0], p[1], p[2]});
    }
    q = join_lanes<kWave>(q);
    if (lane == 0) write_row<T>(a, r, q);
    if (kTop && lane < a.top) write_top(a, r, q, lane, best);
}

// ---------------------------------------------------------------------------------------------------------------------
// Backward: with p = e^(x - lse), log probability l = x - lse and entropy H,
//   d x_j = d_logp (delta_j,token - p_j) - d_entropy p_j (l_j + H)
// Bound by memory: 4,096 x 50,021 bf16 152 us (820 MB, 5.4 TB/s).
//
// lse is what 32 bits hold of it, off by up to half a step, and p by as much of itself: 2^-18 where lse is just below kFar, everything where
// the logits are the type's lowest value (a mask that leaves nothing; lse is that value too, log vocab lies far below its steps).  Of
// such a row e^(x - lse) is added up first, and the logarithm of that sum, the `rest` of lse, taken off every l_j.  One workgroup (of short rows: wavefront)
// does so, also of rows that are otherwise several ones': in place, the others would overwrite what it reads.  4,096 x 50,021 bf16 far from zero 240 us, near it
// 175; 4 x 131,072 42 and 4.2; 19,200 x 10 fp32 7.1 and 4.2.
constexpr float kFar = 64.0f;
struct RowBwd {
    const void *logits;
    void *d_logits;
    const int64_t *tokens;
    const float *lse, *entropy, *d_logp, *d_entropy;
    int64_t rows, row_stride, out_stride;
    int32_t vocab;
    int64_t ignore;
};
struct Factors {
    float lse, rest, by_logp, by_entropy, entropy;
    int64_t token;
    bool none;   // a row without a token whose entropy nobody asks about: nothing, whatever its logits are
};
__device__ __forceinline__ Factors factors_of(const RowBwd &a, int64_t r)
{
    Factors f;
    f.lse = a.lse[r];
    f.rest = 0.0f;
    f.entropy = a.entropy[r];
    f.token = a.tokens[r];
    f.by_logp = f.token == a.ignore ? 0.0f : a.d_logp ? a.d_logp[r] : 0.0f;
    f.by_entropy = a.d_entropy ? a.d_entropy[r] : 0.0f;
    if (f.token != a.ignore && (f.token < 0 || f.token >= a.vocab)) f.by_logp = NAN;   // as its log probability is
    f.none = f.token == a.ignore && f.by_entropy == 0.0f;
    if (f.lse == -INFINITY) f.lse = f.by_logp = f.by_entropy = 0.0f;                      // a row of nothing but -inf: nothing moves it
    return f;
}
__device__ __forceinline__ float gradient(const Factors &f, float x, int j)
{
    const float l = (x - f.lse) - f.rest, p = __builtin_amdgcn_exp2f(l * kLog2e);
    float d = -(p * f.by_logp);
    if (p != 0.0f) d -= p * f.by_entropy * (l + f.entropy);   // (of a logit of -inf there is nothing)
    if (f.none) return 0.0f;
    return j == f.token ? d + f.by_logp : d;
}

__device__ __forceinline__ bool is_far(const Factors &f) { return !f.none && __builtin_fabsf(f.lse) >= kFar; }
// a lane's part of the sum of e^(x - lse); lse is the largest logit at least, rounded as it is, so no term is above 1
template <typename T>
__device__ __forceinline__ float far_sum(const T *row, float lse, int vocab, int first, int by)
{
    float s = 0.0f;
#pragma unroll 8
    for (int j = first; j < vocab; j += by) s += exp_of((float)row[j] - lse);
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kBlock) logprobs_bwd_kernel(const RowBwd a, int length, bool together)
{
    constexpr int N = 16 / sizeof(T);
    const int64_t r = blockIdx.x;
    const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
    T *out = static_cast<T *>(a.d_logits) + r * a.out_stride;
    const int begin = (int)blockIdx.y * length;
    int end = min(a.vocab, begin + length);
    Factors f = factors_of(a, r);
    if (is_far(f)) {
        __shared__ float sums[kBlock / kWave];
        if (begin > 0) return;
        end = a.vocab;
        const float s = sum_lanes<kWave / 2>(far_sum(row, f.lse, a.vocab, threadIdx.x, kBlock));
        if (lane_id() == 0) sums[threadIdx.x / kWave] = s;
        __syncthreads();
        float all = 0.0f;
        for (int w = 0; w < kBlock / kWave; ++w) all += sums[w];
        f.rest = logf(all);
    }
    const int odd = (int)((reinterpret_cast<uintptr_t>(row + begin) & 15) / sizeof(T));
    const int body = !together ? end : min(end, begin + (odd ? N - odd : 0));
    const int packs = (end - body) / N, tail = body + packs * N;
    for (int p = threadIdx.x; p < packs; p += kBlock) {
        Pack<T, N> v = *reinterpret_cast<const Pack<T, N> *>(row + body + p * N);
#pragma unroll
        for (int k = 0; k < N; ++k) v.v[k] = (T)gradient(f, (float)v.v[k], body + p * N + k);
        *reinterpret_cast<Pack<T, N> *>(out + body + p * N) = v;
    }
    const int apart = (body - begin) + (end - tail);
    for (int k = threadIdx.x; k < apart; k += kBlock) {
        const int at = k < body - begin ? begin + k : tail + k - (body - begin);
        out[at] = (T)gradient(f, (float)row[at], at);
    }
}

// short rows: logit by logit
template <typename T>
__global__ void __launch_bounds__(kBlock) logprobs_bwd_short_kernel(const RowBwd a, FastDiv by_vocab)
{
    // a workgroup takes as many rows as it has threads for, or one
    const int64_t block_rows = kBlock > a.vocab ? kBlock / a.vocab : 1;
    const int64_t r0 = (int64_t)blockIdx.x * block_rows;
    const int all = (int)min(block_rows, a.rows - r0) * a.vocab;
    for (int first = 0; first < all; first += kBlock) {
        const int c = first + threadIdx.x;
        bool begins = false;   // a far row
        int64_t r = 0;
        if (c < all) {
            const int k = (int)div_by((uint32_t)c, by_vocab), j = c - k * a.vocab;
            r = r0 + k;
            float x = (float)static_cast<const T *>(a.logits)[r * a.row_stride + j];
            const Factors f = factors_of(a, r);
            asm volatile("" : "+v"(x));   // (asked for before it is known whether the row is far: 19,200 x 500 fp32 25.6 us, 32 otherwise)
            if (!is_far(f)) static_cast<T *>(a.d_logits)[r * a.out_stride + j] = (T)gradient(f, x, j);
            else begins = j == 0;
        }
        // far rows: by the wavefront where they begin, and nobody else
        for (uint64_t left = __ballot(begins); left != 0; left &= left - 1) {
            const int64_t far = (int64_t)bcast_u64((uint64_t)r, __builtin_ctzll(left));
            const T *row = static_cast<const T *>(a.logits) + far * a.row_stride;
            Factors f = factors_of(a, far);
            f.rest = logf(sum_lanes<kWave / 2>(far_sum(row, f.lse, a.vocab, lane_id(), kWave)));
            for (int j = lane_id(); j < a.vocab; j += kWave) static_cast<T *>(a.d_logits)[far * a.out_stride + j] = (T)gradient(f, (float)row[j], j);
        }
    }
}

// Slices of a row: enough workgroups to fill the chip, but no more than one for every two loads a lane (begun ones too: 4,097 bf16 are two slices; 4 x 131,072, top 20, both launches: four 15.8 us, two 14.2, one 15.0)
void slices_of(int64_t rows, int32_t vocab, int32_t dtype, Slices &sl)
{
    const int64_t unit = 2 * kBlock * (16 / (int64_t)type_size(dtype));
    int64_t s = 768 / rows, most = div_up(vocab, unit);
    if (s > most) s = most;
    if (s < 1) s = 1;
    sl.length = (int32_t)(div_up(div_up(vocab, s), 64) * 64);
    sl.count = (int32_t)div_up(vocab, sl.length);
}

int check_logprobs(const char *who, int64_t rows, int32_t vocab, int32_t dtype, int32_t top)
{
    BMTK_REQUIRE(rows > 0 && vocab > 0, "%s: sizes must be positive", who);
    BMTK_REQUIRE(rows < (1ll << 24) && vocab < (1 << 30), "%s: rows must stay below 2^24 and vocab below 2^30", who);
    BMTK_REQUIRE(dtype == BMTK_F32 || dtype == BMTK_BF16 || dtype == BMTK_F16, "%s: unknown type %d", who, dtype);
    BMTK_REQUIRE(top >= 0 && top <= BMTK_LOGPROBS_MAX_TOP && top <= vocab, "%s: top must lie in 0..min(%d, vocab)", who, BMTK_LOGPROBS_MAX_TOP);
    return BMTK_OK;
}

constexpr int kShort = 64;       // a logit a lane
constexpr int kOneWave = 2048;   // rows up to this length: a wavefront each

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_token_logprobs_workspace_bytes(int64_t rows, int32_t vocab, int32_t dtype, int32_t top)
{
    if (check_logprobs("token_logprobs_workspace_bytes", rows, vocab, dtype, top) != BMTK_OK || vocab <= kOneWave) return 0;
    Slices sl{};
    slices_of(rows, vocab, dtype, sl);
    return sl.count > 1 ? rows * sl.count * (int64_t)(top * sizeof(uint64_t) + 3 * sizeof(float)) : 0;
}

extern "C" int bmtk_token_logprobs_fwd(int64_t rows, int32_t vocab, int32_t dtype, const void *logits, int64_t row_stride, const int64_t *tokens,
                                       int64_t ignore, int32_t top, float *logp, float *entropy, float *lse, float *top_logp, int64_t *top_index,
                                       void *workspace, void *stream)
{
    BMTK_REQUIRE(logits && tokens && logp && entropy && lse, "token_logprobs_fwd: pointers must be non-null");
    const int rc = check_logprobs("token_logprobs_fwd", rows, vocab, dtype, top);
    if (rc != BMTK_OK) return rc;
    BMTK_REQUIRE(top == 0 || (top_logp && top_index), "token_logprobs_fwd: the alternatives have nowhere to go");
    Row a{logits, tokens, rows, row_stride, vocab, top, ignore, logp, entropy, lse, top_logp, top_index};
    const hipStream_t st = (hipStream_t)stream;
    if (vocab <= kShort) {
#define BMTK_SHORT(W) hipLaunchKernelGGL((logprobs_short_kernel<T, W>), dim3((unsigned)div_up(rows, kBlock / W)), dim3(kBlock), 0, st, a)
        BMTK_BY_TYPE(dtype, T, {
            if (vocab <= 16) BMTK_SHORT(16);
            else BMTK_SHORT(64);
        });
#undef BMTK_SHORT
        BMTK_CHECK_LAUNCH("token_logprobs_fwd");
        return BMTK_OK;
    }
    Slices sl{1, vocab, nullptr, nullptr};
    if (vocab > kOneWave) slices_of(rows, vocab, dtype, sl);
    if (sl.count > 1) {
        BMTK_REQUIRE(workspace && aligned(workspace, 8), "token_logprobs_fwd: needs its workspace");
        sl.best = static_cast<uint64_t *>(workspace);
        sl.sums = reinterpret_cast<float *>(sl.best + rows * sl.count * (int64_t)top);
    }
    const dim3 grid((unsigned)rows, (unsigned)sl.count);
#define BMTK_ROWS(W, TOP) hipLaunchKernelGGL((logprobs_kernel<T, W, TOP>), grid, dim3(W *kWave), 0, st, a, sl)
    BMTK_BY_TYPE(dtype, T, {
        if (vocab <= kOneWave) {
            if (top) BMTK_ROWS(1, true);
            else BMTK_ROWS(1, false);
        } else {
            if (top) BMTK_ROWS(4, true);
            else BMTK_ROWS(4, false);
        }
        if (sl.count > 1) {
            // (a power of two of wavefronts, one for each slice as far as they go)
            int waves = 1;
            while (waves < kJoinWaves && waves < sl.count) waves *= 2;
            if (top) hipLaunchKernelGGL((logprobs_join_kernel<T, true>), dim3((unsigned)rows), dim3(waves * kWave), 0, st, a, sl);
            else hipLaunchKernelGGL((logprobs_join_kernel<T, false>), dim3((unsigned)rows), dim3(kWave), 0, st, a, sl);
        }
    });
#undef BMTK_ROWS
    BMTK_CHECK_LAUNCH("token_logprobs_fwd");
    return BMTK_OK;
}

extern "C" int bmtk_token_logprobs_bwd(int64_t rows, int32_t vocab, int32_t dtype, const void *logits, int64_t row_stride, const int64_t *tokens,
                                       int64_t ignore, const float *lse, const float *entropy, const float *d_logp, const float *d_entropy, void *d_logits,
                                       int64_t out_stride, void *stream)
{
    BMTK_REQUIRE(logits && tokens && lse && entropy && d_logits, "token_logprobs_bwd: pointers must be non-null");
    const int rc = check_logprobs("token_logprobs_bwd", rows, vocab, dtype, 0);
    if (rc != BMTK_OK) return rc;
    BMTK_REQUIRE(d_logp || d_entropy, "token_logprobs_bwd: no gradient to go on from");
    const RowBwd a{logits, d_logits, tokens, lse, entropy, d_logp, d_entropy, rows, row_stride, out_stride, vocab, ignore};
    const hipStream_t st = (hipStream_t)stream;
    const size_t size = type_size(dtype);
    // loads and stores of 16 bytes: both rows begin at the same place of such a piece
    const bool together = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(d_logits)) & 15) == 0 && (((row_stride - out_stride) * (int64_t)size) & 15) == 0;
    if (vocab < 512) {
        const FastDiv by_vocab = fast_div((uint32_t)vocab);
        BMTK_BY_TYPE(dtype, T, hipLaunchKernelGGL((logprobs_bwd_short_kernel<T>), dim3((unsigned)div_up(rows, vocab < kBlock ? kBlock / vocab : 1)), dim3(kBlock), 0, st, a, by_vocab));
    } else {
        Slices sl{};
        slices_of(rows, vocab, dtype, sl);
        const dim3 grid((unsigned)rows, (unsigned)sl.count);
        BMTK_BY_TYPE(dtype, T, hipLaunchKernelGGL((logprobs_bwd_kernel<T>), grid, dim3(kBlock), 0, st, a, sl.length, together));
    }
    BMTK_CHECK_LAUNCH("token_logprobs_bwd");
    return BMTK_OK;
}
