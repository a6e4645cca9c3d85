// Log probabilities of tokens under the softmax of x @ weight^T, and their gradients by x and weight, without the logits in memory.
//
// Forward: tiles of logits are made on the matrix cores and reduced where they are, to each row's maximum and sum over the tile's vocabulary;
// tiles are joined by a second kernel.  Backward: with p = e^logit / sum and d_logp = m size, size a power of two, G = m (p - delta), dx = -size G weight and d_weight =
// -(G^T (size x)): the logits are made again, a piece of the vocabulary at a time, G of the piece is written in 16 bits, and two more products read it.  All of that is one kernel,
// D[i][j] = sum_k A[i][k] B[j][k], whose operands lie in memory with k contiguous or with i (j) contiguous.
//
// fp32 operands are taken as three bf16 parts each (8 bits of mantissa a part, 24 in all), whose six largest products are added up: what is left out is below 2^-24
// of a term.
#include <type_traits>

#include "readout.hpp"

namespace bmtk {
namespace {

constexpr int kTile = 32;          // of a matrix instruction
constexpr int kDepth = 64;         // k of a step: 128 bytes a row
constexpr int kWaitReads = 0xc07f, kWaitLoads = 0x0f70, kWaitAll = 0x70;   // s_waitcnt of all LDS operations, of all loads, of both
constexpr int kSmallMost = 128;    // of a small vocabulary
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

typedef float Acc __attribute__((ext_vector_type(16)));
typedef float Acc4 __attribute__((ext_vector_type(4)));
template <typename E>
struct Vec;
template <>
struct Vec<bf16> {
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    typedef __bf16 V4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Acc mfma(V8 a, V8 b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc4 mfma16(V8 a, V8 b, Acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc4 mfma16(V4 a, V4 b, Acc4 c)
    {
        typedef short S4 __attribute__((ext_vector_type(4)));
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(S4, a), __builtin_bit_cast(S4, b), c, 0, 0, 0);
    }
};
template <>
struct Vec<f16> {
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    typedef _Float16 V4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Acc mfma(V8 a, V8 b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc4 mfma16(V8 a, V8 b, Acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc4 mfma16(V4 a, V4 b, Acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};

// what a type's products are made of
template <typename T>
struct Element {
    typedef T type;
};
template <>
struct Element<float> {
    typedef bf16 type;
};

// eight numbers from where they begin anywhere
template <typename T>
struct Loose8 {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    typedef Words Loose __attribute__((aligned(2)));
    union {
        Words w[sizeof(T) / 2];
        T v[8];
    };
    __device__ __forceinline__ Loose8() {}
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const Loose *>(p)[i];
    }
    __device__ __forceinline__ void load_some(const T *p, int n)   // n of them; 0 for the others
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.0f;
    }
};

// C numbers (two or four), `some` of them there, the others 0
template <typename T, int C>
struct LooseFew {
    typedef uint32_t Words __attribute__((ext_vector_type(C * sizeof(T) / 4)));
    typedef Words Loose __attribute__((aligned(2)));
    union {
        Words w;
        T v[C];
    };
    __device__ __forceinline__ LooseFew() {}
    __device__ __forceinline__ void load(const T *p, int some)
    {
        if (some >= C) {
            w = *reinterpret_cast<const Loose *>(p);
        } else {
#pragma unroll
            for (int q = 0; q < C; ++q) v[q] = q < some ? p[q] : (T)0.0f;
        }
    }
};

// three bf16 parts of v; of what is not finite the first is it (so that its products are not either), and a number that rounds to infinity is cut
__device__ __forceinline__ void split(float v, bf16 (&p)[3])
{
    p[0] = (bf16)v;
    if (fabsf((float)p[0]) == INFINITY) {
        const uint16_t top = (uint16_t)(__float_as_uint(v) >> 16);
        __builtin_memcpy(&p[0], &top, 2);
    }
    const float r = v - (float)p[0];
    const bool finite = fabsf(v) < INFINITY;
    p[1] = (bf16)(finite ? r : 0.0f);
    p[2] = (bf16)(finite ? r - (float)p[1] : 0.0f);
}
// of the products of parts, in this order: 0 0, 0 1, 1 0, 1 1, 0 2, 2 0
__device__ __forceinline__ int part_a(int combination) { return 0x201100 >> combination * 4 & 3; }
__device__ __forceinline__ int part_b(int combination) { return 0x021010 >> combination * 4 & 3; }

// Exponentials are of base 2, against a base that is a number of eighths near the largest logit times log2 e: it is exact, so that 2^(v log2e - base) is rounded
// in the exponent once, and what log2 e itself is off by is the same in the logit of a token.
__device__ __forceinline__ float base_of(float m) { return rintf(m * (kLog2e * 8.0f)) * 0.125f; }
__device__ __forceinline__ float exp_over(float v, float base) { return __builtin_amdgcn_exp2f(fmaf(v, kLog2e, -base)); }

// What a row's d_logp, over the largest of all rows, does to its gradient: it is m size with size a power of two.  m is in G, so that G is rounded once and x, times size, not at all;
// of a mean, with one d_logp for all rows, m is 1, and G of a row's token is next to -1, which rounding changes by p at most.  whole is the scale of G times m, by_total that over the
// row's sum.  All 0 for rows that have no part; a token outside the vocabulary, or logits that are NaN or +inf (whose sum is NaN), makes everything NaN, with a d_logp of 0 too.
__device__ __forceinline__ bool no_part(int64_t token, int64_t ignore, float peak, float total) { return token == ignore || (peak == -INFINITY && total == 0.0f); }
__device__ __forceinline__ bool undefined(int64_t token, int32_t vocab, float total) { return token < 0 || token >= vocab || total != total; }
struct Share {
    float size, by_total, whole;
    __device__ __forceinline__ Share(float d, int64_t token, int64_t ignore, int32_t vocab, float peak, float total, float g_scale)
    {
        size = by_total = whole = 0.0f;
        if (no_part(token, ignore, peak, total)) return;
        if (undefined(token, vocab, total)) d = NAN;
        if (d == 0.0f) return;
        const uint32_t exponent = __float_as_uint(d) & 0x7f800000u;
        size = exponent == 0x7f800000u ? 1.0f : __uint_as_float(exponent ? exponent : 0x00800000u);
        whole = g_scale * (d / size);
        by_total = whole / total;
    }
};

// fp16: x times size would be among the subnormals, or lost, where one row's d_logp is some 2^14 times another's.  reach is the largest |x| size of the call, and x size is kept times the power of
// two that takes that to 2^14 or more, below 2^15: what is rounded then is 2^-28 of the largest or less.  (Of bf16 and fp32, whose smallest numbers are far away, there is none.)
__device__ __forceinline__ float lift_of(const float *reach)
{
    if (!reach || !(*reach > 0.0f)) return 1.0f;
    return __uint_as_float((127u + 14u + 127u - (__float_as_uint(fmaxf(*reach, 0x1p-100f)) >> 23)) << 23);
}

__device__ __forceinline__ int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// bases and sums over them, joined; -inf: nothing yet
__device__ __forceinline__ float2 join(float2 u, float2 v)
{
    const float m = fmaxf(u.x, v.x), from = m == -INFINITY ? 0.0f : m;
    return make_float2(m, u.y * __builtin_amdgcn_exp2f(u.x - from) + v.y * __builtin_amdgcn_exp2f(v.x - from));
}

// the first `some` of C numbers (two or four) to where they begin anywhere
template <typename T, int C>
__device__ __forceinline__ void put(T *p, const float (&v)[C], int some)
{
    typedef uint32_t Words __attribute__((ext_vector_type(C * sizeof(T) / 4)));
    typedef Words Loose __attribute__((aligned(2)));
    T q[C];
#pragma unroll
    for (int r = 0; r < C; ++r) q[r] = (T)v[r];
    if (some >= C) {
        Words w;
        __builtin_memcpy(&w, q, sizeof(w));
        *reinterpret_cast<Loose *>(p) = w;
    } else {
#pragma unroll
        for (int r = 0; r < C - 1; ++r)
            if (r < some) p[r] = q[r];
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the product

enum { kStats = 0, kGradient = 1, kSlab = 2, kOut = 3 };

struct Source {
    const char *p;
    int64_t stride, part, step, total;   // bytes from row to row, from part to part, from step to step, of a part
    int64_t block;                       // of i (j) contiguous: bytes from 64 numbers of a row to the next 64
};

struct Product {
    Source a, b;
    int32_t ni, nj;                               // sizes
    int32_t tail;                                 // k of the last step that the rows have; what lies behind them is not theirs
    int32_t steps, combinations;                  // steps of kDepth in k; 1 or 6
    int32_t rotate;                               // whether the steps may be begun anywhere: all of them are taken, and none is cut
    int32_t tiles_i, tiles_j, slices;             // slices: parts of the steps, each to a slab of its own
    // kStats, kGradient: i is the vocabulary from first on, j the rows
    int32_t first, vocab;
    const int64_t *tokens;
    int64_t ignore;
    float2 *stats;                                // [tiles_i of all pieces][rows]: maximum, sum of e^(logit - maximum)
    float *label;                                 // [rows]: logit of the row's token
    const float *peak;
    const float2 *shares;                         // by_total and whole of each row's Share
    void *g;                                      // [parts][piece / 64][rows, to a whole tile][64]: a step's operands lie next to one another in both products that read it
    int64_t g_block, g_part;                      // in numbers
    // kSlab: [slices][nj][slab_stride]; kOut: [nj][ni] of T
    float *slab;
    int64_t slab_stride, slab_size;
    int32_t add;                                  // to what is in the slab
    void *out;
    const float *factor, *reach;                  // (one number each) kOut: results times this and out_scale, over lift_of the other
    float out_scale;
};

typedef __attribute__((address_space(3))) uint32_t LdsWord;

// One operand's tile of N rows (i or j) and kDepth k on its way through LDS, 16 bytes a lane straight from memory.
// LDS gives 256 bytes at a time.  Rows of 128 bytes, k contiguous: the 16 bytes c of row r lie at c ^ (r / 2 & 7), so that sixteen rows' same c are in different banks.
// Otherwise N * 2 bytes of a k: their 32 bytes s lie at s ^ 2 (k & 3), so that four rows' s and s ^ 1 are; fragments are transposed as they are read.
// Loads are of a buffer that ends with the operand: what a tile has beyond it is 0, and nothing outside is read.
template <typename E, int N, int Waves, bool KRows>
struct Operand {
    static constexpr int kBytes = N * kDepth * 2, kLoads = kBytes / 1024 / Waves;
    static constexpr int kLoadRows = KRows ? 512 / N : 8;                    // rows that a load of a wavefront takes
    static constexpr int kVary = KRows && kLoadRows != 2 ? 1 : 2;            // loads in a row that differ by their swizzle
    static_assert(kLoads >= 1 && kLoads % kVary == 0, "a load for every wavefront");
    typedef typename Vec<E>::V8 V8;
    uint32_t from[kVary];    // this lane's bytes of a wavefront's first loads
    uint32_t each;           // bytes from one load's rows to the next one's
    const char *at;          // what the tile begins with, at the step that is to be loaded
    int64_t left;            // bytes from there to the operand's end
    __device__ __forceinline__ void start(const Source &s, int32_t row0, int lane, int wave)
    {
        const int64_t skip = KRows ? row0 / 64 * s.block : row0 * s.stride;
        at = s.p + skip;
        left = s.total - skip;
        each = (uint32_t)(kLoadRows * s.stride);
#pragma unroll
        for (int n = 0; n < kVary; ++n) {
            if constexpr (!KRows) {
                const int row = (wave * kLoads + n) * kLoadRows + lane / 8;
                from[n] = (uint32_t)(row - n * kLoadRows) * (uint32_t)s.stride + (uint32_t)((lane & 7) ^ (row / 2 & 7)) * 16;
            } else {
                constexpr int kChunks = N / 8;   // of 16 bytes in a row
                const int k = (wave * kLoads + n) * kLoadRows + lane / kChunks, byte = ((lane % kChunks) ^ ((k & 3) * 4)) * 16;
                from[n] = (uint32_t)(k - n * kLoadRows) * (uint32_t)s.stride + (uint32_t)(byte / 128) * (uint32_t)s.block + (uint32_t)(byte % 128);
            }
        }
    }
    // load n of step `step` of a part, to where the tile's stage begins in LDS
    __device__ __forceinline__ void load(int n, uint32_t lds, const Source &s, int32_t step, int which, int wave) const
    {
#ifdef __HIP_DEVICE_COMPILE__   // (types and registers that the host's compiler does not know)
        const int64_t skip = step * s.step;
        const int64_t records = left - skip;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(at + which * s.part + skip), 0, (int)(uint32_t)(records < 0xfffffff0ll ? records : 0xfffffff0ll), 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsWord *)(uintptr_t)(lds + (wave * kLoads + n) * 1024), 16, from[n % kVary] + n * each, 0, 0, 0);
#endif
    }
    // The same where fragments are transposed as they are read: before such a read the compiler would wait for every load to LDS that it knows of, also for those of
    // the other stage.  (The load has no register for a result, it has read those that say where when it is issued, and the kernel waits for it by itself;
    // nothing else in such a kernel uses m0, which the compiler takes for its own and would warn of here: tests/test_projected_registers.py looks at what it made.  Five wait states: of a scalar register that a vector instruction may just have written.)
    __device__ __forceinline__ void load_untold(int n, uint32_t lds, const Source &s, int32_t step, int which, int wave) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
        const int64_t skip = step * s.step;
        const int64_t records = left - skip;
        const uintptr_t p = reinterpret_cast<uintptr_t>(at + which * s.part + skip);
        const Words rsrc = {(uint32_t)p, (uint32_t)(p >> 32), (uint32_t)(records < 0xfffffff0ll ? records : 0xfffffff0ll), 0x00020000u};
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds + (wave * kLoads + n) * 1024), "v"(from[n % kVary] + n * each), "s"(rsrc) : "memory");
#endif
    }
    // the fragment of 32 rows from `row` (a multiple of 32) on, sixteen k from s * 16 on
    __device__ __forceinline__ V8 fragment(const char *lds, int row, int s, int lane) const
    {
        if constexpr (!KRows) {
            const int r = row + (lane & 31), chunk = (s * 2 + lane / 32) ^ (lane / 2 & 7);
            return *reinterpret_cast<const V8 *>(lds + r * 128 + chunk * 16);
        } else {
            // sixteen lanes read four k of sixteen columns, 8 bytes each, and get a column's four k each
            const int group = lane / 16, l = lane & 15;
            typedef short S4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) S4 *P;
            union {
                S4 half[2];
                V8 v;
            } r;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = s * 16 + (group >> 1) * 8 + q * 4 + l / 4, seg = (row / 16 + (group & 1)) ^ (l / 4 * 2);
                r.half[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + k * (N * 2) + seg * 32 + (l & 3) * 8));
            }
            return r.v;
        }
    }
};

// The order of jobs: workgroups go round the eight XCDs; each XCD gets neighbouring tiles of a slice, in blocks of 8 tiles of j by tiles of i, so that what its
// compute units read at one time stays in its L2.
__device__ __forceinline__ void place(int32_t job, int32_t jobs, int32_t tiles_i, int32_t tiles_j, int32_t &slice, int32_t &ti, int32_t &tj)
{
    const int32_t x = job & 7, each = jobs >> 3, rest = jobs & 7, tiles = tiles_i * tiles_j;
    int32_t id = x * each + min(x, rest) + (job >> 3);
    slice = id / tiles;
    id -= slice * tiles;
    constexpr int32_t kBand = 8;
    const int32_t band = id / (kBand * tiles_i), in_band = id - band * kBand * tiles_i, height = min(kBand, tiles_j - band * kBand);
    ti = in_band / height;
    tj = band * kBand + in_band % height;
}

// 16-bit results of 32 columns (v[i][q]: four of a lane's column) as rows of W * 64 bytes, each written 16 bytes a lane: through a part of LDS of the wavefront's own,
// where the 16 bytes c of a column lie at c ^ column, of as many bits as c has.  `to(r, c)`: where byte c of column r goes, or null.
template <int W, typename V4, typename To>
__device__ __forceinline__ void columns_out(char *lds, const V4 (&v)[W][4], int lane, const To &to)
{
    constexpr int kRow = W * kTile * 2, kChunks = kRow / 16;
    char *mine = lds + (lane & 31) * kRow;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<V4 *>(mine + (((i * 4 + q) ^ (lane & (kChunks - 1))) * 16 + lane / 32 * 8)) = v[i][q];
    __builtin_amdgcn_wave_barrier();   // (the wavefront's own LDS operations are done in order)
#pragma unroll
    for (int n = 0; n < kTile * kChunks / 64; ++n) {
        const int at = n * 64 + lane, r = at / kChunks, c = at % kChunks;
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
        const Words w = *reinterpret_cast<const Words *>(lds + r * kRow + ((c ^ (r & (kChunks - 1))) * 16));
        char *p = to(r, c * 16);
        if (p) *reinterpret_cast<Words *>(p) = w;
    }
    __builtin_amdgcn_wave_barrier();
}

// W: tiles of 32 each way that a wavefront has; a workgroup is 2 x 2 wavefronts.  Workgroups take tiles in turn: the next tile's first two stages are on their way
// while a tile's results are looked after.  Bound by the matrix cores: of 256 x 256 a workgroup, a product of 32 x 32 x 16 takes 512 bytes from LDS, half of what
// that gives in its 32 clocks, and 256 from memory (of 128 x 128 twice that).  One wavefront a SIMD has 256 registers of sums and the fragments of four steps of 16 k.  8,192 x 131,072 x 2,048 bf16 forward 3.66 ms, 1.2 PFLOP/s (with the compiler's order of reads, products
// and loads 4.0); 4,096 x 50,021 x 1,024 both ways 468, 496, 377 and 452 us for the products, 0.84 to 1.1 PFLOP/s.
template <typename E, typename T, int W, bool AK, bool BK, int Mode>
__global__ __launch_bounds__(256, W == 4 ? 1 : 2) void product_kernel(Product p)
{
    constexpr int N = W * 2 * kTile;
    typedef Operand<E, N, 4, AK> OpA;
    typedef Operand<E, N, 4, BK> OpB;
    constexpr int kStage = OpA::kBytes + OpB::kBytes;
    // beside the stages: of kStats, the two halves of a tile's sums; of the 16-bit results, a wavefront's 32 columns, to be written row by row
    constexpr int kRow = W * kTile * 2, kBeside = Mode == kStats ? 2 * N * 8 : Mode == kSlab || (Mode == kOut && std::is_same<T, float>::value) ? 0 : 4 * kTile * kRow;
    __shared__ __align__(1024) char lds[2 * kStage + kBeside];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wi = wave >> 1, wj = wave & 1;
    const int32_t jobs = p.tiles_i * p.tiles_j * p.slices, all = p.steps * p.combinations;
    OpA a;
    OpB b;
    int32_t ti, tj, slice, s0, s1, step, combination;
    const auto fetch_one = [&](int n, int stage) {
        const uint32_t to = (uint32_t)(uintptr_t)(LdsWord *)lds + stage * kStage;
        if constexpr (AK || BK) {
            if (n < OpA::kLoads) a.load_untold(n, to, p.a, step, part_a(combination), wave);
            else b.load_untold(n - OpA::kLoads, to + OpA::kBytes, p.b, step, part_b(combination), wave);
        } else {
            if (n < OpA::kLoads) a.load(n, to, p.a, step, part_a(combination), wave);
            else b.load(n - OpA::kLoads, to + OpA::kBytes, p.b, step, part_b(combination), wave);
        }
    };
    // offsets of loads are made where they are needed: sixteen registers for them, or thirty-two, are not there
    const auto make_here = [&]() {
#pragma unroll
        for (int n = 0; n < OpA::kVary; ++n) asm volatile("" : "+v"(a.from[n]));
#pragma unroll
        for (int n = 0; n < OpB::kVary; ++n) asm volatile("" : "+v"(b.from[n]));
    };
    const auto fetch_next = [&]() {
        make_here();
        const bool more = combination + 1 < p.combinations;
        step = more ? step : step + 1 < p.steps ? step + 1 : 0;   // (behind the last one others are asked for, for nothing)
        combination = more ? combination + 1 : 0;
    };
    constexpr int kLoads = OpA::kLoads + OpB::kLoads;
    const auto begin = [&](int32_t job) {
        place(job, jobs, p.tiles_i, p.tiles_j, slice, ti, tj);
        s0 = (int32_t)((int64_t)all * slice / p.slices), s1 = (int32_t)((int64_t)all * (slice + 1) / p.slices);
        step = s0 / p.combinations, combination = s0 - step * p.combinations;
        // (each XCD begins elsewhere in k, where that can be: rows some power of two apart have the same numbers in the same channels of memory)
        if (p.rotate) step = (int32_t)((int64_t)p.steps * (blockIdx.x & 7) / 8);
        a.start(p.a, ti * N, lane, wave);
        b.start(p.b, tj * N, lane, wave);
        make_here();
#pragma unroll
        for (int stage = 0; stage < 2; ++stage) {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) fetch_one(n, stage);
            fetch_next();
        }
    };
    Acc acc[W][W];
    typename Vec<E>::V8 fa[4][W], fb[4][W];
    // A step is kSlots products of 32 x 32 x 16, a quarter of them for each sixteen k.  Beside them go, one at a time, the reads of the fragments of the other quarters,
    // which are done when kMiddle slots are; then everybody has read this stage, the next one has come, and the tile after it is asked for into this one, beside the
    // reads of the next stage's first fragments.  The order is given: the compiler would read all at once.
    static_assert(kDepth == 64, "four quarters");
    constexpr int kSlots = 4 * W * W, kMiddle = kSlots * 5 / 8, kPerQuarter = 2 * W;
    const auto read = [&](int f, const char *from) {   // fragment f of a step: a's first, then those of b, then the others of a
        const int k = f / kPerQuarter, n = f % kPerQuarter;
        if (n >= 1 && n <= W) fb[k][n - 1] = b.fragment(from + OpA::kBytes, (wj * W + n - 1) * kTile, k, lane);
        else fa[k][n ? n - W : 0] = a.fragment(from, (wi * W + (n ? n - W : 0)) * kTile, k, lane);
    };
    const auto product = [&](int slot) {
        const int k = slot / (W * W), i = slot % (W * W) / W, j = slot % W;
        acc[i][j] = Vec<E>::mfma(fa[k][i], fb[k][j], acc[i][j]);
    };
    const auto cut_fragments = [&](int k) {   // numbers behind the rows, in the last step: of both operands, since what lies there may be NaN
        if (Mode == kSlab || Mode == kOut || p.tail == kDepth) return;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (k * 16 + lane / 32 * 8 >= p.tail) fa[k][j] = fb[k][j] = typename Vec<E>::V8{};
    };
    const auto up_to_the_middle = [&](const char *now, bool last) {
        constexpr int kReads = 3 * kPerQuarter, kOver = kMiddle - kMiddle / 10;
#pragma unroll
        for (int slot = 0; slot < kMiddle; ++slot) {
            if (last && slot % (W * W) == 0) cut_fragments(slot / (W * W));
            product(slot);
#pragma unroll
            for (int f = kReads * min(slot, kOver) / kOver; f < kReads * min(slot + 1, kOver) / kOver; ++f) read(kPerQuarter + f, now);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto everybody = [&]() {
        __builtin_amdgcn_s_waitcnt(kWaitAll);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    if ((int32_t)blockIdx.x >= jobs) return;
    begin(blockIdx.x);
    __builtin_amdgcn_s_waitcnt(kWaitLoads);
    for (int32_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int32_t i0 = ti * N, j0 = tj * N, out_slice = slice;
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int f = 0; f < kPerQuarter; ++f) read(f, lds);
        int32_t s = s0;
        for (; s + 1 < s1; ++s) {
            const int stage = (s - s0) & 1;
            up_to_the_middle(lds + stage * kStage, false);
            everybody();
            constexpr int kLoadsOver = (kSlots - kMiddle) * 2 / 3, kFirst = kMiddle + 2;
#pragma unroll
            for (int slot = kMiddle; slot < kSlots; ++slot) {
                product(slot);
                const int n = slot - kMiddle, r = slot - kFirst;
#pragma unroll
                for (int l = kLoads * min(n, kLoadsOver) / kLoadsOver; l < kLoads * min(n + 1, kLoadsOver) / kLoadsOver; ++l) fetch_one(l, stage);
                constexpr int kReadsOver = kSlots - kFirst - kSlots / 16;
                if (r >= 0)
#pragma unroll
                    for (int f = kPerQuarter * min(r, kReadsOver) / kReadsOver; f < kPerQuarter * min(r + 1, kReadsOver) / kReadsOver; ++f) read(f, lds + (stage ^ 1) * kStage);
                __builtin_amdgcn_sched_barrier(0);
            }
            fetch_next();
        }
        up_to_the_middle(lds + ((s - s0) & 1) * kStage, true);
        everybody();   // (what was asked for behind the last step has come, too)
        // what the results will be asked for, of this lane's column of each tile: before the next tile's loads, so that it is not waited for behind them
        int64_t token[W];
        float peak[W];
        float2 share[W];
        if constexpr (Mode == kStats || Mode == kGradient) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int32_t row = min(j0 + (wj * W + j) * kTile + (lane & 31), p.nj - 1);
                token[j] = p.tokens[row];
                if constexpr (Mode == kGradient) peak[j] = p.peak[row], share[j] = p.shares[row];
            }
        }
        if (job + (int32_t)gridDim.x < jobs) begin(job + gridDim.x);
#pragma unroll
        for (int slot = kMiddle; slot < kSlots; ++slot) {
            if (slot % (W * W) == 0) cut_fragments(slot / (W * W));
            product(slot);
        }
        __builtin_amdgcn_sched_barrier(0);

        // lane l has column j = l % 32 of a tile and its rows i = 8 (r / 4) + 4 (l / 32) + r % 4
        const int half = lane / 32, ii0 = i0 + wi * W * kTile;
        const bool edge = i0 + N > p.ni;
        const auto cut = [&](int j) {   // logits behind the vocabulary
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = ii0 + i * kTile + 8 * (r / 4) + 4 * half + r % 4 >= p.ni ? -INFINITY : acc[i][j][r];
        };
        if constexpr (Mode == kStats) {
            float2 *joined = reinterpret_cast<float2 *>(lds + 2 * kStage);   // [2][N]
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int32_t jj = (wj * W + j) * kTile + (lane & 31), row = j0 + jj;
                if (edge) cut(j);
                float m = acc[0][j][0];
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
                m = fmaxf(m, __shfl_xor(m, 32));
                const float base = base_of(m), from = base == -INFINITY ? 0.0f : base;
                float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s4[r & 3] += exp_over(acc[i][j][r], from);
                float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                sum += __shfl_xor(sum, 32);
                if (half == 0) joined[wi * N + jj] = make_float2(base, sum);
                // the token's logit, where it is in this tile
                const int64_t far = token[j] - p.first - ii0 - 4 * half;
                const int at = row < p.nj && token[j] < p.vocab && far >= 0 && far < W * kTile && !(far & 4) ? (int)far : -1;
                if (__ballot(at >= 0)) {
                    float logit = 0.0f;
#pragma unroll
                    for (int i = 0; i < W; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) logit = at == i * kTile + 8 * (r / 4) + r % 4 ? acc[i][j][r] : logit;
                    if (at >= 0) p.label[row] = logit;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_waitcnt(kWaitReads);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            for (int jj = threadIdx.x; jj < N; jj += 256)
                if (j0 + jj < p.nj) p.stats[(int64_t)(i0 / N) * p.nj + j0 + jj] = join(joined[jj], joined[N + jj]);
            // (the next tile's barriers are between these reads and what it writes there)
        } else if constexpr (Mode == kGradient) {
            typedef typename Vec<E>::V4 V4;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int32_t row = j0 + (wj * W + j) * kTile + (lane & 31);
                const float by_total = share[j].x, whole = share[j].y;
                const bool none = row >= p.nj || whole == 0.0f;
                const int64_t far = token[j] - p.first - ii0 - 4 * half;
                const int at = far >= 0 && far < W * kTile && !(far & 4) ? (int)far : -1;
                if (edge) cut(j);
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] = none ? 0.0f : exp_over(acc[i][j][r], peak[j]) * by_total;
                if (__ballot(at >= 0 && !none)) {
#pragma unroll
                    for (int i = 0; i < W; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][j][r] -= at == i * kTile + 8 * (r / 4) + r % 4 && !none ? whole : 0.0f;
                }
                V4 out[std::is_same<T, float>::value ? 3 : 1][W][4];
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if constexpr (std::is_same<T, float>::value) {
                                bf16 part[3];
                                split(acc[i][j][q * 4 + r], part);
#pragma unroll
                                for (int k = 0; k < 3; ++k) out[k][i][q][r] = part[k];
                            } else {   // (what both products read in 16 bits: gradients are off by 1.3 times what rounding them alone would be, 2.2e-3 of 1.7e-3 in bf16)
                                out[0][i][q][r] = (E)acc[i][j][q * 4 + r];
                            }
                        }
                const int32_t row0 = j0 + (wj * W + j) * kTile;
#pragma unroll
                for (int k = 0; k < (std::is_same<T, float>::value ? 3 : 1); ++k) {
                    char *to = reinterpret_cast<char *>(static_cast<E *>(p.g) + k * p.g_part);
                    columns_out<W>(lds + 2 * kStage + wave * kTile * kRow, out[k], lane, [&](int r, int c) {
                        const int32_t byte = (ii0 * 2 + c) / 128;
                        return to + byte * p.g_block * 2 + (int64_t)(row0 + r) * 128 + (ii0 * 2 + c) % 128;
                    });
                }
            }
        } else {
            const float scale = Mode == kOut ? p.out_scale * *p.factor / lift_of(p.reach) : 1.0f;
            // (rows of whole 16 bytes can go out in those)
            const bool rows_fit = Mode == kOut && sizeof(T) == 2 && p.ni % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int32_t row0 = j0 + (wj * W + j) * kTile, row = row0 + (lane & 31);
                if constexpr (Mode == kOut && sizeof(T) == 2) {
                    if (rows_fit) {
                        typename Vec<E>::V4 out[W][4];
#pragma unroll
                        for (int i = 0; i < W; ++i)
#pragma unroll
                            for (int q = 0; q < 4; ++q)
#pragma unroll
                                for (int r = 0; r < 4; ++r) out[i][q][r] = (E)(acc[i][j][q * 4 + r] * scale);
                        columns_out<W>(lds + 2 * kStage + wave * kTile * kRow, out, lane, [&](int r, int c) {
                            char *to = static_cast<char *>(p.out) + ((int64_t)(row0 + r) * p.ni + ii0) * 2 + c;
                            return row0 + r < p.nj && ii0 + c / 2 < p.ni ? to : nullptr;
                        });
                        continue;
                    }
                }
                if (row >= p.nj) continue;
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int32_t col = ii0 + i * kTile + 8 * q + 4 * half;
                        if (col >= p.ni) continue;
                        float v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = acc[i][j][q * 4 + r] * scale;
                        if constexpr (Mode == kSlab) {   // (rows of a slab are whole fours)
                            Acc4 *to = reinterpret_cast<Acc4 *>(p.slab + out_slice * p.slab_size + row * p.slab_stride + col);
                            const Acc4 sum = {v[0], v[1], v[2], v[3]};
                            *to = p.add ? *to + sum : sum;
                        } else {
                            put<T, 4>(static_cast<T *>(p.out) + (int64_t)row * p.ni + col, v, p.ni - col);
                        }
                    }
            }
        }
        // The next tile's loads have come; the results that were written after them need not have arrived.  (Memory operations are counted in order.)
        constexpr int kWritten = Mode == kGradient ? W * (kTile * kRow / 1024) * (std::is_same<T, float>::value ? 3 : 1) : 0, kMayWait = kWritten < 63 ? kWritten : 63;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(kWaitLoads | kMayWait % 16 | kMayWait / 16 << 14);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// what goes before and after

// Rows of n numbers, `width` (n or more, with zeros; a multiple of 8) apart, of T or as the three parts of float; with `by`, times by[row] and lift_of(reach), and
// rows that have no part are 0.  Eight numbers a lane.
template <typename T, typename E>
__global__ __launch_bounds__(256) void lay_kernel(const T *from, int64_t stride, int64_t rows, int32_t n, int32_t width, int64_t padded_rows, E *to, const float *by, const float *reach)
{
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, row = k / (width / 8);
    const int32_t c = (int32_t)(k - row * (width / 8)) * 8;
    if (row >= padded_rows) return;
    Loose8<T> in;
    const int some = row < rows ? n - c : 0;
    if (some >= 8) in.load(from + row * stride + c);
    else in.load_some(from + row * stride + c, some);
    const float f = by && row < rows ? by[row] * lift_of(reach) : 1.0f;
    typedef typename Vec<E>::V8 V8;
    V8 out[std::is_same<T, float>::value ? 3 : 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = (float)in.v[i];
        if (by) v = f == 0.0f ? 0.0f : v * f;
        if constexpr (std::is_same<T, float>::value) {
            bf16 s[3];
            split(v, s);
#pragma unroll
            for (int j = 0; j < 3; ++j) out[j][i] = s[j];
        } else {
            out[0][i] = (E)v;
        }
    }
#pragma unroll
    for (int j = 0; j < (std::is_same<T, float>::value ? 3 : 1); ++j) *reinterpret_cast<V8 *>(to + j * padded_rows * width + k * 8) = out[j];
}

// The largest finite |d_logp| of the rows that have a token, of those that a workgroup's threads look at: first, first + step, ..., eight at a time
__device__ __forceinline__ float largest(const float *d_logp, const int64_t *tokens, int64_t ignore, int64_t rows, int64_t first, int64_t step)
{
    __shared__ float most[16];
    float m = 0.0f;
    for (int64_t r = first; r < rows; r += 8 * step) {
        float d[8];
        int64_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t at = r + i * step < rows ? r + i * step : r;
            d[i] = fabsf(d_logp[at]), t[i] = tokens[at];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) m = t[i] != ignore && d[i] < INFINITY ? fmaxf(m, d[i]) : m;
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    if (lane_id() == 0) most[threadIdx.x / kWave] = m;
    __syncthreads();
    m = 0.0f;
    for (int k = 0; k < 16; ++k) m = fmaxf(m, most[k]);
    return m;
}
constexpr int kLargest = 256;   // workgroups, of more than 32,768 rows
__global__ __launch_bounds__(1024) void largest_kernel(const float *d_logp, const int64_t *tokens, int64_t ignore, int64_t rows, float *out)
{
    const float m = largest(d_logp, tokens, ignore, rows, (int64_t)blockIdx.x * 1024 + threadIdx.x, kLargest * 1024);
    if (threadIdx.x == 0) out[blockIdx.x] = m;
}

// reach (see lift_of) of finite numbers; weigh_kernel has made it 0.  The largest of all does not depend on who comes first.  Bound by memory, and a launch: 20,000 x 2,000 17 us of the 122 that
// the gradient of 64 words takes, 1,000 x 777 6 of 273 of 32,003 words.
__global__ __launch_bounds__(1024) void reach_kernel(const f16 *x, int64_t stride, int64_t rows, int32_t n, const float *sizes, float *reach)
{
    __shared__ float most[16];
    const int32_t each = (n + 7) / 8;
    float m = 0.0f;
#pragma unroll 4
    for (int64_t k = (int64_t)blockIdx.x * 1024 + threadIdx.x; k < rows * each; k += (int64_t)gridDim.x * 1024) {
        const int64_t row = k / each;
        const int32_t c = (int32_t)(k - row * each) * 8;
        Loose8<f16> in;
        if (c + 8 <= n) in.load(x + row * stride + c);
        else in.load_some(x + row * stride + c, n - c);
        const float size = sizes[row];   // (0: the row may hold anything)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = fabsf((float)in.v[i]);
            m = v < INFINITY ? fmaxf(m, v * size) : m;
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    if (lane_id() == 0) most[threadIdx.x / kWave] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < 16; ++k) m = fmaxf(m, most[k]);
    atomicMax(reinterpret_cast<uint32_t *>(reach), __float_as_uint(m));   // (0 or more: their bits are in their order)
}

// For few rows weights[row] = d_logp, 0 for rows that have no part, NaN where Share has that.  Otherwise, with shares, each row's Share of d_logp over the largest, *factor, and
// its size as weight.  The largest: that of largest_kernel's, or, without those, of all rows, which every workgroup looks at
__global__ __launch_bounds__(1024) void weigh_kernel(const float *d_logp, const int64_t *tokens, int64_t ignore, int64_t rows, int32_t vocab, const float *peak,
                                                     const float *total, float g_scale, float *weights, float2 *shares, float *factor, float *reach, const float *parts)
{
    float c = 1.0f;
    if (shares) {
        float m = 0.0f;
        if (parts) {
            for (int k = 0; k < kLargest; ++k) m = fmaxf(m, parts[k]);
        } else {
            m = largest(d_logp, tokens, ignore, rows, threadIdx.x, 1024);
        }
        c = m > 0.0f ? fmaxf(m, 0x1p-120f) : 1.0f;   // (so that quotients are not lost)
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *factor = c, *reach = 0.0f;
    const int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x;
    if (r < rows) {
        const int64_t token = tokens[r];
        if (shares) {
            const Share share(d_logp[r] / c, token, ignore, vocab, peak[r], total[r], g_scale);
            weights[r] = share.size;
            shares[r] = make_float2(share.by_total, share.whole);
        } else {
            weights[r] = no_part(token, ignore, peak[r], total[r]) ? 0.0f : undefined(token, vocab, total[r]) ? NAN : d_logp[r];
        }
    }
}

// a row's results from its base and sum
__device__ __forceinline__ void finish(float2 sum, int32_t row, float label, const int64_t *tokens, int64_t ignore, int32_t vocab, float *logp, float *lse, float *peak, float *total)
{
    const float m = sum.x, s = sum.y, log_total = logf(s);
    const float l = m == -INFINITY && s == 0.0f ? -INFINITY : fmaf(m, kLn2, log_total);
    const int64_t token = tokens[row];
    peak[row] = m;
    total[row] = s;
    lse[row] = m == INFINITY ? NAN : l;
    logp[row] = token == ignore ? 0.0f : token < 0 || token >= vocab || m == INFINITY ? NAN : l == -INFINITY ? -INFINITY : fmaf(fmaf(label, kLog2e, -m), kLn2, -log_total);
}

// each row's tiles joined: a workgroup takes 64 rows, each of its 16 wavefronts every sixteenth tile
__global__ __launch_bounds__(1024) void stats_join_kernel(const float2 *stats, int32_t tiles, int32_t rows, const float *label, const int64_t *tokens, int64_t ignore, int32_t vocab,
                                                          float *logp, float *lse, float *peak, float *total)
{
    __shared__ float2 parts[16][64];
    const int wave = threadIdx.x / kWave, lane = lane_id();
    const int32_t row = blockIdx.x * 64 + lane;
    float2 sum = make_float2(-INFINITY, 0.0f);
    if (row < rows) {
        for (int k = wave; k < tiles; k += 16 * 4) {
            float2 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = stats[(int64_t)min(k + 16 * i, tiles - 1) * rows + row];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k + 16 * i < tiles) sum = join(sum, q[i]);
        }
    }
    parts[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || row >= rows) return;
    for (int k = 1; k < 16; ++k) sum = join(sum, parts[k][lane]);
    finish(sum, row, label[row], tokens, ignore, vocab, logp, lse, peak, total);
}
// Results from their slabs: rows of `width` numbers, n of them there.  `ways` wavefronts of a workgroup share 64 times four numbers, each takes every so manieth slab.
template <typename T>
__global__ __launch_bounds__(1024) void slab_join_kernel(const float *slab, int32_t slabs, int64_t slab_size, int64_t rows, int32_t n, int32_t width, int32_t ways, const float *by,
                                                         const float *factor, const float *reach, float scale, T *out)
{
    __shared__ Acc4 parts[16][64];
    const int wave = threadIdx.x / kWave, lane = lane_id(), way = wave % ways;
    const int64_t k = ((int64_t)blockIdx.x * (blockDim.x / kWave / ways) + wave / ways) * 64 + lane, row = k / (width / 4);
    const int32_t c = (int32_t)(k - row * (width / 4)) * 4;
    const bool there = row < rows && c < n;
    Acc4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (there) {
        const float *p = slab + row * width + c;
        int32_t i = way;
        for (; i + 3 * ways < slabs; i += 4 * ways) {
            Acc4 q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const Acc4 *>(p + (i + u * ways) * slab_size);
#pragma unroll
            for (int u = 0; u < 4; ++u) v += q[u];
        }
        for (; i < slabs; i += ways) v += *reinterpret_cast<const Acc4 *>(p + i * slab_size);
    }
    if (ways > 1) {
        parts[wave][lane] = v;
        __syncthreads();
        if (way != 0) return;
        for (int w = 1; w < ways; ++w) v += parts[wave + w][lane];
    }
    if (!there) return;
    const float w = by ? by[row] : 1.0f, f = scale * (factor ? *factor : 1.0f) / lift_of(reach) * w;
    const float r[4] = {w == 0.0f ? 0.0f : v[0] * f, w == 0.0f ? 0.0f : v[1] * f, w == 0.0f ? 0.0f : v[2] * f, w == 0.0f ? 0.0f : v[3] * f};
    put<T, 4>(out + row * n + c, r, n - c);
}

// ---------------------------------------------------------------------------------------------------------------------
// few rows: a wavefront takes 32 rows of the weights straight from memory into matrix instructions of 16 x 16, against J times 16 rows of x from the
// caches.  Bound by the weights' bytes (4 x 131,072 x 2,048 bf16 109 us, 4.9 TB/s).

struct Few {
    const void *x, *weight;
    const int64_t *tokens;
    int64_t x_stride, w_stride;   // in numbers
    int32_t rows, vocab, dim;
    float2 *stats;
    float *label;
    // backward
    const float *peak, *total, *weights;   // weights: see weigh_kernel
    int64_t ignore;
    float *g;                              // [vocab, to a whole 128][rows, to a whole 16]: p - delta
    void *d_weight;
    float *slab;                           // [slices][rows][dim, to a whole 8]
    int32_t slices, slice_rows;            // slices of the vocabulary, of so many of its rows (a multiple of 16)
    const float *factor, *reach;           // small vocabulary: the Shares are of d_logp over this number (none: 1), and their scale is 1 / g_unit; see lift_of
    float g_unit;
};

// acc[i][j] += the products of 16 rows of I tiles by 16 rows of J tiles, over the steps of 32 k from first to end; p, q: where this lane's rows have their first eight k
template <typename T, int I, int J>
__device__ __forceinline__ void multiply_rows(const T *const (&p)[I], const T *const (&q)[J], int32_t first, int32_t end, int32_t dim, int quarter, Acc4 (&acc)[I][J])
{
    typedef typename Element<T>::type E;
    typedef typename Vec<E>::V8 V8;
    const auto multiply = [&](const Loose8<T> (&u)[I], const Loose8<T> (&v)[J]) {
        if constexpr (std::is_same<T, float>::value) {
            // (fp32 operands in fp32 instructions, one k of a lane's eight each: at so few rows they keep up with memory)
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int i = 0; i < I; ++i)
#pragma unroll
                    for (int j = 0; j < J; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[i].v[k], v[j].v[k], acc[i][j], 0, 0, 0);
        } else {
            V8 uv[I], vv[J];
#pragma unroll
            for (int i = 0; i < I; ++i) __builtin_memcpy(&uv[i], &u[i], 16);
#pragma unroll
            for (int j = 0; j < J; ++j) __builtin_memcpy(&vv[j], &v[j], 16);
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < J; ++j) acc[i][j] = Vec<E>::mfma16(uv[i], vv[j], acc[i][j]);
        }
    };
    constexpr int kAhead = (std::is_same<T, float>::value ? 2 : 4) / (I + J > 4 ? 2 : 1);   // steps of 32 k that are asked for at once
    const int32_t whole = min(end, dim / 32);
    const auto ask = [&](int32_t k, Loose8<T> (&u)[kAhead][I], Loose8<T> (&v)[kAhead][J]) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
#pragma unroll
            for (int i = 0; i < I; ++i) u[s][i].load(p[i] + (k + s) * 32);
#pragma unroll
            for (int j = 0; j < J; ++j) v[s][j].load(q[j] + (k + s) * 32);
        }
    };
    int32_t k = first;
    if (k + kAhead <= whole) {
        Loose8<T> u_next[kAhead][I], v_next[kAhead][J];
        ask(k, u_next, v_next);
        for (; k + kAhead <= whole; k += kAhead) {
            Loose8<T> u[kAhead][I], v[kAhead][J];
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                for (int i = 0; i < I; ++i) u[s][i] = u_next[s][i];
#pragma unroll
                for (int j = 0; j < J; ++j) v[s][j] = v_next[s][j];
            }
            if (k + 2 * kAhead <= whole) ask(k + kAhead, u_next, v_next);
#pragma unroll
            for (int s = 0; s < kAhead; ++s) multiply(u[s], v[s]);
        }
    }
    for (; k < whole; ++k) {
        Loose8<T> u[I], v[J];
#pragma unroll
        for (int i = 0; i < I; ++i) u[i].load(p[i] + k * 32);
#pragma unroll
        for (int j = 0; j < J; ++j) v[j].load(q[j] + k * 32);
        multiply(u, v);
    }
    for (; k < end; ++k) {
        Loose8<T> u[I], v[J];
        const int n = dim - k * 32 - quarter * 8;
#pragma unroll
        for (int i = 0; i < I; ++i) u[i].load_some(p[i] + k * 32, n);
#pragma unroll
        for (int j = 0; j < J; ++j) v[j].load_some(q[j] + k * 32, n);
        multiply(u, v);
    }
}

// where the wavefronts of a workgroup share a sum: all of it in the first one's registers
template <int Split, int I, int J>
__device__ __forceinline__ void add_up(Acc4 (&acc)[I][J], Acc4 (&sums)[Split - 1][I][J][64], int wave, int lane)
{
    if (wave > 0) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) sums[wave - 1][i][j][lane] = acc[i][j];
    }
    __syncthreads();
    if (wave > 0) return;
    for (int w = 0; w < Split - 1; ++w)
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) acc[i][j] += sums[w][i][j][lane];
}

// Split: wavefronts of a workgroup that share 32 rows of the weights, each a part of the channels.
template <typename T, int J, int Split, bool Gradient>
__global__ __launch_bounds__(Split == 8 ? 512 : 256) void few_rows_kernel(Few a)
{
    constexpr int kBlocks = Split == 1 ? 4 : 1;   // of 32 rows
    __shared__ float2 parts[kBlocks][J * 16];
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    const int32_t v0 = (blockIdx.x * kBlocks + (Split == 1 ? wave : 0)) * 32;
    const T *w_row[2], *x_row[J];
#pragma unroll
    for (int i = 0; i < 2; ++i) w_row[i] = static_cast<const T *>(a.weight) + (int64_t)min(v0 + i * 16 + r16, a.vocab - 1) * a.w_stride + quarter * 8;
#pragma unroll
    for (int j = 0; j < J; ++j) x_row[j] = static_cast<const T *>(a.x) + (int64_t)min(j * 16 + r16, a.rows - 1) * a.x_stride + quarter * 8;
    Acc4 acc[2][J];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) acc[i][j] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    const int32_t steps = (a.dim + 31) / 32, part = Split == 1 ? 0 : wave;
    multiply_rows<T, 2, J>(w_row, x_row, steps * part / Split, steps * (part + 1) / Split, a.dim, quarter, acc);
    if constexpr (Split > 1) {
        __shared__ Acc4 sums[Split - 1][2][J][64];
        add_up<Split>(acc, sums, wave, lane);
        if (wave > 0) return;
    }
    // lane l has column j = l % 16 of a tile and its rows i = 4 (l / 16) + r
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int32_t row = j * 16 + r16;
        const int64_t token = row < a.rows ? a.tokens[row] : -1;
        if constexpr (Gradient) {
            const float peak = row < a.rows ? a.peak[row] : -INFINITY, total = row < a.rows ? a.total[row] : 0.0f, inverse = 1.0f / total;
            const bool none = row >= a.rows || no_part(token, a.ignore, peak, total);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t v = v0 + i * 16 + quarter * 4 + r;
                    const float p = exp_over(acc[i][j][r], peak) * inverse;
                    a.g[(int64_t)v * (J * 16) + row] = none || v >= a.vocab ? 0.0f : v == token ? p - 1.0f : p;
                }
            continue;
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int32_t v = v0 + i * 16 + quarter * 4 + r;
                if (v >= a.vocab) acc[i][j][r] = -INFINITY;
                else if (v == token) a.label[row] = acc[i][j][r];
                m = fmaxf(m, acc[i][j][r]);
            }
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const float base = base_of(m), from = base == -INFINITY ? 0.0f : base;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += exp_over(acc[i][j][r], from);
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (Split > 1 && quarter == 0 && row < a.rows) a.stats[(int64_t)blockIdx.x * a.rows + row] = make_float2(base, s);
        if (Split == 1 && quarter == 0) parts[wave][row] = make_float2(base, s);
    }
    if constexpr (Gradient || Split > 1) return;
    __syncthreads();
    if ((int)threadIdx.x < a.rows) {
        float2 sum = parts[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kBlocks; ++w) sum = join(sum, parts[w][threadIdx.x]);
        a.stats[(int64_t)blockIdx.x * a.rows + threadIdx.x] = sum;
    }
}

// four numbers of a lane's k, one of each, or sixteen k's in one instruction
__device__ __forceinline__ Acc4 multiply_fours(const Acc4 &a, const Acc4 &b, Acc4 c)
{
#pragma unroll
    for (int m = 0; m < 4; ++m) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m], b[m], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ Acc4 multiply_fours(const Vec<bf16>::V4 &a, const Vec<bf16>::V4 &b, Acc4 c) { return Vec<bf16>::mfma16(a, b, c); }
__device__ __forceinline__ Acc4 multiply_fours(const Vec<f16>::V4 &a, const Vec<f16>::V4 &b, Acc4 c) { return Vec<f16>::mfma16(a, b, c); }

// what G is kept in
template <typename T, bool Classes>
struct Kept {
    typedef float type;
    typedef Acc4 V4;
};
template <>
struct Kept<bf16, true> {
    typedef bf16 type;
    typedef Vec<bf16>::V4 V4;
};
template <>
struct Kept<f16, true> {
    typedef f16 type;
    typedef Vec<f16>::V4 V4;
};

// The two products of G for few rows, in one pass over the weights: a wavefront takes 16 C channels (a lane C) of a slice of the vocabulary, and per 16 of its rows
//     dx[r][d] -= G[v][r] w[v][d]   and   d_weight[v][d] = -sum_r G[v][r] d_logp[r] x[r][d]
// in matrix instructions of 32 bits.  A lane's k are 4 (l / 16) .. 4 (l / 16) + 3, of rows as of the vocabulary, which nothing has to be transposed for, and its C channels are C tiles.
// Bound by memory: the weights read, their gradient written (16 x 194,675 x 3,999 fp32 1.86 ms, 3.35 TB/s).
// Classes: a small vocabulary and many rows, the two in each other's place: of each 16 rows d_weight -= G^T (size x) and dx = -size G weight, in 16 bits where the type has them
// (G is rounded to it; size: see Share, and lift_of).  Rows that have no part, of size 0, may hold anything.  A workgroup's wavefronts share a slice of the rows and add up.
template <typename T, int J, int C, bool Classes>
__global__ __launch_bounds__(256) void few_back_kernel(Few a)
{
    typedef LooseFew<T, C> In;
    typedef typename Kept<T, Classes>::type G;
    typedef typename Kept<T, Classes>::V4 V4;
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, kk = lane >> 4;
    const int32_t d0 = (Classes ? blockIdx.x : blockIdx.x * 4 + wave) * (16 * C), d = d0 + r16 * C;
    const int32_t some = a.dim - d;   // this lane's channels that are there, if fewer than C
    if (d0 >= a.dim) return;
    const G *g = reinterpret_cast<const G *>(a.g);
    V4 xw[J][C];   // x d_logp; Classes: weights
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int32_t row = j * 16 + kk * 4 + m;
            const float by = row >= a.rows ? 0.0f : Classes ? 1.0f : a.weights[row];
            In x;
            x.load(static_cast<const T *>(a.x) + (int64_t)min(row, a.rows - 1) * a.x_stride + d, some);
#pragma unroll
            for (int q = 0; q < C; ++q) xw[j][q][m] = (G)(by == 0.0f ? 0.0f : -by * (float)x.v[q]);
        }
    Acc4 dx[J][C];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int q = 0; q < C; ++q) dx[j][q] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kEach = Classes ? 64 : 16;   // rows that a workgroup, or a wavefront of its own, goes on by
    const int32_t v_end = min((int32_t)(blockIdx.y + 1) * a.slice_rows, a.vocab), v_first = blockIdx.y * a.slice_rows + (Classes ? wave * 16 : 0);
    const float factor = !Classes ? 1.0f : a.factor ? *a.factor * a.g_unit : a.g_unit, lift = Classes ? lift_of(a.reach) : 1.0f;
    struct Block {
        In w[4];
        float part[4];
        G by_row[J][4];
        V4 by_vocab[J];
    };
    const auto ask = [&](int32_t v, Block &to) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int32_t at = min(v + kk * 4 + u, a.vocab - 1);
            to.w[u].load(static_cast<const T *>(a.weight) + (int64_t)at * a.w_stride + d, some);
            if (Classes) to.part[u] = a.weights[at];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int u = 0; u < 4; ++u) to.by_row[j][u] = g[(int64_t)(v + kk * 4 + u) * (J * 16) + j * 16 + r16];
            to.by_vocab[j] = *reinterpret_cast<const V4 *>(g + (int64_t)(v + r16) * (J * 16) + j * 16 + kk * 4);
        }
    };
    Block next;
    if (v_first < v_end) ask(v_first, next);
    for (int32_t v = v_first; v < v_end; v += kEach) {
        const Block now = next;
        if (v + kEach < v_end) ask(v + kEach, next);
        V4 w[C];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < C; ++q) w[q][u] = (G)(!Classes ? (float)now.w[u].v[q] : now.part[u] == 0.0f ? 0.0f : (float)now.w[u].v[q] * (now.part[u] * lift));
        Acc4 dw[C];
#pragma unroll
        for (int q = 0; q < C; ++q) dw[q] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const V4 by_row = {now.by_row[j][0], now.by_row[j][1], now.by_row[j][2], now.by_row[j][3]};
#pragma unroll
            for (int q = 0; q < C; ++q) {
                dx[j][q] = multiply_fours(by_row, w[q], dx[j][q]);
                dw[q] = multiply_fours(now.by_vocab[j], xw[j][q], dw[q]);
            }
        }
        // lane l has column l % 16, C channels, and its rows 4 (l / 16) + r
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t at = v + kk * 4 + r;
            if (at >= v_end || some <= 0) continue;
            float out[C];
#pragma unroll
            for (int q = 0; q < C; ++q) out[q] = !Classes ? dw[q][r] : now.part[r] == 0.0f ? 0.0f : dw[q][r] * (now.part[r] * factor);
            put<T, C>(static_cast<T *>(a.d_weight) + (int64_t)at * a.dim + d, out, some);
        }
    }
    if constexpr (Classes) {
        __shared__ Acc4 sums[3][J][C][64];
        add_up<4>(dx, sums, wave, lane);
        if (wave > 0) return;
    }
    const int64_t width = up8(a.dim);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t row = j * 16 + kk * 4 + r;
            typedef float Out __attribute__((ext_vector_type(C)));
            Out out;
#pragma unroll
            for (int q = 0; q < C; ++q) out[q] = dx[j][q][r];
            if (row < a.rows && some > 0) *reinterpret_cast<Out *>(a.slab + ((int64_t)blockIdx.y * a.rows + row) * width + d) = out;
        }
}

// ---------------------------------------------------------------------------------------------------------------------
// a small vocabulary: a wavefront takes R times 16 rows of x straight from memory against J times 16 rows of weights from the caches, and has all of a row's logits, four of each tile in
// each of four lanes.  Bound by the bytes of x (18,124 x 2 x 1,930 bf16 16 us, 4.4 TB/s; fp32 30 us, 4.7 TB/s), and from four tiles of weights on by theirs from the caches (20,000 x 64 x 2,000
// bf16 32 us, 2.6 TB/s).

struct Small {
    const void *x, *weight;
    const int64_t *tokens;
    int64_t x_stride, w_stride, ignore;
    int32_t rows, vocab, dim;
    float *logp, *lse, *peak, *total;   // (peak and total: read by the backward pass)
    const float *d_logp;
    void *g;                            // [rows, to a whole 32][vocab, to a whole 16]: p - delta times the Share's whole
    float *weights;                     // the Shares' sizes
    const float2 *shares;               // where weigh_kernel has made them, and the sizes; else none
};

// Split: wavefronts of a workgroup that share rows, each a part of the channels
template <typename T, int J, int Split, bool Gradient>
__global__ __launch_bounds__(Split == 8 ? 512 : 256) void small_kernel(Small a)
{
    constexpr int R = Split == 8 ? 1 : 2;
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    const int32_t row0 = (Split == 1 ? blockIdx.x * 4 + wave : blockIdx.x) * (R * 16);
    if (row0 >= a.rows) return;   // (of workgroups that share rows, all or none)
    const T *w_row[J], *x_row[R];
#pragma unroll
    for (int j = 0; j < J; ++j) w_row[j] = static_cast<const T *>(a.weight) + (int64_t)min(j * 16 + r16, a.vocab - 1) * a.w_stride + quarter * 8;
#pragma unroll
    for (int i = 0; i < R; ++i) x_row[i] = static_cast<const T *>(a.x) + (int64_t)min(row0 + i * 16 + r16, a.rows - 1) * a.x_stride + quarter * 8;
    Acc4 acc[J][R];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < R; ++i) acc[j][i] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    const int32_t steps = (a.dim + 31) / 32, part = Split == 1 ? 0 : wave;
    multiply_rows<T, J, R>(w_row, x_row, steps * part / Split, steps * (part + 1) / Split, a.dim, quarter, acc);
    if constexpr (Split > 1) {
        __shared__ Acc4 sums[Split - 1][J][R][64];
        add_up<Split>(acc, sums, wave, lane);
        if (wave > 0) return;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int32_t row = row0 + i * 16 + r16;
        const bool there = row < a.rows;
        const int64_t token = there ? a.tokens[row] : -1;
        if constexpr (Gradient) {
            const float peak = there ? a.peak[row] : 0.0f;
            float by_total = 0.0f, whole = 0.0f;
            if (there && a.shares) {
                by_total = a.shares[row].x, whole = a.shares[row].y;
            } else if (there) {
                const Share share(a.d_logp[row], token, a.ignore, a.vocab, peak, a.total[row], 1.0f);
                by_total = share.by_total, whole = share.whole;
                if (quarter == 0) a.weights[row] = share.size;
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                typename Kept<T, true>::V4 g;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t v = j * 16 + quarter * 4 + r;
                    const float p = exp_over(acc[j][i][r], peak) * by_total;
                    g[r] = (typename Kept<T, true>::type)(whole == 0.0f || v >= a.vocab ? 0.0f : v == token ? p - whole : p);
                }
                *reinterpret_cast<typename Kept<T, true>::V4 *>(static_cast<typename Kept<T, true>::type *>(a.g) + (int64_t)row * (J * 16) + j * 16 + quarter * 4) = g;
            }
        } else {
            float m = -INFINITY, label = 0.0f, s = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t v = j * 16 + quarter * 4 + r;
                    if (v >= a.vocab) acc[j][i][r] = -INFINITY;
                    else if (v == token) label = acc[j][i][r];
                    m = fmaxf(m, acc[j][i][r]);
                }
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            const float base = base_of(m), from = base == -INFINITY ? 0.0f : base;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += exp_over(acc[j][i][r], from);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            label += __shfl_xor(label, 16);   // (one lane has it, the others 0)
            label += __shfl_xor(label, 32);
            if (there && quarter == 0) finish(make_float2(base, s), row, label, a.tokens, a.ignore, a.vocab, a.logp, a.lse, a.peak, a.total);
        }
    }
}

// the same of few rows: a workgroup to a row, its threads each every 256th tile
__global__ __launch_bounds__(256) void few_join_kernel(const float2 *stats, int32_t tiles, int32_t rows, const float *label, const int64_t *tokens, int64_t ignore, int32_t vocab,
                                                       float *logp, float *lse, float *peak, float *total)
{
    __shared__ float2 parts[4];
    const int32_t row = blockIdx.x;
    float2 sum = make_float2(-INFINITY, 0.0f);
    for (int k = threadIdx.x; k < tiles; k += 256) sum = join(sum, stats[(int64_t)k * rows + row]);
#pragma unroll
    for (int k = 32; k; k >>= 1) sum = join(sum, make_float2(__shfl_xor(sum.x, k), __shfl_xor(sum.y, k)));
    if (lane_id() == 0) parts[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) finish(join(join(parts[0], parts[1]), join(parts[2], parts[3])), row, label[row], tokens, ignore, vocab, logp, lse, peak, total);
}

// ---------------------------------------------------------------------------------------------------------------------

// Up to how many rows the kernels for few rows take.  us of 100,000 x 2,000, forward and both ways, few / large tiles: bf16 12 rows 100/148, 484/560; 17: 118/150, 603/561; 33:
// 143/152, 1021/566; 64: 171/152, 1191/571; fp32 12: 203/889, 785/2553; 64: 514/900, 1928/2691.  Large tiles of 16-bit weights whose rows do not
// begin at whole 16 bytes copy them first, 170 us each way here.
int32_t few_most(int32_t dtype, bool w_fits, bool backward) { return dtype == BMTK_F32 ? 64 : w_fits ? (backward ? 16 : 32) : (backward ? 32 : 64); }
// Whether a vocabulary is taken by the kernels for a small one.  Not where there are fewer rows than that, and few.  Of fp32 always: the large tiles copy it in parts first (us forward, both
// ways, small / large: 20,000 x 128 x 2,000 fp32 129/210, 545/768; 18,124 x 2 x 1,930 30/195, 138/660).  Of 16 bits up to 64 (20,000 x 30 x 4,000 36/49, 163/416; 20,000 x 64 x 2,000 32/31,
// 137/238); above, where each workgroup's weights weigh less than what the large tiles cost (20,000 x 100 x 250 13/22; 5,000 x 100 x 1,000 12/16, 89/75; 20,000 x 128 x 2,000 60/35, 322/257;
// 2,000 x 100 x 2,000 16/23, 76/88); and of long rows that do not begin at whole 16 bytes up to 32 (5,000 x 50 x 3,001 67/50, 176/151).
bool small_vocab(int64_t rows, int64_t vocab, int32_t dim, int32_t dtype, bool x_fits, bool w_fits, bool backward)
{
    if (vocab > kSmallMost || (vocab > rows && rows <= few_most(dtype, w_fits, backward))) return false;
    if (dtype == BMTK_F32 || vocab <= 32) return true;
    if (dim > 512 && !(x_fits && w_fits)) return false;
    return vocab <= 64 || (backward ? rows <= 4096 : rows * dim <= (5 << 20));
}
int32_t small_tiles(int64_t vocab) { return vocab <= 16 ? 1 : vocab <= 32 ? 2 : vocab <= 64 ? 4 : 8; }
// wavefronts that share rows: where those would leave the chip empty and channels are enough
int32_t small_split(int64_t rows, int32_t dim) { return rows >= 32 * 2048 || dim < 256 ? 1 : rows >= 32 * 256 || dim < 1024 ? 4 : 8; }
constexpr int64_t kPieceBytes = int64_t{512} << 20;   // of G: pieces of the vocabulary are as large as that allows, of 256 words at least

int64_t up(int64_t n, int64_t to) { return div_up(n, to) * to; }

// tiles of 256 or 128 a workgroup: the large ones need half the reads for a product, and at least as many as three quarters of the chip's compute units
int32_t tile_of(int64_t ni, int64_t nj, int64_t slices = 1) { return div_up(ni, 256) * div_up(nj, 256) * slices >= 192 ? 256 : 128; }

struct Plan {
    int32_t parts, combinations, depth;          // depth: dim to whole steps
    bool small, few, copy_x, copy_w;             // the kernels for a small vocabulary, for few rows; operands that are laid out anew
    int64_t piece, pieces, g_rows, g_width, out_width;
    int32_t dx_tile, dx_slices, dw_tile, dw_slices, logit_tile;
    int64_t x_copy, w_copy, x_weighted, g, dx_slab, dw_slab, stats, label, weights;   // bytes
    Plan(int64_t rows, int64_t vocab, int32_t dim, int32_t dtype, bool x_fits, bool w_fits, bool backward)
    {
        parts = dtype == BMTK_F32 ? 3 : 1;
        combinations = parts == 3 ? 6 : 1;
        depth = (int32_t)up(dim, kDepth);
        small = small_vocab(rows, vocab, dim, dtype, x_fits, w_fits, backward);
        few = !small && rows <= few_most(dtype, w_fits, backward);
        copy_x = parts == 3 || !x_fits;
        copy_w = parts == 3 || !w_fits;
        x_copy = w_copy = x_weighted = g = dx_slab = dw_slab = stats = label = weights = 0;
        pieces = 1, piece = vocab, g_rows = g_width = out_width = 0;
        dx_tile = dx_slices = dw_tile = dw_slices = logit_tile = 0;
        if (small) {
            if (!backward) return;
            out_width = up(dim, 8);
            weights = up(rows * 12 + 8 + kLargest * 4, 256);
            const int32_t j = small_tiles(vocab);
            g = up(up(rows, 64) * j * 16 * 4, 256);
            // slices of the rows, each with sums of its own for d_weight: as many workgroups as the chip holds at once, one or two a compute unit of eight or four tiles of the
            // vocabulary (us both ways of 1,024, 512, 256 workgroups: 19,200 x 100 x 64 fp32 60, 56, 47; 20,000 x 64 x 2,000 303, 292, 294), but of eight tiles and many channels
            // (20,000 x 128 x 2,000 fp32 546, 605, 692); slabs of up to 64 MB
            const int64_t fill = j == 8 ? (dim <= 512 ? 256 : 1024) : j == 4 ? 512 : 1024;
            int64_t s = div_up(fill, div_up(dim, j == 8 ? 32 : 64));
            const int64_t most = (int64_t{64} << 20) / (vocab * out_width * 4);
            s = s > most ? most : s;
            s = s < 1 ? 1 : s;
            piece = up(div_up(rows, s), 64);
            dw_slices = (int32_t)div_up(rows, piece);
            dw_slab = up(dw_slices * vocab * out_width * 4, 256);
            return;
        }
        if (!backward) {
            logit_tile = tile_of(vocab, rows);
            label = up(rows * 4, 256);
            if (few) {
                stats = up(div_up(vocab, 32) * rows * 8, 256);
                return;
            }
            stats = up(div_up(vocab, logit_tile) * rows * 8, 256);
            x_copy = copy_x ? up(parts * rows * depth * 2, 256) : 0;
            w_copy = copy_w ? up(parts * vocab * depth * 2, 256) : 0;
            return;
        }
        out_width = up(dim, 8);
        weights = up(rows * 12 + 8 + kLargest * 4, 256);
        if (few) {
            // slices of the vocabulary, each with sums of its own for dx: as many workgroups as fill the chip some times, slabs of up to 64 MB
            g = up(up(vocab, 128) * (rows <= 16 ? 16 : rows <= 32 ? 32 : 64) * 4, 256);
            int64_t s = div_up(2048, div_up(dim, 256));
            const int64_t most = (int64_t{64} << 20) / (rows * out_width * 4);
            s = s > most ? most : s;
            s = s < 1 ? 1 : s;
            piece = up(div_up(vocab, s), 16);
            dx_slices = (int32_t)div_up(vocab, piece);
            dx_slab = up(dx_slices * rows * out_width * 4, 256);
            return;
        }
        x_copy = copy_x ? up(parts * rows * depth * 2, 256) : 0;
        w_copy = copy_w ? up(parts * vocab * depth * 2, 256) : 0;
        g_rows = up(rows, 256);
        const int64_t most = kPieceBytes / (parts * g_rows * 2) / 256 * 256;
        piece = most < 256 ? 256 : most;
        if (piece > vocab) piece = vocab;
        pieces = div_up(vocab, piece);
        piece = up(div_up(vocab, pieces), 256);
        pieces = div_up(vocab, piece);
        g_width = piece;
        logit_tile = tile_of(piece < vocab ? piece : vocab, rows);
        g = up(parts * g_rows * g_width * 2, 256);
        x_weighted = up(parts * up(rows, kDepth) * out_width * 2, 256);
        const auto slices_of = [](int64_t ni, int64_t nj, int64_t steps, int32_t &tile, int32_t &slices) {
            // the sum over k in as many parts as fill the chip, of eight steps at least
            const auto wanted = [&](int64_t t, int64_t fill) {
                const int64_t tiles = div_up(ni, t) * div_up(nj, t), s = fill / tiles;
                const int64_t most = div_up(steps, 8);
                return s < 1 ? 1 : s > most ? most : s;
            };
            const int64_t large = wanted(256, 256);
            tile = tile_of(ni, nj, large);
            slices = (int32_t)(tile == 256 ? large : wanted(128, 512));
        };
        const int64_t columns = piece < vocab ? piece : vocab;
        slices_of(dim, rows, div_up(columns, kDepth) * combinations, dx_tile, dx_slices);
        slices_of(dim, columns, div_up(rows, kDepth) * combinations, dw_tile, dw_slices);
        dx_slab = up(dx_slices * rows * out_width * 4, 256);
        dw_slab = dw_slices > 1 ? up(dw_slices * columns * out_width * 4, 256) : 0;
    }
    int64_t bytes() const { return x_copy + w_copy + x_weighted + g + dx_slab + dw_slab + stats + label + weights; }
};

bool sizes_fit(int64_t rows, int64_t vocab, int64_t dim, int32_t dtype)
{
    return rows > 0 && vocab > 0 && dim > 0 && dtype >= 0 && dtype <= 2 && rows < (1 << 22) && vocab < (1 << 28) && dim <= 65536;
}

// whether rows can be read 16 bytes at a time, and offsets within a tile of 256 of them are in 32 bits
bool fits(const void *p, int64_t stride, int32_t dim, int32_t dtype) { return dtype != BMTK_F32 && dim % 8 == 0 && aligned(p, 16) && stride % 8 == 0 && stride < (1 << 21); }

template <typename E, typename T, bool AK, bool BK, int Mode>
void multiply(Product &p, int32_t tile, hipStream_t s)
{
    p.tiles_i = (int32_t)div_up(p.ni, tile);
    p.tiles_j = (int32_t)div_up(p.nj, tile);
    const uint32_t jobs = (uint32_t)p.tiles_i * p.tiles_j * p.slices;
    // (a compute unit holds one workgroup of the large tiles, two of the small ones)
    if (tile == 256) product_kernel<E, T, 4, AK, BK, Mode><<<jobs < 256 ? jobs : 256, 256, 0, s>>>(p);
    else product_kernel<E, T, 2, AK, BK, Mode><<<jobs < 512 ? jobs : 512, 256, 0, s>>>(p);
}

template <typename T>
void lay(const void *from, int64_t stride, int64_t rows, int32_t n, int64_t width, int64_t padded_rows, void *to, const float *by, const float *reach, hipStream_t s)
{
    typedef typename Element<T>::type E;
    lay_kernel<T, E><<<(uint32_t)div_up(padded_rows * width / 8, 256), 256, 0, s>>>(static_cast<const T *>(from), stride, rows, n, (int32_t)width, padded_rows, static_cast<E *>(to), by, reach);
}

// Few rows of the weights leave the chip empty where a wavefront takes 32 of them: then a workgroup's wavefronts share them, four or eight.
int32_t few_split(int64_t vocab) { return vocab >= 32 * 2048 ? 1 : vocab >= 32 * 512 ? 4 : 8; }
int32_t few_tiles(int64_t vocab) { return (int32_t)div_up(vocab, few_split(vocab) == 1 ? 128 : 32); }

template <typename T, int J, bool Gradient>
void few_rows(const Few &f, hipStream_t s)
{
    const uint32_t tiles = (uint32_t)few_tiles(f.vocab);
    switch (few_split(f.vocab)) {
        case 1: few_rows_kernel<T, J, 1, Gradient><<<tiles, 256, 0, s>>>(f); break;
        case 4: few_rows_kernel<T, J, 4, Gradient><<<tiles, 256, 0, s>>>(f); break;
        default: few_rows_kernel<T, J, 8, Gradient><<<tiles, 512, 0, s>>>(f);
    }
}

template <typename T, int J, bool Gradient>
void small_rows(const Small &m, hipStream_t s)
{
    switch (small_split(m.rows, m.dim)) {
        case 1: small_kernel<T, J, 1, Gradient><<<(uint32_t)div_up(m.rows, 128), 256, 0, s>>>(m); break;
        case 4: small_kernel<T, J, 4, Gradient><<<(uint32_t)div_up(m.rows, 32), 256, 0, s>>>(m); break;
        default: small_kernel<T, J, 8, Gradient><<<(uint32_t)div_up(m.rows, 16), 512, 0, s>>>(m);
    }
}

template <typename T, bool Gradient>
void small_any(const Small &m, hipStream_t s)
{
    switch (small_tiles(m.vocab)) {
        case 1: return small_rows<T, 1, Gradient>(m, s);
        case 2: return small_rows<T, 2, Gradient>(m, s);
        case 4: return small_rows<T, 4, Gradient>(m, s);
        default: return small_rows<T, 8, Gradient>(m, s);
    }
}

struct Call {
    int64_t rows, vocab, x_stride, w_stride, ignore;
    int32_t dim, dtype;
    const void *x, *weight;
    const int64_t *tokens;
    char *ws;
    hipStream_t stream;
    char *next(int64_t bytes)
    {
        char *p = ws;
        ws += bytes;
        return p;
    }
};

// rows of n numbers, `stride` apart, as an operand: their numbers as k, or the rows
Source by_numbers(const char *p, int64_t stride, int64_t part, int64_t rows, int64_t n) { return {p, stride * 2, part * 2, kDepth * 2, ((rows - 1) * stride + n) * 2, 128}; }
Source by_rows(const char *p, int64_t stride, int64_t part, int64_t rows, int64_t n) { return {p, stride * 2, part * 2, kDepth * stride * 2, ((rows - 1) * stride + n) * 2, 128}; }

// logits as a product: i the vocabulary from `first` on, j the rows
template <typename T>
Product logits(const Call &c, const Plan &plan, const char *x, const char *w, int64_t first, int64_t count)
{
    Product p{};
    const int64_t w_stride = plan.copy_w ? plan.depth : c.w_stride, x_stride = plan.copy_x ? plan.depth : c.x_stride;
    p.a = by_numbers(w + first * w_stride * 2, w_stride, c.vocab * plan.depth, count, plan.copy_w ? plan.depth : c.dim);
    p.b = by_numbers(x, x_stride, c.rows * plan.depth, c.rows, plan.copy_x ? plan.depth : c.dim);
    // (copies have zeros behind the rows' channels; what lies there of an operand that is read as it is may be NaN, whatever the other one has)
    p.tail = plan.copy_x && plan.copy_w ? kDepth : c.dim - (plan.depth - kDepth);
    p.ni = (int32_t)count, p.nj = (int32_t)c.rows;
    p.steps = plan.depth / kDepth, p.combinations = plan.combinations, p.slices = 1;
    p.rotate = p.tail == kDepth;
    p.first = (int32_t)first, p.vocab = (int32_t)c.vocab, p.tokens = c.tokens, p.ignore = c.ignore;
    return p;
}

template <typename T>
void forward(Call c, float *logp, float *lse, float *peak, float *total)
{
    typedef typename Element<T>::type E;
    const bool x_fits = fits(c.x, c.x_stride, c.dim, c.dtype), w_fits = fits(c.weight, c.w_stride, c.dim, c.dtype);
    const Plan plan(c.rows, c.vocab, c.dim, c.dtype, x_fits, w_fits, false);
    if (plan.small) {
        Small m{};
        m.x = c.x, m.weight = c.weight, m.tokens = c.tokens, m.x_stride = c.x_stride, m.w_stride = c.w_stride, m.ignore = c.ignore;
        m.rows = (int32_t)c.rows, m.vocab = (int32_t)c.vocab, m.dim = c.dim, m.logp = logp, m.lse = lse, m.peak = peak, m.total = total;
        return small_any<T, false>(m, c.stream);
    }
    float2 *stats = reinterpret_cast<float2 *>(c.next(plan.stats));
    float *label = reinterpret_cast<float *>(c.next(plan.label));
    int32_t tiles;
    if (plan.few) {
        Few f{};
        f.x = c.x, f.weight = c.weight, f.tokens = c.tokens, f.x_stride = c.x_stride, f.w_stride = c.w_stride, f.rows = (int32_t)c.rows, f.vocab = (int32_t)c.vocab, f.dim = c.dim;
        f.stats = stats, f.label = label;
        tiles = few_tiles(c.vocab);
        if (c.rows <= 16) few_rows<T, 1, false>(f, c.stream);
        else if (c.rows <= 32) few_rows<T, 2, false>(f, c.stream);
        else few_rows<T, 4, false>(f, c.stream);
        few_join_kernel<<<(uint32_t)c.rows, 256, 0, c.stream>>>(stats, tiles, (int32_t)c.rows, label, c.tokens, c.ignore, (int32_t)c.vocab, logp, lse, peak, total);
        return;
    } else {
        const char *x = static_cast<const char *>(c.x), *w = static_cast<const char *>(c.weight);
        if (plan.copy_x) {
            char *to = c.next(plan.x_copy);
            lay<T>(c.x, c.x_stride, c.rows, c.dim, plan.depth, c.rows, to, nullptr, nullptr, c.stream);
            x = to;
        }
        if (plan.copy_w) {
            char *to = c.next(plan.w_copy);
            lay<T>(c.weight, c.w_stride, c.vocab, c.dim, plan.depth, c.vocab, to, nullptr, nullptr, c.stream);
            w = to;
        }
        Product p = logits<T>(c, plan, x, w, 0, c.vocab);
        p.stats = stats, p.label = label;
        multiply<E, T, false, false, kStats>(p, plan.logit_tile, c.stream);
        tiles = p.tiles_i;
    }
    stats_join_kernel<<<(uint32_t)div_up(c.rows, 64), 1024, 0, c.stream>>>(stats, tiles, (int32_t)c.rows, label, c.tokens, c.ignore, (int32_t)c.vocab, logp, lse, peak, total);
}

template <typename T>
void join_slabs(const float *slab, int32_t slabs, int64_t slab_size, int64_t rows, int32_t n, int64_t width, const float *by, const float *factor, const float *reach, float scale, void *out, hipStream_t s)
{
    const int32_t ways = slabs <= 4 ? 1 : slabs < 64 ? 4 : 16;
    const uint32_t waves = ways == 16 ? 16 : 4;
    slab_join_kernel<T><<<(uint32_t)div_up(rows * (width / 4), 64 * (waves / ways)), waves * kWave, 0, s>>>(slab, slabs, slab_size, rows, n, (int32_t)width, ways, by, factor, reach, scale,
                                                                                                          static_cast<T *>(out));
}

template <typename T, int J>
void few_backward(const Few &f, hipStream_t s)
{
    few_rows<T, J, true>(f, s);
    few_back_kernel<T, J, 4, false><<<dim3((uint32_t)div_up(f.dim, 256), (uint32_t)f.slices), 256, 0, s>>>(f);
}

template <typename T>
void backward(Call c, const float *peak, const float *total, const float *d_logp, void *dx, void *d_weight)
{
    typedef typename Element<T>::type E;
    const bool x_fits = fits(c.x, c.x_stride, c.dim, c.dtype), w_fits = fits(c.weight, c.w_stride, c.dim, c.dtype);
    const Plan plan(c.rows, c.vocab, c.dim, c.dtype, x_fits, w_fits, true);
    const bool half = std::is_same<T, f16>::value;
    // fp16: p down to 2^-38 keeps bits (its subnormals are not lost in the matrix instructions), and G, up to 2, stays below the largest
    const float g_scale = half ? 16384.0f : 1.0f;
    float2 *shares = reinterpret_cast<float2 *>(c.next(plan.weights));
    float *weights = reinterpret_cast<float *>(shares + c.rows), *factor = weights + c.rows, *reach = factor + 1;
    char *g = c.next(plan.g), *x_weighted = c.next(plan.x_weighted);
    float *dx_slab = reinterpret_cast<float *>(c.next(plan.dx_slab)), *dw_slab = reinterpret_cast<float *>(c.next(plan.dw_slab));
    // (nothing of fp32 is rounded by which the largest d_logp would matter: of a small vocabulary its shares are made beside G)
    const bool beside = plan.small && c.dtype == BMTK_F32;
    float *parts = !beside && !plan.few && c.rows > 32768 ? factor + 2 : nullptr;
    if (parts) largest_kernel<<<kLargest, 1024, 0, c.stream>>>(d_logp, c.tokens, c.ignore, c.rows, parts);
    if (!beside)
        weigh_kernel<<<(uint32_t)div_up(c.rows, 1024), 1024, 0, c.stream>>>(d_logp, c.tokens, c.ignore, c.rows, (int32_t)c.vocab, peak, total, g_scale, weights,
                                                                            plan.few ? nullptr : shares, factor, reach, parts);
    if constexpr (std::is_same<T, f16>::value) {
        if (!plan.few) {
            const int64_t groups = div_up(c.rows * div_up(c.dim, 8), 1024);
            reach_kernel<<<(uint32_t)(groups < 256 ? groups : 256), 1024, 0, c.stream>>>(static_cast<const f16 *>(c.x), c.x_stride, c.rows, c.dim, weights, reach);
        }
    } else {
        reach = nullptr;
    }
    if (plan.small) {
        Small m{};
        m.x = c.x, m.weight = c.weight, m.tokens = c.tokens, m.x_stride = c.x_stride, m.w_stride = c.w_stride, m.ignore = c.ignore;
        m.rows = (int32_t)c.rows, m.vocab = (int32_t)c.vocab, m.dim = c.dim, m.peak = const_cast<float *>(peak), m.total = const_cast<float *>(total);
        m.d_logp = d_logp, m.g = g, m.weights = weights, m.shares = beside ? nullptr : shares;
        small_any<T, true>(m, c.stream);
        Few f{};
        f.x = c.weight, f.weight = c.x, f.x_stride = c.w_stride, f.w_stride = c.x_stride, f.rows = (int32_t)c.vocab, f.vocab = (int32_t)c.rows, f.dim = c.dim;
        f.weights = weights, f.g = reinterpret_cast<float *>(g), f.d_weight = dx, f.slab = dw_slab, f.slices = plan.dw_slices, f.slice_rows = (int32_t)plan.piece;
        f.factor = beside ? nullptr : factor, f.reach = reach, f.g_unit = 1.0f / g_scale;
        const int32_t j = small_tiles(c.vocab);
        const dim3 grid((uint32_t)div_up(c.dim, j == 8 ? 32 : 64), (uint32_t)f.slices);
        // (a lane has two channels instead of four where there are eight tiles of the vocabulary: registers)
        if (j == 1) few_back_kernel<T, 1, 4, true><<<grid, 256, 0, c.stream>>>(f);
        else if (j == 2) few_back_kernel<T, 2, 4, true><<<grid, 256, 0, c.stream>>>(f);
        else if (j == 4) few_back_kernel<T, 4, 4, true><<<grid, 256, 0, c.stream>>>(f);
        else few_back_kernel<T, 8, 2, true><<<grid, 256, 0, c.stream>>>(f);
        join_slabs<T>(dw_slab, plan.dw_slices, c.vocab * plan.out_width, c.vocab, c.dim, plan.out_width, nullptr, f.factor, reach, -f.g_unit, d_weight, c.stream);
        return;
    }
    if (plan.few) {
        Few f{};
        f.x = c.x, f.weight = c.weight, f.tokens = c.tokens, f.x_stride = c.x_stride, f.w_stride = c.w_stride, f.rows = (int32_t)c.rows, f.vocab = (int32_t)c.vocab, f.dim = c.dim;
        f.peak = peak, f.total = total, f.weights = weights, f.ignore = c.ignore, f.g = reinterpret_cast<float *>(g), f.d_weight = d_weight, f.slab = dx_slab;
        f.slices = plan.dx_slices, f.slice_rows = (int32_t)plan.piece;
        if (c.rows <= 16) few_backward<T, 1>(f, c.stream);
        else if (c.rows <= 32) few_backward<T, 2>(f, c.stream);
        else few_backward<T, 4>(f, c.stream);
        join_slabs<T>(dx_slab, plan.dx_slices, c.rows * plan.out_width, c.rows, c.dim, plan.out_width, weights, nullptr, nullptr, -1.0f, dx, c.stream);
        return;
    }
    const char *x = static_cast<const char *>(c.x), *w = static_cast<const char *>(c.weight);
    if (plan.copy_x) {
        char *to = c.next(plan.x_copy);
        lay<T>(c.x, c.x_stride, c.rows, c.dim, plan.depth, c.rows, to, nullptr, nullptr, c.stream);
        x = to;
    }
    if (plan.copy_w) {
        char *to = c.next(plan.w_copy);
        lay<T>(c.weight, c.w_stride, c.vocab, c.dim, plan.depth, c.vocab, to, nullptr, nullptr, c.stream);
        w = to;
    }
    const int64_t k_rows = up(c.rows, kDepth);
    lay<T>(c.x, c.x_stride, c.rows, c.dim, plan.out_width, k_rows, x_weighted, weights, reach, c.stream);
    for (int64_t q = 0; q < plan.pieces; ++q) {
        const int64_t first = q * plan.piece, count = c.vocab - first < plan.piece ? c.vocab - first : plan.piece;
        Product p = logits<T>(c, plan, x, w, first, count);
        p.peak = peak, p.shares = shares, p.g = g, p.g_block = plan.g_rows * 64, p.g_part = plan.g_rows * plan.g_width;
        multiply<E, T, false, false, kGradient>(p, plan.logit_tile, c.stream);

        // dx: i a channel, j a row, k the vocabulary
        Product d{};
        d.a = by_rows(p.a.p, p.a.stride / 2, p.a.part / 2, count, plan.copy_w ? plan.depth : c.dim);
        d.b = {g, 128, p.g_part * 2, plan.g_rows * 128, p.g_part * 2, 0};
        d.ni = c.dim, d.nj = (int32_t)c.rows;
        d.steps = (int32_t)div_up(count, kDepth), d.combinations = plan.combinations;
        // (a last piece may have fewer steps than there are slabs, and a slice without one would take its neighbour's: the other slabs keep the sums that they have)
        const int64_t steps = (int64_t)d.steps * d.combinations;
        d.slices = (int32_t)(steps < plan.dx_slices ? steps : plan.dx_slices);
        d.slab = dx_slab, d.slab_stride = plan.out_width, d.slab_size = c.rows * plan.out_width, d.add = q > 0;
        multiply<E, T, true, false, kSlab>(d, plan.dx_tile, c.stream);

        // d_weight: i a channel, j the vocabulary, k a row
        Product e{};
        e.a = by_rows(x_weighted, plan.out_width, k_rows * plan.out_width, k_rows, plan.out_width);
        e.b = {g, 128, p.g_part * 2, kDepth * 128, p.g_part * 2, plan.g_rows * 128};
        e.ni = c.dim, e.nj = (int32_t)count;
        e.steps = (int32_t)(k_rows / kDepth), e.combinations = plan.combinations, e.slices = plan.dw_slices;
        T *out = static_cast<T *>(d_weight) + first * c.dim;
        e.out = out, e.factor = factor, e.reach = reach, e.out_scale = -1.0f / g_scale;
        e.slab = dw_slab, e.slab_stride = plan.out_width, e.slab_size = count * plan.out_width;
        if (plan.dw_slices == 1) {
            multiply<E, T, true, true, kOut>(e, plan.dw_tile, c.stream);
        } else {
            multiply<E, T, true, true, kSlab>(e, plan.dw_tile, c.stream);
            join_slabs<T>(dw_slab, plan.dw_slices, e.slab_size, count, c.dim, plan.out_width, nullptr, factor, reach, e.out_scale, out, c.stream);
        }
    }
    join_slabs<T>(dx_slab, plan.dx_slices, c.rows * plan.out_width, c.rows, c.dim, plan.out_width, weights, factor, nullptr, -1.0f / g_scale, dx, c.stream);
}

int check(const char *name, const Call &c, bool backward)
{
    BMTK_REQUIRE(c.rows > 0 && c.vocab > 0 && c.dim > 0, "%s: sizes must be positive", name);
    BMTK_REQUIRE(c.dtype >= 0 && c.dtype <= 2, "%s: unknown type %d", name, c.dtype);
    BMTK_REQUIRE(c.rows < (1 << 22), "%s: rows must be below 2^22", name);
    BMTK_REQUIRE(c.vocab < (1 << 28), "%s: vocab must be below 2^28", name);
    BMTK_REQUIRE(c.dim <= 65536, "%s: up to 65,536 channels", name);
    BMTK_REQUIRE(c.x_stride >= 0 && c.w_stride >= 0, "%s: strides must not be negative", name);
    // (a launch has up to 2^32 threads: of eight numbers where operands are laid out anew, of four where dx is put together)
    BMTK_REQUIRE(up(c.vocab, 256) * up(c.dim, 64) < (int64_t{1} << 35) && up(c.rows, 256) * up(c.dim, 64) < (int64_t{1} << 34), "%s: too many numbers for a launch", name);
    BMTK_REQUIRE(div_up(c.rows, 128) * div_up(c.vocab, 128) < (int64_t{1} << 31), "%s: too many logits for a launch", name);
    BMTK_REQUIRE(c.ws || !Plan(c.rows, c.vocab, c.dim, c.dtype, fits(c.x, c.x_stride, c.dim, c.dtype), fits(c.weight, c.w_stride, c.dim, c.dtype), backward).bytes(),
                 "%s: needs a workspace", name);
    return 0;
}

}  // namespace
}  // namespace bmtk

using namespace bmtk;

extern "C" int64_t bmtk_projected_logprobs_workspace_bytes(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void *x, int64_t x_stride, const void *weight,
                                                           int64_t weight_stride, int32_t backward)
{
    if (!sizes_fit(rows, vocab, dim, dtype)) return 0;
    return Plan(rows, vocab, dim, dtype, fits(x, x_stride, dim, dtype), fits(weight, weight_stride, dim, dtype), backward != 0).bytes();
}

extern "C" int bmtk_projected_logprobs_fwd(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void *x, int64_t x_stride, const void *weight, int64_t weight_stride,
                                           const int64_t *tokens, int64_t ignore, float *logp, float *lse, float *peak, float *total, void *workspace, void *stream)
{
    BMTK_REQUIRE(x && weight && tokens && logp && lse && peak && total, "projected_logprobs_fwd: null pointer");
    const Call c{rows, vocab, x_stride, weight_stride, ignore, dim, dtype, x, weight, tokens, static_cast<char *>(workspace), static_cast<hipStream_t>(stream)};
    if (const int failed = check("projected_logprobs_fwd", c, false)) return failed;
    BMTK_BY_TYPE(dtype, T, { forward<T>(c, logp, lse, peak, total); });
    BMTK_CHECK_LAUNCH("projected_logprobs_fwd");
    return 0;
}

extern "C" int bmtk_projected_logprobs_bwd(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void *x, int64_t x_stride, const void *weight, int64_t weight_stride,
                                           const int64_t *tokens, int64_t ignore, const float *peak, const float *total, const float *d_logp, void *dx, void *d_weight, void *workspace,
                                           void *stream)
{
    BMTK_REQUIRE(x && weight && tokens && peak && total && d_logp && dx && d_weight, "projected_logprobs_bwd: null pointer");
    const Call c{rows, vocab, x_stride, weight_stride, ignore, dim, dtype, x, weight, tokens, static_cast<char *>(workspace), static_cast<hipStream_t>(stream)};
    if (const int failed = check("projected_logprobs_bwd", c, true)) return failed;
    BMTK_BY_TYPE(dtype, T, { backward<T>(c, peak, total, d_logp, dx, d_weight); });
    BMTK_CHECK_LAUNCH("projected_logprobs_bwd");
    return 0;
}
