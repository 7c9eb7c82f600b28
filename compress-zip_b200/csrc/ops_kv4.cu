// ops_kv4.cu -- the key/value cache held in 4 bits (include/czg_ops.h): append, read
// and attention.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "ops_kv4.cuh"
#include "tc_common.cuh"

namespace czg {
namespace {

// x (finite) as bf16 rounded towards minus / plus infinity.  A bf16 is the high half of a
// float's bits: dropping the low half rounds towards zero, one more step away from it.
__device__ __forceinline__ float bf16_down(float x) {
    uint32_t u = __float_as_uint(x);
    if (u & 0xFFFFu) u = (u & 0x80000000u ? u + 0x10000u : u) & 0xFFFF0000u;
    return __uint_as_float(u);
}
__device__ __forceinline__ float bf16_up(float x) {
    uint32_t u = __float_as_uint(x);
    if (u & 0xFFFFu) u = (u & 0x80000000u ? u : u + 0x10000u) & 0xFFFF0000u;
    return __uint_as_float(u);
}

struct Strides { int64_t b, t, h; };

constexpr float kFltMax = 3.402823466e38f;

// D / 4 lanes a row (a warp takes 128 / D rows side by side), four values each: the row's
// range by shuffles, then the codes.  4096 rows of D = 64: 5 us, latency.  lo is rounded down and step up (each operation with
// the same direction), so every quotient lies in [0, 15].  A key's row and its value's are
// neighbours.  CTA 0 looks for repeated slots.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv4_append(czg_kv4 c, const T *k, Strides ks, const T *v,
                                                    Strides vs, int vec, const int32_t *slots,
                                                    const int32_t *lengths, int b, int t) {
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0) {
        kv4_check_distinct(c, slots, b);
        return;
    }
    constexpr int LR = D / 4;
    const uint32_t id = (blockIdx.x - 1) * (256 / LR) + threadIdx.x / LR, part = threadIdx.x % LR;
    const uint32_t row = id >> 1;   // fewer than 2^31 of them (checked by the host)
    uint32_t s = 0, i = 0, h = 0;
    bool there = row < (uint32_t)b * t * c.n_heads;
    int slot = -1;
    int64_t entry = 0;
    if (there) {
        const uint32_t of_t = c.n_heads == 1 ? row : row / c.n_heads;
        h = row - of_t * c.n_heads;
        s = t == 1 ? of_t : of_t / t;
        i = of_t - s * t;
        const bool first = part == 0 && h == 0 && (id & 1) == 0;
        slot = kv4_slot(c, slots, s, first);
        const int n = lengths[s];
        entry = (int64_t)n - t + i;
        if (slot >= 0 && first && (n < 0 || entry >= c.capacity)) atomicOr(c.status, CZG_KV4_BAD_LENGTH);
        there = slot >= 0 && entry >= 0 && entry < c.capacity;
    }
    const Strides &st = id & 1 ? vs : ks;
    const T *src = (id & 1 ? v : k) + (there ? s * st.b + i * st.t + h * st.h : 0) + part * 4;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (there && vec) {
        __align__(16) T y[4];
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(src);
        else *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = to_f32(y[j]);
    } else if (there) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = to_f32(src[j]);
    }
    float lo = INFINITY, hi = -INFINITY;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        fine &= fabsf(x[j]) <= kFltMax;
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
    if (!fine) hi = INFINITY;   // NaN too: the row's range is not finite
#pragma unroll
    for (int o = 1; o < LR; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (!there) return;
    lo = bf16_down(lo);
    float step = bf16_up(__fdiv_ru(__fsub_ru(hi, lo), 15.0f));
    if (!(fabsf(lo) <= kFltMax) || !(step <= kFltMax)) step = lo = NAN;
    uint32_t code = 0;
    if (step > 0.0f) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            code |= (__float_as_uint(__fadd_rn(__fdiv_rn(__fsub_rn(x[j], lo), step), kM1)) & 15u) << (4 * j);   // rounded by the sum
    }
    const int64_t at = kv4_row(c, slot, h, (int)entry);
    reinterpret_cast<uint16_t *>((id & 1 ? c.v : c.k) + at * (D / 2))[part] = (uint16_t)code;
    if (part == 0) {
        const uint32_t range = __float_as_uint(step) >> 16 | (__float_as_uint(lo) & 0xFFFF0000u);   // both are bf16
        reinterpret_cast<uint32_t *>(static_cast<KvScale *>(c.scales) + at)[id & 1] = range;
        if (c.weights && (id & 1) == 0) c.weights[at] = 0.0f;
    }
}

// D / 8 threads a row, 8 codes of its key and 8 of its value each; a thread takes two rows.
// Bound by its writes: 48 x 1024 entries of 8 heads (D = 128, 54 MB read, 201 MB written)
// take 47 us, 5.4 TB/s.  (16 codes a thread, whose 32 bytes are written in two halves, were
// as fast; a grid row a sequence took twice as long for 4096 sequences of one entry.)
template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv4_read(czg_kv4 c, const int32_t *slots,
                                                  const int32_t *starts, uint32_t rows, uint32_t all,
                                                  T *__restrict__ k_out, T *__restrict__ v_out) {
    constexpr int P = D / 8, N = 2;
    pdl_wait();
    pdl_trigger();
    const int part = threadIdx.x % P;
    uint2 range[N];
    uint32_t codes[N][2];
    bool there[N];
    const uint32_t row0 = blockIdx.x * (N * 256 / P) + threadIdx.x / P;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t row = row0 + i * (256 / P);
        there[i] = false;
        range[i] = make_uint2(0, 0);
        codes[i][0] = codes[i][1] = 0;
        if (row >= all) continue;
        const uint32_t s = row / rows, of = row - s * rows, place = c.n_heads == 1 ? of : of / c.n_heads, h = of - place * c.n_heads;
        const bool first = part == 0 && h == 0;
        const int slot = kv4_slot(c, slots, s, first);
        const int64_t entry = (int64_t)starts[s] + place;
        there[i] = slot >= 0 && entry >= 0 && entry < c.capacity;
        if (slot >= 0 && !there[i] && first) atomicOr(c.status, CZG_KV4_BAD_LENGTH);
        if (!there[i]) continue;
        const int64_t at = kv4_row(c, slot, h, (int)entry);
        range[i] = *reinterpret_cast<const uint2 *>(static_cast<const KvScale *>(c.scales) + at);
        if (k_out) codes[i][0] = reinterpret_cast<const uint32_t *>(c.k + at * (D / 2))[part];
        if (v_out) codes[i][1] = reinterpret_cast<const uint32_t *>(c.v + at * (D / 2))[part];
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t row = row0 + i * (256 / P);
        if (row >= all) continue;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            T *out = w ? v_out : k_out;
            if (!out) continue;
            const uint32_t r = w ? range[i].y : range[i].x;
            const float step = __uint_as_float(r << 16), lo = __uint_as_float(r & 0xFFFF0000u);
            __align__(16) T y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // a code under the bits of 2^23 is 2^23 + code
                const float code = __fsub_rn(__uint_as_float((codes[i][w] >> (4 * j) & 15u) | 0x4B000000u), 8388608.0f);
                y[j] = from_f32<T>(__fmaf_rn(step, code, lo));
            }
            uint4 *dst = reinterpret_cast<uint4 *>(out + (int64_t)row * D + 8 * part);
            const uint4 *src = reinterpret_cast<const uint4 *>(y);
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; j++) dst[j] = src[j];
        }
    }
}

// ---- attention ---------------------------------------------------------------------------
//
// A CTA takes one unit of a sequence's entries (unit_of its length, at a fixed place
// whatever the batch), one key head and up to 8 NB rows (query heads of that key head, times the
// call's rows).  Its two or four warps take tiles of kTile entries in turn, each through a ring of
// its own that TMA fills (swizzled for ldmatrix); many such small CTAs share an SM and
// cover one another's beginnings and ends.
//
// Products are on mma.sync m16n8k16 (fp16, fp32 sums) with the cache as the A operand and
// the rows as N: 8 rows fill an MMA, where tcgen05 would need 64 or 128 and the codes
// unpacked to shared memory first.  A nibble becomes an fp16 number by one AND: bits
// 0x000n are the subnormal n 2^-24, bits 0x00n0 are 16 n 2^-24, exactly, and the powers of
// two go into the factors outside.  One word of 8 codes takes a shift and four ANDs:
//   K: ldmatrix gives a lane 8 dimensions of entries i and i + 8; the pairs (0, 4), (1, 5),
//      (2, 6), (3, 7) are the k of two MMAs (the query is permuted alike, and its share of
//      the high nibbles divided by 16);
//   V: ldmatrix.trans gives a lane 4 dimensions of entries 2c, 2c + 1: nibble i of both is
//      the pair of dimension 4g + i (for odd i the byte, taken apart at the end).
// With x = lo + step c:  s_j = step_j (q.c_j) + lo_j sum(q);  out = sum p_j step_j c_j + sum p_j lo_j.
// The query is held in fp16 after a power of two that brings its largest value to
// [2^13, 2^14): exact but for values below 2^-23 of the largest.  p_j step_j is
// held in fp16 likewise: off by 2^-11 of itself, against 2^-8 of a bf16 result (for an fp16 one
// in two parts, to 2^-22), and by no less than 2^-25.  Where the steps of a unit are alike, all
// are brought to one power of two, 2^7 to 2^15 for the largest step at the largest p_j; where
// some entry's step and lower end are both below 2^-6 of the largest step, an entry far below
// (or one that a row does not see at all) could push those that count out of fp16's range,
// and each row has a power of two of its own, which follows its largest p_j step_j.  Either
// power of two is the step's alone: the sums of p_j and of p_j lo_j are of plain weights, up to
// 2^8, so that neither their overflow nor what ex2 takes for 0 (weights below 2^-126) depends
// on the steps.  Scores, maxima and sums are fp32; exponentials are ex2.approx (2^-22).
//
// Measured: one sequence of 131,071 entries, 32 heads on 8, D = 128, bf16 (143 MB): 37 us with
// the join, 3.8 TB/s; 4096 sequences of up to 512, 6 heads on 1, D = 64 (84 MB): 33.5 us.  The
// loads alone take 25 and 21 us (the second mostly the CTAs' beginnings and ends).  No pipe is
// full (ALU 44%, DRAM 49% and 28%, 18% and 26% of the warps active): loads, arithmetic, half of
// it unpacking on the half-rate ALU pipe, and a CTA's ends overlap too little.  Units whose rows
// scale their weights themselves take a quarter to a third more (46.6 and 45.1 us).  Tiles of 32
// entries and two stages hold the most CTAs on an SM (8 at D = 128): tiles of 64 took 43 us, three
// and four stages 46 and 47; units of 256 took 7% more, one warp a unit as much.
//
// Between the warps of a CTA, and between units (k_kv4_join), partial results are joined
// in a fixed order, so a row's bits do not depend on the batch or the grid.
constexpr int kChunk = 512, kTile = 32, kRing = 2;
// Entries of a unit of a sequence of n: enough that none has more than kUnits units.
constexpr int kUnits = 128;
__host__ __device__ constexpr int unit_of(int n) {
    int64_t u = kChunk;
    while (u * kUnits < n) u *= 2;
    return (int)u;   // 2^24 at most
}
__host__ __device__ constexpr int attend_warps(int nb) { return nb == 1 ? 2 : 4; }   // more rows, longer tiles: more warps to share a unit

struct AttendArgs {
    czg_kv4 c;
    const void *q;
    Strides qs;
    const int32_t *slots, *lengths;
    int t, g, rows, row_blocks, max_len, units, vec, out_vec, whole;
    uint64_t g_inv;     // 2^32 / g, rounded up: r g_inv / 2^32 is r / g while r g < 2^32
    float scale_log2;   // scale * log2 e
    void *out;
    Strides os;
    // not whole, that is more than one unit (or row block with weights): partial results to join
    float *part;        // [b][head][unit][rows padded][D]
    float4 *stat;       // [b][head][unit][rows padded] (maximum, sum, what a score is multiplied by); the
                        // sum is negative where the partial result is taken kHuge-fold
    float *score;       // weights: [b][head][rows][max_len]
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void add_scaled(float4 &x, float f, float4 v) {
    x.x = __fmaf_rn(f, v.x, x.x);
    x.y = __fmaf_rn(f, v.y, x.y);
    x.z = __fmaf_rn(f, v.z, x.z);
    x.w = __fmaf_rn(f, v.w, x.w);
}
// Four dimensions of a result: x f up.
template <typename T>
__device__ __forceinline__ void store4(T *dst, float4 x, float f, float up, bool vec) {
    __align__(8) T y[4] = {from_f32<T>(x.x * f * up), from_f32<T>(x.y * f * up), from_f32<T>(x.z * f * up), from_f32<T>(x.w * f * up)};
    if (vec) {
        *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) dst[i] = y[i];
    }
}
// What sums taken from the maximum m are worth from the maximum `top` (both may be -infinity).
__device__ __forceinline__ float share(float m, float top) { return m == top ? 1.0f : ex2(m - top); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return done != 0;
}

// Row r of a sequence and key head: place i = r / g of the call's rows, query head h g + r % g.
__device__ __forceinline__ int row_place(const AttendArgs &p, int r) { return (int)((uint64_t)(uint32_t)r * p.g_inv >> 32); }
__device__ __forceinline__ int64_t row_offset(const AttendArgs &p, const Strides &s, int b, int h, int r) {
    const int i = row_place(p, r);
    return b * s.b + i * s.t + (int64_t)((h - i) * p.g + r) * s.h;
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// The smallest power of two that steps are taken to be of: 2^(7 - te) stays inside fp32.
constexpr int kLeastTe = -119;
// A unit whose least entry (its step, or a sixteenth of its lower end) is below the largest step
// by more than this power of two keeps a scale for each row.
constexpr int kAlike = 6;
// Sums of weights (below 2^8) times values below 2^87 stay inside fp32 for 2^31 entries.  Where a
// value of a unit is larger, its values are taken kHuge-fold: below 2^80.
constexpr float kHuge = 3.5527136788005009e-15f;   // 2^-48
constexpr int kHugeTe = 83;                        // 15 steps of 2^te and more may pass 2^87
constexpr uint32_t kHugeLo = (87 + 127) << 7;      // bits of 2^87

// CTAs an SM is to hold: what the sums (D NB / 4 registers), query and scores leave room
// for.  With the weights in two parts (exact) fewer of them spill less (attend of 64
// sequences of up to 4096, 32 heads on 4, D = 128, with weights: 43.4 us, 45.0 with 8).
constexpr int attend_ctas(int d, int nb, bool exact) {
    return d == 64 ? (nb == 1 ? (exact ? 8 : 10) : exact ? 3 : 4) : nb == 1 ? (exact ? 6 : 8) : exact ? 2 : 3;
}

template <int D, int W>
struct AttendSmem {
    static constexpr int kTileCodes = kTile * D / 2;   // of keys, and as many of values behind them
    static constexpr int kScales = W * kRing * 2 * kTileCodes, kBars = kScales + kChunk * 16;
    static constexpr size_t kBytes = 1024 + kBars + W * kRing * 8;
};

template <typename T, int D, int NB, bool TRACK>
__global__ void __launch_bounds__(attend_warps(NB) * 32, attend_ctas(D, NB, DType<T>::kCode == CZG_F16))
k_kv4_attend(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttendArgs p) {
    constexpr int kWarps = attend_warps(NB);
    using L = AttendSmem<D, kWarps>;
    constexpr int CH = D / 32;      // 16-byte chunks of a row of codes
    constexpr int R = 8 * NB, THREADS = kWarps * 32;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float4 *sc = reinterpret_cast<float4 *>(smem + L::kScales);   // a chunk's ranges: k step, k lo, v step, v lo
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + L::kBars);
    __shared__ uint4 s_q[NB * CH * 32];      // the query as B fragments: [nb][chunk][lane]
    __shared__ float2 s_qs[R];               // a row's factors
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    __shared__ uint2 s_top[kWarps];          // bits of a block's largest step, and of the unit's least entry
    __shared__ float2 s_scale[kWarps][R];    // spread: the row's largest weight times step so far, and its power of two
    __shared__ float2 s_row[R];              // maximum and sum over the warps
    __shared__ int64_t s_out[R];             // where the row's output begins

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, c4 = lane & 3;
    const int unit = blockIdx.x, h = p.row_blocks == 1 ? blockIdx.y : blockIdx.y / p.row_blocks, b = blockIdx.z;
    const int rb = blockIdx.y - h * p.row_blocks;
    const bool first = tid == 0 && unit == 0 && blockIdx.y == 0;
    pdl_wait();
    pdl_trigger();   // k_kv4_join may begin to launch
    if (TRACK && unit == 0 && b == 0 && blockIdx.y == 0) kv4_check_distinct(p.c, p.slots, gridDim.z);
    const int slot = kv4_slot(p.c, p.slots, b, first);
    const int n = slot < 0 ? 0 : kv4_length(p.c, p.lengths, b, min(p.max_len, p.c.capacity), first);
    const int len = unit_of(n);
    if (unit > 0 && (int64_t)unit * len >= n) return;
    const int j0 = unit * len, here = min(n - j0, len);   // entries of this unit
    const int64_t base = kv4_row(p.c, max(slot, 0), h, 0);

    // each warp asks for its first tiles
    uint8_t *ring = smem + warp * kRing * 2 * L::kTileCodes;
    uint64_t *ring_bar = bar + warp * kRing;
    auto ask = [&](int it) {   // one lane
        uint8_t *to = ring + (it % kRing) * 2 * L::kTileCodes;
        const int y = j0 + (it * kWarps + warp) * kTile, z = slot * p.c.n_heads + h;
        mbar_expect_tx(&ring_bar[it % kRing], 2 * L::kTileCodes);
        tma_load_3d(to, &map_k, &ring_bar[it % kRing], 0, y, z);
        tma_load_3d(to + L::kTileCodes, &map_v, &ring_bar[it % kRing], 0, y, z);
    };
    const int turns = max(0, (here - warp * kTile + kTile * kWarps - 1) / (kTile * kWarps));   // tiles of this warp
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kRing; i++) mbar_init(&ring_bar[i], 1);
        s_top[warp].y = 0x7FFFu;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < min(kRing, turns); i++) ask(i);
    }
    __syncwarp();

    // ranges of kChunk entries; 0 behind the end, whatever lies there
    uint2 raw[kChunk / THREADS];
    const KvScale *ranges = static_cast<const KvScale *>(p.c.scales) + base + j0;
    auto load_ranges = [&](int from) {
#pragma unroll
        for (int i = 0; i < kChunk / THREADS; i++) {
            const int j = from + tid + i * THREADS;
            raw[i] = j < here ? *reinterpret_cast<const uint2 *>(ranges + j) : make_uint2(0, 0);
        }
    };
    // Lays them down.  2^te is from then on not below any of their values' steps, huge says
    // whether some value passes 2^87, and spread whether the entries are not alike; none of
    // them falls along a unit.  A value's step carries the 2^(7 - te) of the fp16 weights
    // (spread: none, the rows' scales do), so that the weights themselves, which the sums of
    // fp32 take, need none.
    int te = kLeastTe;
    bool huge = false, spread = false;
    auto put_ranges = [&](int from) {
        uint32_t most = 0, low = 0x7FFF7FFFu;   // of the steps and, in the high half, of the lower ends: a bf16's bits without its sign order like its magnitude
#pragma unroll
        for (int i = 0; i < kChunk / THREADS; i++) {
            most = __vmaxu2(most, raw[i].y & 0x7FFF7FFFu);
            if (from + tid + i * THREADS < here) low = __vminu2(low, raw[i].y & 0x7FFF7FFFu);
        }
        if (__any_sync(0xffffffffu, (most & 0xFFFFu) >= 0x7F80u || most >= 0x7F800000u)) {   // what is not finite does not count
            most = 0;
#pragma unroll
            for (int i = 0; i < kChunk / THREADS; i++) {
                const uint32_t step = raw[i].y & 0x7FFFu, lo = raw[i].y & 0x7FFF0000u;
                most = __vmaxu2(most, (step < 0x7F80u ? step : 0u) | (lo < 0x7F800000u ? lo : 0u));
            }
        }
        uint32_t top = __reduce_max_sync(0xffffffffu, most & 0xFFFFu);
        const bool far = __any_sync(0xffffffffu, most >> 16 >= kHugeLo);
        uint32_t least = __reduce_min_sync(0xffffffffu, max(low & 0xFFFFu, (low >> 16) - min(low >> 16, 4u << 7)));
        if (lane == 0) s_top[warp] = make_uint2(top | (uint32_t)far << 16, min(least, s_top[warp].y));
        __syncthreads();
        for (int w = 0; w < kWarps; w++) {
            top = max(top, s_top[w].x & 0xFFFFu);
            least = min(least, s_top[w].y);
            huge |= s_top[w].x >> 16;
        }
        if (top) te = max(te, (int)(top >> 7) - 126);
        huge |= te > kHugeTe;
        spread |= te > kLeastTe && te + 126 - (int)(least >> 7) > kAlike;
        const float down = huge ? kHuge : 1.0f, up = spread ? down : pow2f(7 - te);
#pragma unroll
        for (int i = 0; i < kChunk / THREADS; i++)
            sc[tid + i * THREADS] = make_float4(__uint_as_float(raw[i].x << 16), __uint_as_float(raw[i].x & 0xFFFF0000u),
                                                __uint_as_float(raw[i].y << 16) * up, __uint_as_float(raw[i].y & 0xFFFF0000u) * down);
        __syncthreads();
    };
    load_ranges(0);

    // the query: D / 8 threads a row, 8 dimensions each, which are one lane's share of a chunk
    constexpr int TR = D / 8;
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += THREADS / TR) {
        const int r = r0 + tid / TR, part = tid % TR, row = rb * R + r;
        if (r < R) {   // whole warps
            const bool there = row < p.rows;
            const T *src = static_cast<const T *>(p.q) + (there ? row_offset(p, p.qs, b, h, row) : 0) + part * 8;
            __align__(16) T v[8];
            if (there && p.vec) {
                *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(src);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = there ? src[i] : from_f32<T>(0.0f);
            }
            float x[8], big = 0.0f, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = to_f32(v[i]);
                big = fmaxf(big, fabsf(x[i]));
                sum += x[i];
            }
#pragma unroll
            for (int o = 1; o < TR; o <<= 1) {
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
            int e = (int)(__float_as_uint(big) >> 23) - 127;
            e = e > 127 ? 0 : min(max(e, -100), 126);
            // a negative scale turns the query round, so that larger is larger in what follows
            const float up = copysignf(pow2f(13 - e), p.scale_log2), u16 = up * 0.0625f;
            s_q[((r >> 3) * CH + (part >> 2)) * 32 + (r & 7) * 4 + (part & 3)] =
                make_uint4(pack_half(x[0] * up, x[4] * up), pack_half(x[1] * u16, x[5] * u16),
                           pack_half(x[2] * up, x[6] * up), pack_half(x[3] * u16, x[7] * u16));
            if (part == 0) {   // q.c is the MMA's times 2^24 2^(e - 13)
                s_qs[r] = make_float2(fabsf(p.scale_log2) * 2048.0f * pow2f(e), copysignf(pow2f(-e), p.scale_log2) * (sum * (1.0f / 2048.0f)));
                s_out[r] = there ? row_offset(p, p.os, b, h, row) : 0;
            }
        }
    }
    // weight times 2^(7 - te) times step is below 2^15 for weights up to 2^8
    put_ranges(0);   // a barrier: the query is there too
    if (spread && lane < R) s_scale[warp][lane] = make_float2(0.0f, __int_as_float(0));
    __syncwarp();

    const int warps = max(1, min(kWarps, (here + kTile - 1) / kTile));   // that have a tile
    constexpr int LD = D + 4;
    float *so = reinterpret_cast<float *>(smem);   // [warp][row][LD], over codes and ranges once all are read
    static_assert(kWarps * R * LD * 4 <= L::kBars, "the warps' sums fit where the codes were");
    // scores of this CTA's rows from entry j0 on, kept for the weights
    float *score = TRACK ? p.score + (((int64_t)b * p.c.n_heads + h) * p.rows + rb * R) * p.max_len + j0 : nullptr;
    const int rows_here = min(R, p.rows - rb * R);
    // kExact: the weights' rounding to fp16, 2^-12 of each, is as large as that of an fp16
    // result, so there what it leaves is a second fp16 weight of its own, to 2^-22
    constexpr bool kExact = DType<T>::kCode == CZG_F16;
    float m[NB][2], l[NB][2], z[NB][2], o[NB][CH][2][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            m[nb][i] = -INFINITY;
            l[nb][i] = z[nb][i] = 0.0f;
        }
#pragma unroll
        for (int ch = 0; ch < CH; ch++)
#pragma unroll
            for (int i = 0; i < 8; i++) o[nb][ch][i >> 2][i & 3] = 0.0f;
    }
    {
        uint4 qf[NB][CH];
        float qs[NB][2], zq[NB][2];   // of rows 2 c4, 2 c4 + 1
        int seen[NB][2], least = 0x7FFFFFFF;   // entries of this unit that the row sees; what all rows see at least
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int ch = 0; ch < CH; ch++) qf[nb][ch] = s_q[(nb * CH + ch) * 32 + lane];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = nb * 8 + 2 * c4 + i;
                qs[nb][i] = s_qs[r].x;
                zq[nb][i] = s_qs[r].y;
                seen[nb][i] = r < rows_here ? here : 0x7FFFFFFF;
                if (p.t > 1 && r < rows_here) seen[nb][i] = n - (p.t - 1 - row_place(p, rb * R + r)) - j0;
                least = min(least, seen[nb][i]);
            }
        }
        least = __reduce_min_sync(0xffffffffu, least);
        // ldmatrix: lane i gives the address of row i % 8 of matrix i / 8; matrices are
        // (entries 0-7, 8-15) x (two chunks)
        const int lm_row = (lane & 7) + (lane & 8), lm_ch = lane >> 4;
        const uint32_t swz = D == 64 ? (uint32_t)(lm_row >> 2 & 1) : (uint32_t)(lm_row >> 1 & 3);

        float mq[NB][2];   // reference times factor
        auto tile_of = [&](int it, auto cut_of) {
            constexpr bool CUT = decltype(cut_of)::value;   // some row does not see some of the tile's entries, or spread
            const int t0 = (it * kWarps + warp) * kTile;   // within the unit
            const float4 *range = sc + t0 % kChunk + g8;
            const uint32_t ka = smem_addr(ring + (it % kRing) * 2 * L::kTileCodes) + (uint32_t)lm_row * (D / 2), va = ka + L::kTileCodes;
            constexpr int KB = kTile / 16;
            float s[NB][KB][4];
            // entries inside, so that neighbouring MMAs add to different sums
#pragma unroll
            for (int cp = 0; cp < CH; cp += 2) {
                uint32_t w[KB][4];
#pragma unroll
                for (int kb = 0; kb < KB; kb++) ldsm4(w[kb], ka + kb * 16 * (D / 2) + (((uint32_t)(cp + lm_ch) ^ swz) << 4));
#pragma unroll
                for (int ci = 0; ci < 2; ci++)
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int kb = 0; kb < KB; kb++) {
                            const uint32_t a = w[kb][2 * ci] >> (8 * half), c = w[kb][2 * ci + 1] >> (8 * half);
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) {
                                const uint4 &f = qf[nb][cp + ci];
                                if (cp + ci + half == 0) mma_f16_first(s[nb][kb], a & 0x000F000Fu, c & 0x000F000Fu, a & 0x00F000F0u, c & 0x00F000F0u, f.x, f.y);
                                else mma_f16(s[nb][kb], a & 0x000F000Fu, c & 0x000F000Fu, a & 0x00F000F0u, c & 0x00F000F0u, half ? f.z : f.x, half ? f.w : f.y);
                            }
                        }
            }
            // scores over the row's factor
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int j = t0 + kb * 16 + hf * 8 + g8;
                    const float2 kr = *reinterpret_cast<const float2 *>(&range[kb * 16 + hf * 8]);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float &x = s[nb][kb][2 * hf + i];
                            x = __fmaf_rn(kr.x, x, kr.y * zq[nb][i]);
                            if (TRACK && nb * 8 + 2 * c4 + i < rows_here && (!CUT || j < here))
                                score[(int64_t)(nb * 8 + 2 * c4 + i) * p.max_len + j] = x;
                        }
                }
            // Weights are taken from a reference that follows the maximum only where a weight
            // would pass 2^8 (each row by itself, so that its bits are its own): after the
            // first tile there is hardly anything to look for, or to take down.
            float mt[NB][2];
            bool over = it == 0;
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mt[nb][i] = -INFINITY;
#pragma unroll
                    for (int kb = 0; kb < KB; kb++) {
                        const int j = t0 + kb * 16 + g8;
                        const float x = CUT && j >= seen[nb][i] ? -INFINITY : s[nb][kb][i];
                        const float y = CUT && j + 8 >= seen[nb][i] ? -INFINITY : s[nb][kb][2 + i];
                        mt[nb][i] = fmaxf(mt[nb][i], fmaxf(x, y));
                    }
                    over |= (mt[nb][i] - m[nb][i]) * qs[nb][i] > 8.0f;
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mt[nb][i] = fmaxf(mt[nb][i], __shfl_xor_sync(0xffffffffu, mt[nb][i], x));
                        const float was = m[nb][i];
                        if (was == -INFINITY || (mt[nb][i] - was) * qs[nb][i] > 8.0f) m[nb][i] = fmaxf(was, mt[nb][i]);
                        const float now = m[nb][i];
                        mq[nb][i] = now == -INFINITY ? 0.0f : now * qs[nb][i];
                        if (it > 0) {
                            const float f = was == now ? 1.0f : was == -INFINITY ? 0.0f : ex2((was - now) * qs[nb][i]);
                            l[nb][i] *= f;
                            z[nb][i] *= f;
                            if (CUT && spread && g8 == 0) s_scale[warp][nb * 8 + 2 * c4 + i].x *= f;
#pragma unroll
                            for (int ch = 0; ch < CH; ch++)
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    o[nb][ch][y][i] *= f;
                                    o[nb][ch][y][2 + i] *= f;
                                }
                        }
                    }
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                uint32_t pf[NB][2], pl[NB][2];
                float w[2][NB][2];
                auto pack = [&](int hf, int nb) {
                    const uint32_t wp = pack_half(w[hf][nb][0], w[hf][nb][1]);
                    if (kExact) {
                        const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&wp));
                        pl[nb][hf] = transpose8(pack_half(w[hf][nb][0] - back.x, w[hf][nb][1] - back.y));
                    }
                    pf[nb][hf] = transpose8(wp);
                };
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int j = t0 + kb * 16 + hf * 8 + g8;
                    const float2 vr = *reinterpret_cast<const float2 *>(&range[kb * 16 + hf * 8].z);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const bool off = CUT && j >= seen[nb][i];   // what is not seen may be anything
                            const float y = off ? 0.0f : ex2(__fmaf_rn(s[nb][kb][2 * hf + i], qs[nb][i], -mq[nb][i]));
                            l[nb][i] += y;
                            z[nb][i] = off ? z[nb][i] : __fmaf_rn(y, vr.y, z[nb][i]);
                            w[hf][nb][i] = off ? 0.0f : y * vr.x;
                        }
                        if (!CUT) pack(hf, nb);
                    }
                }
                if (CUT && spread) {   // keeps the row's largest weight times step between 2^8 and 2^15
                    __syncwarp();
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float2 sc = s_scale[warp][nb * 8 + 2 * c4 + i];
                            float most = fmaxf(fabsf(w[0][nb][i]), fabsf(w[1][nb][i]));
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
                            most = fmaxf(most, sc.x);
                            int k = __float_as_int(sc.y);
                            const int e = (int)(__float_as_uint(most) >> 23) - 127;
                            if (e + k < 8 || e + k >= 15 || abs(k) > 126) {
                                const int was = k;
                                k = min(max(13 - e, -126), 126);
                                const int by = min(max(k - was, -252), 252), half = by / 2;
                                const float f = pow2f(half), f2 = pow2f(by - half);
#pragma unroll
                                for (int ch = 0; ch < CH; ch++)
#pragma unroll
                                    for (int y = 0; y < 2; y++) {
                                        o[nb][ch][y][i] = o[nb][ch][y][i] * f * f2;
                                        o[nb][ch][y][2 + i] = o[nb][ch][y][2 + i] * f * f2;
                                    }
                            }
                            w[0][nb][i] *= pow2f(k);
                            w[1][nb][i] *= pow2f(k);
                            __syncwarp();   // all lanes have read it
                            if (g8 == 0) s_scale[warp][nb * 8 + 2 * c4 + i] = make_float2(most, __int_as_float(k));
                        }
                }
                if (CUT)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) pack(hf, nb);
#pragma unroll
                for (int cp = 0; cp < CH; cp += 2) {
                    uint32_t w[4];
                    ldsm4_trans(w, va + kb * 16 * (D / 2) + (((uint32_t)(cp + lm_ch) ^ swz) << 4));
#pragma unroll
                    for (int ci = 0; ci < 2; ci++) {
                        // the odd rows take whole bytes, 16 times their code and the even row's once:
                        // one operation less than masking the code, and taken off at the end
                        const uint32_t a = w[2 * ci], c = w[2 * ci + 1];
                        const uint32_t a8 = __byte_perm(a, 0u, 0x4341), c8 = __byte_perm(c, 0u, 0x4341);
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            mma_f16(o[nb][cp + ci][0], a & 0x000F000Fu, a & 0x00FF00FFu, c & 0x000F000Fu, c & 0x00FF00FFu, pf[nb][0], pf[nb][1]);
                            mma_f16(o[nb][cp + ci][1], a8 & 0x000F000Fu, a8, c8 & 0x000F000Fu, c8, pf[nb][0], pf[nb][1]);
                            if (kExact) {
                                mma_f16(o[nb][cp + ci][0], a & 0x000F000Fu, a & 0x00FF00FFu, c & 0x000F000Fu, c & 0x00FF00FFu, pl[nb][0], pl[nb][1]);
                                mma_f16(o[nb][cp + ci][1], a8 & 0x000F000Fu, a8, c8 & 0x000F000Fu, c8, pl[nb][0], pl[nb][1]);
                            }
                        }
                    }
                }
            }
        };
        constexpr int kTurns = kChunk / (kTile * kWarps);   // a warp's tiles of a chunk
        int it = 0;
#pragma unroll 1
        for (int j = 0;; j += kChunk) {
#pragma unroll 1
            for (const int end = min(turns, j / kChunk * kTurns + kTurns); it < end; it++) {
                if (!mbar_try(&ring_bar[it % kRing], (it / kRing) & 1) && !mbar_wait(&ring_bar[it % kRing], (it / kRing) & 1, nullptr)) {
                    atomicOr(&g_ops_timeout, 1);
                    mbar_wait(&ring_bar[it % kRing], (it / kRing) & 1, nullptr);   // once more for the copies, before anything ends
                }
                __syncwarp();
                if (spread || (it * kWarps + warp + 1) * kTile > least) tile_of(it, std::true_type{}); else tile_of(it, std::false_type{});
                __syncwarp();   // all lanes have read the tile
                if (lane == 0 && it + kRing < turns) ask(it + kRing);
            }
            if (j + kChunk >= here) break;
            load_ranges(j + kChunk);
            __syncthreads();   // all warps are through with the last chunk's ranges
            const int was = te;
            const bool was_huge = huge, was_spread = spread;
            put_ranges(j + kChunk);
            if (huge && !was_huge) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int i = 0; i < 2; i++) z[nb][i] *= kHuge;
            }
            if (spread) {
                __syncwarp();
                if (lane < R) {   // the sums of codes so far have the unit's scale, or lose that of the values
                    float2 sc = s_scale[warp][lane];
                    if (!was_spread) sc = make_float2(pow2f(min(was + 7, 126)) * (huge ? kHuge : 1.0f), __int_as_float(7 - was + (huge ? 48 : 0)));
                    else if (huge && !was_huge) sc = make_float2(sc.x * kHuge, __int_as_float(__float_as_int(sc.y) + 48));
                    s_scale[warp][lane] = sc;
                }
                __syncwarp();
            } else if (te > was) {    // a larger step: the sums of codes so far by the smaller power of two of the next
                const float f = pow2f(max(was - te, -126)), f2 = pow2f(min(was - te + 126, 0));   // their product is 2^(was - te)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int ch = 0; ch < CH; ch++)
#pragma unroll
                        for (int i = 0; i < 8; i++) o[nb][ch][i >> 2][i & 3] = o[nb][ch][i >> 2][i & 3] * f * f2;
            }
        }
        // sums over the lanes that share a row
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    l[nb][i] += __shfl_xor_sync(0xffffffffu, l[nb][i], x);
                    z[nb][i] += __shfl_xor_sync(0xffffffffu, z[nb][i], x);
                }
                m[nb][i] = m[nb][i] == -INFINITY ? -INFINITY : m[nb][i] * qs[nb][i];
                if (g8 == 0 && warp < warps) {
                    s_m[warp][nb * 8 + 2 * c4 + i] = m[nb][i];
                    s_l[warp][nb * 8 + 2 * c4 + i] = l[nb][i];
                }
            }
    }
    // the warps' rows together, in their order
    __syncthreads();
    if (tid < R) {
        float top_m = s_m[0][tid], sum = 0.0f;
        for (int w = 1; w < warps; w++) top_m = fmaxf(top_m, s_m[w][tid]);
        for (int w = 0; w < warps; w++) sum += s_l[w][tid] * share(s_m[w][tid], top_m);
        s_row[tid] = make_float2(top_m, sum);
    }
    if (warp < warps) {
        float down = pow2f(te - 7), up24 = huge ? 16777216.0f * kHuge : 16777216.0f;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = nb * 8 + 2 * c4 + i;
                float top_m = s_m[0][r];
                for (int w = 1; w < warps; w++) top_m = fmaxf(top_m, s_m[w][r]);
                if (spread) {
                    const int k = __float_as_int(s_scale[warp][r].y);
                    down = pow2f(max(-k, -126)) * pow2f(min(126 - k, 0));
                    up24 = 16777216.0f;
                }
                const float f = share(m[nb][i], top_m), zz = z[nb][i] * f, even = down * f, odd = even * 0.0625f;
#pragma unroll
                for (int ch = 0; ch < CH; ch++)
#pragma unroll
                    for (int y = 0; y < 2; y++)   // dimensions 32 ch + 4 g8 + 2 y and the next
                        *reinterpret_cast<float2 *>(&so[(warp * R + r) * LD + ch * 32 + 4 * g8 + 2 * y]) =
                            make_float2(__fmaf_rn(o[nb][ch][y][i] * up24, even, zz),
                                        __fmaf_rn((o[nb][ch][y][2 + i] - o[nb][ch][y][i]) * up24, odd, zz));
            }
    }
    __syncthreads();
    const bool whole = p.whole;   // nothing to join: this is the result
    const int64_t at = whole ? 0 : (((int64_t)b * p.c.n_heads + h) * p.units + unit) * ((int64_t)p.row_blocks * R) + rb * R;
    for (int i = tid; i < rows_here * (D / 4); i += THREADS) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        const float2 row = s_row[r];
        float4 x = *reinterpret_cast<const float4 *>(&so[r * LD + d]);
        for (int w = 1; w < warps; w++) {
            const float4 v = *reinterpret_cast<const float4 *>(&so[(w * R + r) * LD + d]);
            x.x += v.x;
            x.y += v.y;
            x.z += v.z;
            x.w += v.w;
        }
        if (whole) {
            store4(static_cast<T *>(p.out) + s_out[r] + d, x, row.y == 0.0f ? 0.0f : 1.0f / row.y, huge ? 1.0f / kHuge : 1.0f, p.out_vec);   // a row that sees nothing: 0
        } else {
            *reinterpret_cast<float4 *>(p.part + (at + r) * D + d) = x;
            if (d == 0) p.stat[at + r] = make_float4(row.x, huge ? -row.y : row.y, s_qs[r].x, 0.0f);
        }
    }
    if (TRACK && whole)   // the scores that this CTA wrote
        for (int j = tid; j < here; j += THREADS) {
            float add = 0.0f;
            for (int r = 0; r < rows_here; r++) {
                const float2 row = s_row[r];
                if (j < n - (p.t - 1 - row_place(p, rb * R + r)))
                    add += ex2(__fmaf_rn(score[(int64_t)r * p.max_len + j], s_qs[r].x, -row.x)) * (1.0f / row.y);
            }
            if (add != 0.0f) p.c.weights[base + j0 + j] += add;
        }
}

// Joins the units of rows: the first row_ctas CTAs of x write the rows' results, the others
// the weights of kChunk entries each.  A row's units are taken in RUNS interleaved runs and
// those in order: places that depend on its length alone.  Up to kFew units make one run,
// and a CTA takes RUNS rows of them (so fewer row_ctas do where no sequence may have more).
// Bound by latency, one round of loads each for the statistics and what they scale: 5 us
// for 128 units of 4 rows and 8 heads, 9 us with the weights of 64 sequences of up to 4096.
constexpr int kJoinThreads = 256, kFew = 8;
static_assert(kUnits <= kJoinThreads, "a thread a unit");
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_kv4_join(const __grid_constant__ AttendArgs p, int rows_padded, int row_ctas) {
    constexpr int TR = D / 4, RUNS = kJoinThreads / TR;   // TR threads a run, four dimensions each
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int slot = kv4_slot(p.c, p.slots, b, false);
    const int n = slot < 0 ? 0 : kv4_length(p.c, p.lengths, b, min(p.max_len, p.c.capacity), false);
    const int len = unit_of(n), units = n == 0 ? 0 : (n - 1) / len + 1;
    const int64_t first = ((int64_t)b * p.c.n_heads + h) * p.units * rows_padded;
    pdl_wait();   // slots and lengths are older than the kernel before this one, which waited for them
    if ((int)blockIdx.x < row_ctas) {
        const int d = 4 * (tid % TR), run = tid / TR;
        if (units <= kFew) {
            // each CTA the next RUNS rows
            const int r = blockIdx.x * RUNS + run;
            if (r >= p.rows) return;
            float4 st[kFew];
            float m = -INFINITY, l = 0.0f;
            bool huge = false;   // some partial result is taken kHuge-fold: all are
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int64_t at = first + r;
#pragma unroll
            for (int u = 0; u < kFew; u++) st[u] = u < units ? p.stat[at + (int64_t)u * rows_padded] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < kFew; u++) {
                m = fmaxf(m, st[u].x);
                huge |= signbit(st[u].y);
            }
#pragma unroll
            for (int u0 = 0; u0 < kFew; u0 += 4) {
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (u0 + u < units) v[u] = *reinterpret_cast<const float4 *>(p.part + (at + (int64_t)(u0 + u) * rows_padded) * D + d);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (u0 + u < units) {
                        const float f = share(st[u0 + u].x, m);
                        add_scaled(x, huge && !signbit(st[u0 + u].y) ? f * kHuge : f, v[u]);
                        l = __fmaf_rn(f, fabsf(st[u0 + u].y), l);
                    }
            }
            store4(static_cast<T *>(p.out) + row_offset(p, p.os, b, h, r) + d, x, l == 0.0f ? 0.0f : 1.0f / l, huge ? 1.0f / kHuge : 1.0f, p.out_vec);
            return;
        }
        __shared__ float s_f[kUnits], red[kJoinThreads / 32];
        __shared__ float4 runs[RUNS][TR];
        const int r = blockIdx.x;
        float4 st = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        if (tid < units) st = p.stat[first + (int64_t)tid * rows_padded + r];
        float m = st.x;
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((tid & 31) == 0) red[tid >> 5] = m;
        const bool huge = __syncthreads_or(signbit(st.y));   // as above
        for (int w = 0; w < kJoinThreads / 32; w++) m = fmaxf(m, red[w]);
        const float f = share(st.x, m);
        float l = f * fabsf(st.y);
        if (tid < units) s_f[tid] = huge && !signbit(st.y) ? f * kHuge : f;
        __syncthreads();
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 16
        for (int u = run; u < units; u += RUNS)
            add_scaled(x, s_f[u], *reinterpret_cast<const float4 *>(p.part + (first + (int64_t)u * rows_padded + r) * D + d));
        runs[run][tid % TR] = x;
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = l;
        __syncthreads();
        if (run > 0) return;
        l = 0.0f;
        for (int w = 0; w < kJoinThreads / 32; w++) l += red[w];
        for (int i = 1; i < RUNS; i++) add_scaled(x, 1.0f, runs[i][tid]);
        store4(static_cast<T *>(p.out) + row_offset(p, p.os, b, h, r) + d, x, l == 0.0f ? 0.0f : 1.0f / l, huge ? 1.0f / kHuge : 1.0f, p.out_vec);
        return;
    }
    // weights of kChunk entries, a thread two of them, 8 rows at a time: their scores are
    // under way while a warp a row makes up the row's maximum and sum
    const int j0 = ((int)blockIdx.x - row_ctas) * kChunk;
    if (j0 >= n) return;
    constexpr int RB = kJoinThreads / 32, EACH = kChunk / kJoinThreads;
    __shared__ float4 s_row[RB];
    float *w = p.c.weights + kv4_row(p.c, slot, h, j0);
    float add[EACH] = {}, old[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) old[i] = j0 + i * kJoinThreads + tid < n ? w[i * kJoinThreads + tid] : 0.0f;
    for (int r0 = 0; r0 < p.rows; r0 += RB) {
        const float *s = p.score + (((int64_t)b * p.c.n_heads + h) * p.rows + r0) * p.max_len + j0 + tid;
        float v[RB][EACH];
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int i = 0; i < EACH; i++)
                if (r0 + r < p.rows && j0 + i * kJoinThreads + tid < n) v[r][i] = s[(int64_t)r * p.max_len + i * kJoinThreads];
        const int mine = r0 + (tid >> 5), u0 = tid & 31;
        float4 st = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        if (mine < p.rows) {
            if (u0 < units) st = p.stat[first + (int64_t)u0 * rows_padded + mine];
            float m = st.x;
            for (int u = u0 + 32; u < units; u += 32) m = fmaxf(m, p.stat[first + (int64_t)u * rows_padded + mine].x);
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            float l = fabsf(st.y) * share(st.x, m);
            for (int u = u0 + 32; u < units; u += 32) {
                const float4 more = p.stat[first + (int64_t)u * rows_padded + mine];
                l += fabsf(more.y) * share(more.x, m);
            }
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            st = make_float4(m, l == 0.0f ? 0.0f : 1.0f / l, st.z, 0.0f);
        }
        __syncthreads();   // s_row's readers of the last rows are done
        if (u0 == 0) s_row[tid >> 5] = st;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RB; r++) {
            if (r0 + r >= p.rows) break;
            const int seen = n - (p.t - 1 - row_place(p, r0 + r)) - j0 - tid;
            const float4 row = s_row[r];
#pragma unroll
            for (int i = 0; i < EACH; i++)
                if (i * kJoinThreads < seen) add[i] += ex2(__fmaf_rn(v[r][i], row.z, -row.x)) * row.y;
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; i++)
        if (add[i] != 0.0f) w[i * kJoinThreads + tid] = old[i] + add[i];
}

// Rows of 4-bit codes as a map of boxes of kTile entries of one slot and head.
bool kv4_map(CUtensorMap *map, uint8_t *p, const czg_kv4 &c) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t row = (cuuint64_t)c.head_dim / 2;
    cuuint64_t dims[3] = {row, (cuuint64_t)c.capacity, (cuuint64_t)c.n_slots * c.n_heads};
    cuuint64_t strides[2] = {row, row * c.capacity};
    cuuint32_t box[3] = {(cuuint32_t)row, kTile, 1};
    cuuint32_t one[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              c.head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a call is cut, and where its workspace's parts lie.
struct AttendPlan {
    int rows, nb, row_blocks, units, chunks;
    bool join;
    uint64_t part, stat, score, bytes;
};

AttendPlan attend_plan(const czg_kv4 &c, int64_t b, int t, int hq, int max_len) {
    AttendPlan a{};
    const int n = max_len < c.capacity ? max_len : c.capacity;
    a.rows = t * (hq / c.n_heads);
    a.nb = a.rows <= 8 ? 1 : 2;
    a.row_blocks = (a.rows + 8 * a.nb - 1) / (8 * a.nb);
    a.units = n <= kChunk ? 1 : n > kChunk * kUnits ? kUnits : (n + kChunk - 1) / kChunk;   // of the longest, or of a shorter one
    a.chunks = (n + kChunk - 1) / kChunk;
    a.join = a.units > 1 || (c.weights && a.row_blocks > 1);
    const uint64_t sets = a.join ? (uint64_t)b * c.n_heads * a.units * a.row_blocks * 8 * a.nb : 0;
    a.stat = sets * c.head_dim * 4;
    a.score = a.stat + sets * 16;
    a.bytes = a.score + (c.weights ? (uint64_t)b * c.n_heads * a.rows * (uint64_t)max_len * 4 : 0);
    return a;
}

template <typename T>
int append(const czg_kv4 &c, const void *k, Strides ks, const void *v, Strides vs, const int32_t *slots,
           const int32_t *lengths, int b, int t, cudaStream_t st) {
    const int64_t rows = (int64_t)b * t * c.n_heads;
    if (rows >= 1ll << 30) return ops_fail(CZG_E_LIMIT, "too many rows");
    const int64_t per = 1024 / c.head_dim;   // rows of keys and of values a CTA
    auto vec_of = [](const void *p, const Strides &x) {
        return aligned(p, 4 * sizeof(T)) && x.b % 4 == 0 && x.t % 4 == 0 && x.h % 4 == 0;
    };
    const int vec = vec_of(k, ks) && vec_of(v, vs);
    auto kern = c.head_dim == 64 ? k_kv4_append<T, 64> : k_kv4_append<T, 128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)((2 * rows + per - 1) / per + 1)), 256, 0, st, true, 1, c,
                               static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, vec, slots, lengths, b, t));
}

template <typename T>
int read(const czg_kv4 &c, const int32_t *slots, const int32_t *starts, int b, int count, void *k, void *v, cudaStream_t st) {
    const int64_t rows = (int64_t)count * c.n_heads, all = rows * b;   // of a sequence, of the call
    if (all >= 1ll << 31) return ops_fail(CZG_E_LIMIT, "too many entries");
    const int64_t per = 4096 / c.head_dim;
    auto kern = c.head_dim == 64 ? k_kv4_read<T, 64> : k_kv4_read<T, 128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)((all + per - 1) / per)), 256, 0, st, true, 1, c, slots, starts,
                               (uint32_t)rows, (uint32_t)all, static_cast<T *>(k), static_cast<T *>(v)));
}

template <typename T, int D, int NB, bool TRACK>
int attend_with(const AttendPlan &plan, const AttendArgs &p, int b, cudaStream_t st) {
    alignas(64) CUtensorMap mk, mv;
    if (!kv4_map(&mk, p.c.k, p.c) || !kv4_map(&mv, p.c.v, p.c)) return ops_fail(CZG_E_DEVICE, "no tensor map for the cache");
    constexpr int kWarps = attend_warps(NB);
    const size_t smem = AttendSmem<D, kWarps>::kBytes;
    static std::atomic<int> ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return ops_fail(CZG_E_DEVICE, "no device");
    if (!ready[dev]) {
        if (int e = ops_cuda(cudaFuncSetAttribute(k_kv4_attend<T, D, NB, TRACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)))
            return e;
        ready[dev] = 1;
    }
    const dim3 grid((unsigned)plan.units, (unsigned)(p.c.n_heads * plan.row_blocks), (unsigned)b);
    if (int e = ops_cuda(ops_launch(k_kv4_attend<T, D, NB, TRACK>, grid, kWarps * 32, smem, st, true, 1, mk, mv, p))) return e;
    if (!plan.join) return CZG_OK;
    constexpr int kRuns = kJoinThreads / (D / 4);
    const int row_ctas = plan.units <= kFew ? (plan.rows + kRuns - 1) / kRuns : plan.rows;
    const dim3 join((unsigned)(row_ctas + (TRACK ? plan.chunks : 0)), (unsigned)p.c.n_heads, (unsigned)b);
    return ops_cuda(ops_launch(k_kv4_join<T, D>, join, kJoinThreads, 0, st, true, 1, p, plan.row_blocks * 8 * NB, row_ctas));
}

template <typename T>
int attend(const AttendPlan &plan, const AttendArgs &p, int b, cudaStream_t st) {
    const bool track = p.c.weights != nullptr;
    if (p.c.head_dim == 64) {
        if (plan.nb == 1) return track ? attend_with<T, 64, 1, true>(plan, p, b, st) : attend_with<T, 64, 1, false>(plan, p, b, st);
        return track ? attend_with<T, 64, 2, true>(plan, p, b, st) : attend_with<T, 64, 2, false>(plan, p, b, st);
    }
    if (plan.nb == 1) return track ? attend_with<T, 128, 1, true>(plan, p, b, st) : attend_with<T, 128, 1, false>(plan, p, b, st);
    return track ? attend_with<T, 128, 2, true>(plan, p, b, st) : attend_with<T, 128, 2, false>(plan, p, b, st);
}

}  // namespace

int kv4_timeouts(int *bits) { return take_timeouts(bits); }

const char *check_kv4(const czg_kv4 *c) {
    if (!c || !c->k || !c->v || !c->scales || !c->status) return "null pointer in the cache";
    if (c->n_slots < 1 || c->n_heads < 1 || c->capacity < 1) return "a cache has at least one slot, head and entry";
    if ((int64_t)c->n_slots * c->n_heads > 0x7FFFFFFF) return "slots times heads must be below 2^31";
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 8) || !aligned(c->weights, 4) || !aligned(c->status, 4))
        return "the cache's buffers are not aligned";
    return nullptr;
}

}  // namespace czg

using namespace czg;

namespace {

constexpr int kMaxSequences = 65535;   // a grid dimension

int check_call(const czg_kv4 *c, const int32_t *slots, const int32_t *counts, int b) {
    if (const char *why = check_kv4(c)) return ops_fail(CZG_E_ARG, why);
    if (c->head_dim != 64 && c->head_dim != 128) return ops_fail(CZG_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (b > kMaxSequences) return ops_fail(CZG_E_LIMIT, "more than 65,535 sequences in a call");
    if (!slots || !counts) return ops_fail(CZG_E_ARG, "null pointer");
    return CZG_OK;
}

}  // namespace

extern "C" int czg_kv4_append(const czg_kv4 *cache, const void *k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void *v,
                              int64_t v_sb, int64_t v_st, int64_t v_sh, int dtype, const int32_t *slots,
                              const int32_t *lengths, int32_t b, int32_t t, void *stream) {
    if (b < 0 || t < 0) return ops_fail(CZG_E_ARG, "b and t must not be negative");
    if (int st = check_call(cache, slots, lengths, b)) return st;
    if (b == 0 || t == 0) return CZG_OK;
    if (!k || !v) return ops_fail(CZG_E_ARG, "null pointer");
    if (!dtype_ok(dtype)) return ops_fail(CZG_E_ARG, "unknown dtype");
    if (!aligned(k, (uintptr_t)elem_bytes(dtype)) || !aligned(v, (uintptr_t)elem_bytes(dtype)))
        return ops_fail(CZG_E_ARG, "k and v must be aligned to their type");
    const Strides ks{k_sb, k_st, k_sh}, vs{v_sb, v_st, v_sh};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CZG_F32) return append<float>(*cache, k, ks, v, vs, slots, lengths, b, t, st);
    if (dtype == CZG_BF16) return append<__nv_bfloat16>(*cache, k, ks, v, vs, slots, lengths, b, t, st);
    return append<__half>(*cache, k, ks, v, vs, slots, lengths, b, t, st);
}

extern "C" int czg_kv4_read(const czg_kv4 *cache, const int32_t *slots, const int32_t *starts, int32_t b, int32_t count,
                            void *k_out, void *v_out, int dtype, void *stream) {
    if (b < 0 || count < 0) return ops_fail(CZG_E_ARG, "b and count must not be negative");
    if (int st = check_call(cache, slots, starts, b)) return st;
    if (!dtype_ok(dtype)) return ops_fail(CZG_E_ARG, "unknown dtype");
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return ops_fail(CZG_E_ARG, "outputs must begin on 16-byte boundaries");
    if (b == 0 || count == 0 || (!k_out && !v_out)) return CZG_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CZG_F32) return read<float>(*cache, slots, starts, b, count, k_out, v_out, st);
    if (dtype == CZG_BF16) return read<__nv_bfloat16>(*cache, slots, starts, b, count, k_out, v_out, st);
    return read<__half>(*cache, slots, starts, b, count, k_out, v_out, st);
}

extern "C" uint64_t czg_kv4_attend_workspace(const czg_kv4 *cache, int32_t b, int32_t t, int32_t hq, int32_t max_len) {
    if (!cache || cache->n_heads < 1 || cache->capacity < 1 || b < 1 || t < 1 || hq < cache->n_heads || max_len < 0 ||
        (int64_t)t * hq > 0x7FFFFFFF)
        return 0;
    return attend_plan(*cache, b, t, hq, max_len).bytes;
}

extern "C" int czg_kv4_attend(const czg_kv4 *cache, const void *q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype,
                              const int32_t *slots, const int32_t *lengths, int32_t b, int32_t t, int32_t hq,
                              int32_t max_len, float scale, void *out, int64_t o_sb, int64_t o_st, int64_t o_sh, void *ws,
                              uint64_t ws_bytes, void *stream) {
    if (b < 0 || t < 0 || max_len < 0) return ops_fail(CZG_E_ARG, "b, t and max_len must not be negative");
    if (int st = check_call(cache, slots, lengths, b)) return st;
    if (hq < 1 || hq % cache->n_heads != 0) return ops_fail(CZG_E_ARG, "hq must be a multiple of the cache's heads");
    if (dtype != CZG_BF16 && dtype != CZG_F16) return ops_fail(CZG_E_UNSUPPORTED, "q must be bf16 or fp16");
    if (b == 0 || t == 0) return CZG_OK;
    if (!q || !out) return ops_fail(CZG_E_ARG, "null pointer");
    if (!aligned(q, 2) || !aligned(out, 2)) return ops_fail(CZG_E_ARG, "q and out must be aligned to their type");
    if ((int64_t)t * hq > 0x7FFFFFFF || (int64_t)t * hq / cache->n_heads * (hq / cache->n_heads) >= 1ll << 32)
        return ops_fail(CZG_E_LIMIT, "too many rows");
    const Strides qs{q_sb, q_st, q_sh}, os{o_sb, o_st, o_sh};
    const int64_t d = cache->head_dim;
    if ((b > 1 && o_sb == 0) || (t > 1 && o_st == 0) || (hq > 1 && o_sh == 0)) return ops_fail(CZG_E_ARG, "rows of out overlap");
    // a row's output may take its query's place (both are one CTA's), no other's
    if (!(q == out && q_sb == o_sb && q_st == o_st && q_sh == o_sh)) {
        auto last = [&](const void *p, const Strides &s) {
            return reinterpret_cast<intptr_t>(p) + 2 * ((b - 1) * s.b + (t - 1) * s.t + (hq - 1) * s.h + d);
        };
        if (reinterpret_cast<intptr_t>(out) < last(q, qs) && reinterpret_cast<intptr_t>(q) < last(out, os)) {
            // but for heads side by side in rows of one stride
            const int64_t width = (hq - 1) * o_sh + d, off = (static_cast<const char *>(q) - static_cast<char *>(out)) / 2;
            const bool alike = q_sb == o_sb && q_st == o_st && q_sh == o_sh && o_sh > 0 && o_st > 0 && o_sb % o_st == 0;
            const int64_t from = alike ? (off % o_st + o_st) % o_st : 0;
            if (!alike || from < width || from + width > o_st) return ops_fail(CZG_E_ARG, "out lies over q");
        }
    }
    const AttendPlan plan = attend_plan(*cache, b, t, hq, max_len);
    if (ws_bytes < plan.bytes || !aligned(ws, 16) || (plan.bytes && !ws))
        return ops_fail(CZG_E_ARG, "the workspace is too small or not 16-byte aligned");
    if ((int64_t)cache->n_heads * plan.row_blocks > kMaxSequences || cache->n_heads > kMaxSequences)
        return ops_fail(CZG_E_LIMIT, "more than 65,535 blocks of rows");
    const int es = 2;
    AttendArgs p{};
    p.c = *cache;
    p.q = q;
    p.qs = qs;
    p.slots = slots;
    p.lengths = lengths;
    p.t = t;
    p.g = hq / cache->n_heads;
    p.rows = plan.rows;
    p.row_blocks = plan.row_blocks;
    p.max_len = max_len;
    p.units = plan.units;
    p.vec = aligned(q, 16) && (q_sb * es) % 16 == 0 && (q_st * es) % 16 == 0 && (q_sh * es) % 16 == 0;
    p.out_vec = aligned(out, 8) && o_sb % 4 == 0 && o_st % 4 == 0 && o_sh % 4 == 0;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    p.out = out;
    p.os = os;
    p.whole = !plan.join;
    p.g_inv = ((1ull << 32) + p.g - 1) / p.g;
    uint8_t *w = static_cast<uint8_t *>(ws);
    p.part = reinterpret_cast<float *>(w);
    p.stat = reinterpret_cast<float4 *>(w + plan.stat);
    p.score = reinterpret_cast<float *>(w + plan.score);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == CZG_BF16 ? attend<__nv_bfloat16>(plan, p, b, st) : attend<__half>(plan, p, b, st);
}
