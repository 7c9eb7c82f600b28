// ops_linear.cu -- int8 product with a scale for each token and each channel
// (include/czg_ops.h): the row quantiser and the product.
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "ops_common.cuh"
#include "tc_common.cuh"

namespace czg {

static thread_local char g_ops_error[256];   // no allocation: nothing can throw across the C boundary

int ops_fail(int status, const char *why) {
    std::strncpy(g_ops_error, why, sizeof(g_ops_error) - 1);
    return status;
}
int ops_cuda(cudaError_t e) {
    if (e == cudaSuccess) return CZG_OK;
    (void)cudaGetLastError();   // a refused launch leaves no error behind for the next caller
    return ops_fail(CZG_E_DEVICE, cudaGetErrorString(e));
}

namespace {

// code = rne(127 x / a).  r = x (127 / a) in fp32 is off by 2^-22 of itself at most: where
// r (1 - 2^-20) and r (1 + 2^-20) round to the same integer, that is the code.  Rounding is
// the addition of M1 = 1.5 * 2^23 (common.cuh), whose sum's low byte is the code.  Where one
// of 8 values is nearer to a half than that, all 8 are decided exactly: with
// k = rne(r - 1/2), which is the integer below the half in question, the code is k + 1, k, or
// the even one of the two as 127 x is above, below or at (k + 1/2) a.  For 16-bit x both
// products are exact (7 + 11 and 8 + 11 bits), and a fused multiply-add gives their
// difference's sign; for fp32 x they are not, and the rounded quotient of the rounded
// product decides.
__device__ __forceinline__ uint2 pack8(const uint32_t (&n)[8]) {
    return make_uint2(__byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410));
}
// Out of line: one copy of it leaves the unrolled kernels in the instruction cache.
template <bool EXACT>
__device__ __noinline__ uint2 codes8_at_halves(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7, float a) {
    const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
    // a power of two keeps a, 127 x and 127 / a inside fp32
    const float f = a > 1.2676506e30f ? 9.5367431640625e-7f : a < 8.6736174e-19f ? 1.2089258196146292e24f : 1.0f;
    const float af = a * f, inv = __fdiv_rn(127.0f, af);
    uint32_t n[8];
#pragma unroll
    for (int c = 0; c < 8; c++) {
        const float y = x[c] * f;
        if (EXACT) {
            const float k = __fsub_rn(__fadd_rn(__fmaf_rn(y, inv, -0.5f), kM1), kM1);
            const float d = __fmaf_rn(y, 127.0f, -__fmul_rn(k + 0.5f, af));
            const uint32_t b = __float_as_uint(__fadd_rn(k, kM1));
            n[c] = b + (d > 0.0f || (d == 0.0f && (b & 1u)));
        } else {
            n[c] = __float_as_uint(__fadd_rn(__fdiv_rn(y * 127.0f, af), kM1));
        }
    }
    return pack8(n);
}

// 8 values of a row as they lie in memory.  Their magnitudes' bits order like the
// magnitudes, infinity and NaN above all others.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
    uint32_t w[8];
    __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
    __device__ static __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
    static constexpr uint32_t kInf = 0x7F800000u;
    __device__ __forceinline__ void put(int i, float x) { w[i] = __float_as_uint(x); }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(w[i]); }
};
template <typename T> struct Raw8 {   // 16 bits: two values a word, the maximum of both halves at once
    uint32_t w[4];
    __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 4; i++) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return m;
    }
    static constexpr uint32_t kInf = DType<T>::kCode == CZG_BF16 ? 0x7F80u : 0x7C00u;
    __device__ static __forceinline__ T half_of(uint32_t h) {
        const uint16_t u = (uint16_t)h;
        return *reinterpret_cast<const T *>(&u);
    }
    __device__ static __forceinline__ float value(uint32_t m) { return to_f32(half_of(m)); }
    __device__ __forceinline__ void put(int i, T x) {
        const uint32_t u = *reinterpret_cast<const uint16_t *>(&x);
        if (i & 1) w[i / 2] |= u << 16; else w[i / 2] = u;
    }
    __device__ __forceinline__ float get(int i) const { return to_f32(half_of(w[i / 2] >> (16 * (i & 1)))); }
};

// Values i .. i + 7 of a row, 0 behind its end.
template <typename T>
__device__ __forceinline__ void load8(const T *row, int64_t i, int64_t k, bool vec, Raw8<T> &v) {
    if (vec && i + 8 <= k) {
#pragma unroll
        for (int c = 0; c < (int)sizeof(T) / 2; c++) {
            const uint4 t = reinterpret_cast<const uint4 *>(row + i)[c];
            v.w[4 * c] = t.x; v.w[4 * c + 1] = t.y; v.w[4 * c + 2] = t.z; v.w[4 * c + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 8; c++) v.put(c, i + c < k ? row[i + c] : from_f32<T>(0.0f));
    }
}

// What a row's maximum (its magnitude's bits) makes of its values.
template <typename T>
struct RowScale {
    float a, low, high;   // 127 / a less and more 2^-20 of itself
    uint32_t none;          // not 0: 127 / a would overflow, and nothing is decided by it
    bool fine;
    __device__ __forceinline__ explicit RowScale(uint32_t m) {
        fine = m < Raw8<T>::kInf;   // NaN and infinities both end as a row of NaN
        a = Raw8<T>::value(m);
        none = a < 1.5e-36f;
        const float inv = __fdiv_rn(127.0f, none ? 1.0f : a);
        low = inv * (1.0f - 9.5367431640625e-7f);
        high = inv * (1.0f + 9.5367431640625e-7f);
    }
    __device__ __forceinline__ float scale() const { return fine ? __fdiv_rn(a, 127.0f) : NAN; }
    __device__ __forceinline__ uint2 codes(const Raw8<T> &w) const {
        if (!(fine && a > 0.0f)) return make_uint2(0, 0);
        uint32_t n[8], differ = none;
#pragma unroll
        for (int c = 0; c < 8; c++) {
            n[c] = __float_as_uint(__fmaf_rn(w.get(c), low, kM1));
            differ |= n[c] ^ __float_as_uint(__fmaf_rn(w.get(c), high, kM1));
        }
        if (differ)
            return codes8_at_halves<sizeof(T) == 2>(w.get(0), w.get(1), w.get(2), w.get(3), w.get(4), w.get(5), w.get(6), w.get(7), a);
        return pack8(n);
    }
};

// One CTA a row (48 x 4096: 2.8 us): its maximum, then its codes, 8 values a thread and turn; rows of up to
// kHeld turns stay in registers between the two, longer ones are read again.
constexpr int kQuantThreads = 256, kHeld = 4;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) k_quantize_rows(const T *x, int64_t ldx, int64_t k, int vec,
                                                                 int8_t *__restrict__ codes, int64_t ldc,
                                                                 float *__restrict__ scales) {
    pdl_wait();
    pdl_trigger();   // the product may set itself up meanwhile
    const T *row = x + (int64_t)blockIdx.x * ldx;
    int8_t *out = codes + (int64_t)blockIdx.x * ldc;
    __shared__ uint32_t part[kQuantThreads / 32];
    const int64_t turn = (int64_t)blockDim.x * 8, i0 = threadIdx.x * 8;
    const bool held = k <= turn * kHeld;
    Raw8<T> v[kHeld];
    uint32_t m = 0;
    if (held) {
#pragma unroll
        for (int t = 0; t < kHeld; t++)
            if (i0 + t * turn < k) load8(row, i0 + t * turn, k, vec, v[t]);
#pragma unroll
        for (int t = 0; t < kHeld; t++)
            if (i0 + t * turn < k) m = v[t].most(m);
    } else {
        for (int64_t i = i0; i < k; i += turn) {
            load8(row, i, k, vec, v[0]);
            m = v[0].most(m);
        }
    }
    if (sizeof(T) == 2) m = max(m & 0xFFFFu, m >> 16);
    m = __reduce_max_sync(0xffffffffu, m);
    if (blockDim.x > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        m = part[(threadIdx.x & 31) < blockDim.x / 32 ? threadIdx.x & 31 : 0];
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const RowScale<T> rs(m);
    if (threadIdx.x == 0) scales[blockIdx.x] = rs.scale();
    auto put = [&](int64_t i, const Raw8<T> &w) { *reinterpret_cast<uint2 *>(out + i) = rs.codes(w); };
    if (held) {
#pragma unroll
        for (int t = 0; t < kHeld; t++)
            if (i0 + t * turn < k) put(i0 + t * turn, v[t]);
    } else {
        for (int64_t i = i0; i < k; i += turn) {
            load8(row, i, k, vec, v[0]);
            put(i, v[0]);
        }
    }
    // rows of codes end on 16 bytes: the second half of the last 16 may still be to fill
    const int64_t end = (k + 7) & ~(int64_t)7;
    if (threadIdx.x == 0 && (end & 15)) *reinterpret_cast<uint2 *>(out + end) = make_uint2(0, 0);
}

// Many rows of up to 256 V values: a warp a row, all of it in registers, no barrier; the
// CTA's four rows and its neighbours' cover one another's latency.
template <typename T, int V>
__global__ void __launch_bounds__(128) k_quantize_rows_warp(const T *x, int64_t ldx, int m, int k, int vec,
                                                            int8_t *__restrict__ codes, int64_t ldc, float *__restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= m) return;
    const T *row = x + r * ldx;
    int8_t *out = codes + r * ldc;
    Raw8<T> v[V];
    uint32_t most = 0;
#pragma unroll
    for (int t = 0; t < V; t++)
        if ((t * 32 + lane) * 8 < k) load8(row, (t * 32 + lane) * 8, k, vec, v[t]);
#pragma unroll
    for (int t = 0; t < V; t++)
        if ((t * 32 + lane) * 8 < k) most = v[t].most(most);
    if (sizeof(T) == 2) most = max(most & 0xFFFFu, most >> 16);
    const RowScale<T> rs(__reduce_max_sync(0xffffffffu, most));
#pragma unroll
    for (int t = 0; t < V; t++)
        if ((t * 32 + lane) * 8 < k) *reinterpret_cast<uint2 *>(out + (t * 32 + lane) * 8) = rs.codes(v[t]);
    if (lane == 0) {
        scales[r] = rs.scale();
        const int end = (k + 7) & ~7;   // as above
        if (end & 15) *reinterpret_cast<uint2 *>(out + end) = make_uint2(0, 0);
    }
}

// ---- the product -------------------------------------------------------------------
//
// out^T tile = W tile (128 channels, the M of tcgen05.mma kind::i8) times NT tokens (its N):
// D[channel][token] in TMEM, so a lane of the epilogue holds one channel, its scale and
// bias stay in registers, and a warp's store of one token is 32 adjacent channels whatever
// the row stride of out.
//   warp 0      one lane loads, by TMA, 128 bytes of k of 128 weight rows and NT token rows
//               a stage (128-byte swizzle; rows and bytes outside are zeros, which add
//               nothing to the sums).  Weights do not depend on the kernel before this
//               one (the quantiser), so the first stages' weight boxes are asked for
//               before griddepcontrol.wait and only the tokens' after it.
//   warp 1      one lane issues 4 MMAs (k = 32 each) a stage
//   the others  epilogue, EW / 4 warps a quadrant of TMEM lanes
// S = 1: the CTA walks tiles (gridDim.x apart) with two accumulators, so the epilogue of
// one overlaps the MMAs of the next.  S > 1 (few tokens): a cluster of S CTAs shares one
// tile, each a stretch of k; each lays its int32 sums down in its shared memory, and CTA r
// adds up all CTAs' sums of the tokens r NT / S .. (16 bytes a lane through distributed
// shared memory; 4-byte stores to the other CTAs instead took 4 us more at NT = 64):
// integers, so the split does not show in the result.
// Measured: 48 x 4096 x 4096 (16.8 MB of weights): 9.8 us, and 11 with the quantiser; 4.5 us of
// any call are the setup, the first loads and the epilogue.  1333 x 1000 x 1100: 10.6 us.
constexpr int LT = 128;   // channels of a tile

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int4 load_remote(uint32_t addr, uint32_t rank) {
    uint32_t a;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// Barrier of the N threads of the epilogue, and whether any of them says so.
template <int N>
__device__ __forceinline__ bool epilogue_any(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)x), "n"(N) : "memory");
    return r != 0;
}

struct LinearArgs {
    const float *xs, *ws, *bias;
    void *out;
    int64_t ldo;
    int m, n, steps, tiles_n, tiles, stages, split, vec_out;
    const void *x;   // of the kernel that quantises: [m][k], ldx elements apart, vec: rows of 16-byte pieces
    int64_t ldx;
    int k, vec;
};

constexpr int kRingBytes = 220 * 1024;   // of shared memory, for the ring and the sums

template <int NT>
struct LinearCfg {
    static constexpr int kStage = LT * TC_BK + NT * TC_BK;
    static constexpr int kWarps = NT >= 128 ? 10 : 6;
    static size_t smem(int stages, int split) {
        return 1024 + (size_t)stages * kStage + (split > 1 ? LT * NT * 4 : 0) + (2 * stages + 5) * 8 + 16 + NT * 4 * 2;
    }
};

template <typename T>
__device__ __forceinline__ T finish(int acc, float xs, float ws, float bias, bool has_bias) {
    float y = __fmul_rn(__fmul_rn((float)acc, xs), ws);
    if (has_bias) y = __fadd_rn(y, bias);
    return from_f32<T>(y);
}

// TX: void, or the type of x rows that the kernel quantises itself.  Then every CTA reads
// all of x for the rows' maxima and writes the codes of its stretch of k where TMA would
// have put them; a cluster has one tile and the ring holds all of it.  For a few short
// rows, where a launch costs more than reading x once in every CTA.
template <int NT, typename T, typename TX>
__global__ void __launch_bounds__(LinearCfg<NT>::kWarps * 32, 1)
k_linear_tc(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, LinearArgs p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int STAGE = LinearCfg<NT>::kStage, W_BYTES = LT * TC_BK, EW = LinearCfg<NT>::kWarps - 2;
    constexpr int COLS = 2 * NT < 32 ? 32 : 2 * NT;
    constexpr bool kQuantises = !std::is_void<TX>::value;
    const int STAGES = p.stages, S = p.split;
    uint8_t *tail = smem + STAGES * STAGE;
    int *sums = reinterpret_cast<int *>(tail);   // S > 1: [token][channel]
    if (S > 1) tail += LT * NT * 4;
    uint64_t *full = reinterpret_cast<uint64_t *>(tail);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + 2;
    uint64_t *drain = tempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    float *s_xs = reinterpret_cast<float *>(tmem_slot + 4);   // 2 x NT
    __shared__ volatile int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = S > 1 ? (int)cluster_rank() : 0;
    const int k0 = (int)((int64_t)p.steps * rank / S), k1 = (int)((int64_t)p.steps * (rank + 1) / S);
    const int tile0 = S > 1 ? blockIdx.x / S : blockIdx.x, dt = S > 1 ? gridDim.x / S : gridDim.x;
    const int early = min(STAGES, k1 - k0);   // stages of the first tile that need no wait
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], EW);
        }
        mbar_init(drain, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // the first loads are on their way before the others are through the setup
        const int n0 = (tile0 % p.tiles_n) * LT, m0 = (tile0 / p.tiles_n) * NT;
        for (int i = 0; i < early; i++) {
            mbar_expect_tx(&full[i], kQuantises ? W_BYTES : STAGE);
            tma_load_2d(smem + i * STAGE, &map_w, &full[i], (k0 + i) * TC_BK, n0);
        }
        pdl_wait();
        for (int i = 0; i < early && !kQuantises; i++) tma_load_2d(smem + i * STAGE + W_BYTES, &map_x, &full[i], (k0 + i) * TC_BK, m0);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if constexpr (kQuantises) {
        constexpr int THREADS = LinearCfg<NT>::kWarps * 32;
        __shared__ uint32_t s_most[NT];
        if (threadIdx.x < NT) s_most[threadIdx.x] = 0;
        __syncthreads();
        const TX *x = static_cast<const TX *>(p.x);
#pragma unroll 4
        for (int r = 0; r < p.m; r++) {
            uint32_t most = 0;
#pragma unroll 4
            for (int i = threadIdx.x * 8; i < p.k; i += THREADS * 8) {
                Raw8<TX> v;
                load8(x + r * p.ldx, i, p.k, p.vec, v);
                most = v.most(most);
            }
            if (sizeof(TX) == 2) most = max(most & 0xFFFFu, most >> 16);
            most = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) atomicMax(&s_most[r], most);   // a maximum: in any order
        }
        __syncthreads();
        const int pieces = (k1 - k0) * (TC_BK / 8);   // of 8 values, of a row
        for (int t = threadIdx.x; t < p.m * pieces; t += THREADS) {
            const int r = t / pieces, at = t - r * pieces, step = at / (TC_BK / 8), c = at % (TC_BK / 8) / 2;
            Raw8<TX> v;
            load8(x + r * p.ldx, (k0 * (TC_BK / 8) + at) * 8, p.k, p.vec, v);
            // row r of a box, its 16-byte piece c: the 128-byte swizzle
            *reinterpret_cast<uint2 *>(smem + step * STAGE + W_BYTES + r * TC_BK + ((c ^ (r & 7)) << 4) + 8 * (at & 1)) =
                RowScale<TX>(s_most[r]).codes(v);
        }
        if (threadIdx.x < NT) s_xs[threadIdx.x] = (int)threadIdx.x < p.m ? RowScale<TX>(s_most[threadIdx.x]).scale() : 0.0f;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMAs read what the threads wrote
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int tile = tile0; tile < p.tiles && ok; tile += dt) {
                const int n0 = (tile % p.tiles_n) * LT, m0 = (tile / p.tiles_n) * NT;
                for (int kb = k0; kb < k1; kb++, it++) {
                    if (it < early) continue;   // under way already
                    const int s = it % STAGES;
                    uint8_t *sw = smem + s * STAGE;
                    if (it >= STAGES && !mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&full[s], STAGE);
                    tma_load_2d(sw, &map_w, &full[s], kb * TC_BK, n0);
                    tma_load_2d(sw + W_BYTES, &map_x, &full[s], kb * TC_BK, m0);
                }
            }
            if (!ok) {
                atomicOr(&g_ops_timeout, 1);
                abort_flag = 1;
                for (int k = max(0, it - STAGES); k < it; k++) mbar_wait(&full[k % STAGES], (k / STAGES) & 1, nullptr);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_i8(LT, NT);
            int it = 0, tc = 0;
            bool ok = true;
            for (int tile = tile0; tile < p.tiles && ok; tile += dt, tc++) {
                const int b = tc & 1;
                if (tc >= 2 && !mbar_wait(&tempty[b], ((tc >> 1) - 1) & 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = k0; kb < k1; kb++, it++) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&full[s], (it / STAGES) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t wd = smem_desc_sw128(smem_addr(smem + s * STAGE));
                    const uint64_t xd = smem_desc_sw128(smem_addr(smem + s * STAGE + W_BYTES));
#pragma unroll
                    for (int k = 0; k < TC_BK / 32; k++)
                        mma_i8(tmem + (uint32_t)(b * NT), wd + 2 * k, xd + 2 * k, idesc, kb > k0 || k > 0);
                    mma_commit(&empty[s]);
                }
                if (ok) mma_commit(&tfull[b]);
            }
            if (!ok) {
                atomicOr(&g_ops_timeout, 1);
                abort_flag = 1;
            }
            mma_commit(drain);
            mbar_wait(drain, 0, nullptr);
        }
    } else {
        const int q = warp & 3;             // TMEM lanes 32q .. 32q + 31
        const int part = (warp - 2) >> 2;   // of EW / 4 parts of the tokens
        constexpr int PC = NT / (EW / 4);   // tokens of a part
        pdl_wait();
        T *out = static_cast<T *>(p.out);
        int tc = 0;
        for (int tile = tile0; tile < p.tiles; tile += dt, tc++) {
            const int b = tc & 1;
            const int n0 = (tile % p.tiles_n) * LT, m0 = (tile / p.tiles_n) * NT;
            const int ch = n0 + 32 * q + lane;
            const bool there = ch < p.n;
            const float ws = there ? p.ws[ch] : 0.0f, bias = there && p.bias ? p.bias[ch] : 0.0f;
            float *xs = s_xs + b * NT;      // the accumulator's half: its readers are done when tempty[b] fired
            if (S == 1 && !kQuantises)
                for (int i = threadIdx.x - 64; i < NT; i += EW * 32) xs[i] = m0 + i < p.m ? p.xs[m0 + i] : 0.0f;
            const bool got = mbar_wait(&tfull[b], (tc >> 1) & 1, &abort_flag);
            if (epilogue_any<EW * 32>(!got)) {   // one answer for all of them: no warp waits for one that left
                if (!got) {
                    atomicOr(&g_ops_timeout, 1);
                    abort_flag = 1;
                }
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tbase = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(b * NT + part * PC);
            constexpr int CW = PC < 32 ? 16 : 32;
#pragma unroll 1
            for (int c0 = 0; c0 < PC; c0 += CW) {
                uint32_t v[CW];
                if constexpr (CW == 32) tmem_ld32(tbase + c0, v); else tmem_ld16(tbase + c0, v);
                if (c0 + CW == PC) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tempty[b]);
                }
                const int j0 = part * PC + c0;
                if (S > 1) {
#pragma unroll
                    for (int j = 0; j < CW; j++) sums[(j0 + j) * LT + 32 * q + lane] = (int)v[j];
                } else if (there) {
                    T *o = out + (int64_t)(m0 + j0) * p.ldo + ch;
                    const int most = p.m - m0 - j0;
#pragma unroll
                    for (int j = 0; j < CW; j++)
                        if (j < most) o[j * p.ldo] = finish<T>((int)v[j], xs[j0 + j], ws, bias, p.bias != nullptr);
                }
            }
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();   // every CTA of the cluster comes here, whatever it met, and has laid its sums down
        if (warp >= 2) {
            const int per = NT / S, n0 = (tile0 % p.tiles_n) * LT + 4 * lane, m0 = (tile0 / p.tiles_n) * NT + rank * per;
            const bool vec = p.vec_out && n0 + 4 <= p.n;
            float ws[4], bias[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ws[i] = n0 + i < p.n ? p.ws[n0 + i] : 0.0f;
                bias[i] = n0 + i < p.n && p.bias ? p.bias[n0 + i] : 0.0f;
            }
#pragma unroll 4
            for (int j = warp - 2; j < per; j += EW) {
                if (m0 + j >= p.m) break;
                int acc[4] = {0, 0, 0, 0};
                const uint32_t at = smem_addr(sums + (rank * per + j) * LT + 4 * lane);
#pragma unroll
                for (int r = 0; r < 8; r++)
                    if (r < S) {
                        const int4 v = load_remote(at, r);
                        acc[0] += v.x;
                        acc[1] += v.y;
                        acc[2] += v.z;
                        acc[3] += v.w;
                    }
                const float xs = kQuantises ? s_xs[rank * per + j] : p.xs[m0 + j];
                __align__(16) T y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = finish<T>(acc[i], xs, ws[i], bias[i], p.bias != nullptr);
                T *o = static_cast<T *>(p.out) + (int64_t)(m0 + j) * p.ldo + n0;
                if (vec) {
                    if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(y);
                    else *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(y);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (n0 + i < p.n) o[i] = y[i];
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();   // no CTA ends while another reads its sums
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

// ---- the product, two CTAs a tile --------------------------------------------------
//
// For large m the loads of 128 x 256 tiles are what one CTA waits for (8192 x 8192 x 4096:
// 145 of 211 us with the MMAs left out).  A pair of CTAs (tcgen05 cta_group::2) shares
// 256 channels x 256 tokens: each loads its 128 weight rows and half of the tokens, and
// the MMAs of the first CTA read both, so a byte loaded serves a third more products:
// 191 us, 2.88 POP/s, 87% of twice the measured bf16 rate, the tensor pipe 74% active.
// Each CTA's sums of its channels land in its own TMEM; the epilogue is as above.
//   full[s]   of the first CTA: both CTAs' loads of the stage (64 KB)
//   empty[s]  of each CTA: the MMAs have read it (committed to both)
//   tfull[b]  of each CTA; tempty[b] of the first: both CTAs' epilogues have read it
// A CTA whose wait runs out stops; the other's waits run out after it, and both come to
// the cluster barrier at the end, so neither leaves while the other may signal it.
constexpr int kPairTokens = 256, kPairStages = 6, kPairWarps = 10;
constexpr int kPairStage = LT * TC_BK + kPairTokens / 2 * TC_BK;   // a CTA's bytes
constexpr size_t kPairSmem = 1024 + (size_t)kPairStages * kPairStage + (2 * kPairStages + 5) * 8 + 16 + 2 * kPairTokens * 4;

// A TMA load into this CTA that counts on the barrier at the same place of the pair's first CTA.
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar) & 0xFEFFFFFFu) : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar) {   // on the barrier of both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void arrive_first(uint64_t *bar) {   // on the barrier of the pair's first CTA
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(bar)));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kPairWarps * 32, 1)
k_linear_pair(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, LinearArgs p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int NT = kPairTokens, STAGES = kPairStages, STAGE = kPairStage, W_BYTES = LT * TC_BK, EW = kPairWarps - 2, COLS = 512;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + STAGES * STAGE);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + 2;
    uint64_t *drain = tempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    float *s_xs = reinterpret_cast<float *>(tmem_slot + 4);   // 2 x NT
    __shared__ volatile int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
    const int tile0 = blockIdx.x / 2, dt = gridDim.x / 2;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 2 * EW);
        }
        mbar_init(drain, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    __syncwarp();
    cluster_arrive();
    cluster_wait();   // both CTAs' barriers are set up and both have their TMEM
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            pdl_wait();
            for (int tile = tile0; tile < p.tiles && ok; tile += dt) {
                const int n0 = (tile % p.tiles_n) * 2 * LT + rank * LT, m0 = (tile / p.tiles_n) * NT + rank * (NT / 2);
                for (int kb = 0; kb < p.steps; kb++, it++) {
                    const int s = it % STAGES;
                    uint8_t *sw = smem + s * STAGE;
                    if (it >= STAGES && !mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * STAGE);
                    tma_load_2d_pair(sw, &map_w, &full[s], kb * TC_BK, n0);
                    tma_load_2d_pair(sw + W_BYTES, &map_x, &full[s], kb * TC_BK, m0);
                }
            }
            if (!ok) {
                atomicOr(&g_ops_timeout, 1);
                abort_flag = 1;
            }
            // copies in flight: the first CTA sees all of both
            if (!ok && rank == 0)
                for (int k = max(0, it - STAGES); k < it; k++) mbar_wait(&full[k % STAGES], (k / STAGES) & 1, nullptr);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = idesc_i8(2 * LT, NT);
            int it = 0, tc = 0;
            bool ok = true;
            for (int tile = tile0; tile < p.tiles && ok; tile += dt, tc++) {
                const int b = tc & 1;
                if (tc >= 2 && !mbar_wait(&tempty[b], ((tc >> 1) - 1) & 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < p.steps; kb++, it++) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&full[s], (it / STAGES) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t wd = smem_desc_sw128(smem_addr(smem + s * STAGE));
                    const uint64_t xd = smem_desc_sw128(smem_addr(smem + s * STAGE + W_BYTES));
#pragma unroll
                    for (int k = 0; k < TC_BK / 32; k++)
                        mma_i8_pair(tmem + (uint32_t)(b * NT), wd + 2 * k, xd + 2 * k, idesc, kb > 0 || k > 0);
                    mma_commit_pair(&empty[s]);
                }
                if (ok) mma_commit_pair(&tfull[b]);
            }
            if (!ok) {
                atomicOr(&g_ops_timeout, 1);
                abort_flag = 1;
            }
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(drain)) : "memory");
            mbar_wait(drain, 0, nullptr);
        }
    } else {
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int PC = NT / (EW / 4);
        pdl_wait();
        T *out = static_cast<T *>(p.out);
        int tc = 0;
        for (int tile = tile0; tile < p.tiles; tile += dt, tc++) {
            const int b = tc & 1;
            const int n0 = (tile % p.tiles_n) * 2 * LT + rank * LT, m0 = (tile / p.tiles_n) * NT;
            const int ch = n0 + 32 * q + lane;
            const bool there = ch < p.n;
            const float ws = there ? p.ws[ch] : 0.0f, bias = there && p.bias ? p.bias[ch] : 0.0f;
            float *xs = s_xs + b * NT;
            for (int i = threadIdx.x - 64; i < NT; i += EW * 32) xs[i] = m0 + i < p.m ? p.xs[m0 + i] : 0.0f;
            const bool got = mbar_wait(&tfull[b], (tc >> 1) & 1, &abort_flag);
            if (epilogue_any<EW * 32>(!got)) {
                if (!got) {
                    atomicOr(&g_ops_timeout, 1);
                    abort_flag = 1;
                }
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tbase = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(b * NT + part * PC);
#pragma unroll 1
            for (int c0 = 0; c0 < PC; c0 += 32) {
                uint32_t v[32];
                tmem_ld32(tbase + c0, v);
                if (c0 + 32 == PC) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive_first(&tempty[b]);
                }
                if (!there) continue;
                const int j0 = part * PC + c0, most = p.m - m0 - j0;
                T *o = out + (int64_t)(m0 + j0) * p.ldo + ch;
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j < most) o[j * p.ldo] = finish<T>((int)v[j], xs[j0 + j], ws, bias, p.bias != nullptr);
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_arrive();
    cluster_wait();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

// Rows of codes as a TMA map of boxes of `box` rows by 128 bytes, 128-byte swizzled.
bool codes_map(CUtensorMap *map, const int8_t *p, int64_t ld, int64_t rows, int64_t k, int box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld : (k + 15) / 16 * 16)};
    cuuint32_t boxes[2] = {TC_BK, (cuuint32_t)box};
    cuuint32_t one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), dims, strides, boxes, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, typename T, typename TX>
int launch_linear(const int8_t *x, int64_t ldx, const int8_t *w, int64_t ldw, int64_t k, LinearArgs p, bool after_quantise,
                  cudaStream_t st) {
    constexpr bool kQuantises = !std::is_void<TX>::value;
    alignas(64) CUtensorMap mw, mx;
    if (!codes_map(&mw, w, ldw, p.n, k, LT) || (!kQuantises && !codes_map(&mx, x, ldx, p.m, k, NT)))
        return ops_fail(CZG_E_DEVICE, "no tensor map for the operands");
    const int64_t tiles = (int64_t)p.tiles_n * ((p.m + NT - 1) / NT);
    if (tiles > 0x7FFFFFFF / 8) return ops_fail(CZG_E_LIMIT, "too many tiles");
    p.tiles = (int)tiles;
    const int per_cta = (p.steps + p.split - 1) / p.split;   // the ring need not be longer than a tile's stretch of k
    const int fit = (int)((kRingBytes - (p.split > 1 ? LT * NT * 4 : 0)) / LinearCfg<NT>::kStage);
    if (kQuantises && per_cta > fit) return ops_fail(CZG_E_LIMIT, "more steps than the ring holds");
    p.stages = per_cta < fit && (p.split > 1 || kQuantises) ? per_cta : fit;
    const size_t smem = LinearCfg<NT>::smem(p.stages, p.split);
    static std::atomic<int> ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return ops_fail(CZG_E_DEVICE, "no device");
    if (!ready[dev]) {
        if (int e = ops_cuda(cudaFuncSetAttribute(k_linear_tc<NT, T, TX>, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024)))
            return e;
        ready[dev] = 1;
    }
    const int grid = p.split > 1 || kQuantises ? p.tiles * p.split : p.tiles < sm_count() ? p.tiles : sm_count();
    return ops_cuda(ops_launch(k_linear_tc<NT, T, TX>, dim3((unsigned)grid), LinearCfg<NT>::kWarps * 32, smem, st, after_quantise,
                               p.split, mw, mx, p));
}

template <typename T>
int launch_pair(const int8_t *x, int64_t ldx, const int8_t *w, int64_t ldw, int64_t k, LinearArgs p, bool after_quantise,
                cudaStream_t st) {
    alignas(64) CUtensorMap mw, mx;
    if (!codes_map(&mw, w, ldw, p.n, k, LT) || !codes_map(&mx, x, ldx, p.m, k, kPairTokens / 2))
        return ops_fail(CZG_E_DEVICE, "no tensor map for the operands");
    p.tiles_n = (int)(((int64_t)p.n + 2 * LT - 1) / (2 * LT));
    const int64_t tiles = (int64_t)p.tiles_n * (((int64_t)p.m + kPairTokens - 1) / kPairTokens);
    if (tiles > 0x7FFFFFFF / 8) return ops_fail(CZG_E_LIMIT, "too many tiles");
    p.tiles = (int)tiles;
    static std::atomic<int> ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return ops_fail(CZG_E_DEVICE, "no device");
    if (!ready[dev]) {
        if (int e = ops_cuda(cudaFuncSetAttribute(k_linear_pair<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem)))
            return e;
        ready[dev] = 1;
    }
    const int pairs = sm_count() / 2;
    return ops_cuda(ops_launch(k_linear_pair<T>, dim3((unsigned)(2 * (p.tiles < pairs ? p.tiles : pairs))), kPairWarps * 32,
                               kPairSmem, st, after_quantise, 2, mw, mx, p));
}

// Calls whose x rows the product can quantise itself: at most 16 rows, 64 KB of bf16 in all, whose
// codes a cluster's rings hold.
constexpr int kSmallRows = 16, kSmallValues = 32768, kSmallSteps = 11;   // steps a CTA's ring holds
static_assert(kSmallSteps * LinearCfg<kSmallRows>::kStage + LT * kSmallRows * 4 <= kRingBytes, "the codes of all steps have their place");
bool small_call(int64_t m, int64_t k) {
    return m <= kSmallRows && m * k <= kSmallValues && k <= 8 * kSmallSteps * TC_BK;
}
// Over how many CTAs it splits k: as many as there are SMs, of at least two steps each, and
// no more steps than the ring holds.
int small_split(int64_t tiles_n, int steps) {
    int split = 1;
    while (split < 8 && (steps > split * kSmallSteps || (tiles_n * split * 2 <= sm_count() && steps >= split * 4))) split *= 2;
    return split;
}
// Whether that is the better form.  It saves a launch (4 us of a Python call), but each tile's CTA
// loads its steps of weights with no other tile's under way behind them, and quantises all of x.  On
// the device, one kernel and the two of two calls, us, for 1 x 384: 5.0 and 5.6 at 512 channels, 6.2 and 7.5 at
// 32,768, 15.4 and 14.2 at 128,000; 1 x 2048: 6.1 and 6.9, 31.8 and 18.1, 116 and 50; 8 x 2048: 10.4
// and 7.1, 54.8 and 18.3, 209 and 51.  So: while an SM has at most kSmallTurns steps to load, one
// wave of tiles after the other.
constexpr int64_t kSmallTurns = 8;
bool small_pays(int64_t n, int64_t k) {
    const int64_t tiles = (n + LT - 1) / LT, steps = (k + TC_BK - 1) / TC_BK;
    const int split = small_split(tiles, (int)steps), sms = sm_count();
    return (tiles * split + sms - 1) / sms * ((steps + split - 1) / split) <= kSmallTurns;
}

// Which tile, and over how many CTAs k is split: the least of a model of the time in
// cycles.  A step (128 bytes of k) costs about 600 + 1.5 nt in one CTA, whatever its
// tokens (4096 x 4096 weights, one tile a CTA, 32 steps: 15.2 us at nt = 16, 17.9 at 128,
// 21 at 256), so more tokens a tile pay as long as the tiles fill the SMs, and below that
// a split of k does (48 tokens: 17.3 us whole, 9.7 in 4; 128: 17.9 and 10.5).
struct LinearShape { int nt, split; };

LinearShape linear_shape(int64_t m, int64_t n, int steps) {
    const int sms = sm_count();
    LinearShape best{16, 1};
    double least = 1e300;
    for (int nt : {16, 32, 64, 128, 256, 512}) {
        const bool pair = nt == 512;   // two CTAs, 256 x 256
        const int64_t tiles = ((n + LT - 1) / LT + pair) / (1 + pair) * ((m + (pair ? 256 : nt) - 1) / (pair ? 256 : nt));
        for (int s : {1, 2, 4, 8}) {
            if (s > 1 && (nt > 128 || nt * s > 512 || s > steps || tiles * s > sms)) break;
            const int64_t places = pair ? sms / 2 : sms;
            const double waves = (double)((tiles * s + places - 1) / places);
            const double step = pair ? 760.0 : 600.0 + 1.5 * nt;
            const double cost = waves * ((steps + s - 1) / s) * step + 10.0 * nt + (s > 1 ? 1200 + 20.0 * nt : 0);
            if (cost < least) {
                least = cost;
                best = {nt, s};
            }
        }
    }
    return best;
}

template <typename T>
int quantize(const void *x, int64_t ldx, int64_t m, int64_t k, int8_t *codes, int64_t ldc, float *scales, cudaStream_t st) {
    const int64_t turns = (k + 7) / 8;
    const int vec = aligned(x, 16) && (m == 1 || ldx * sizeof(T) % 16 == 0);
    // With rows for all of an SM's warps: a warp a row while it fits its registers (8192 x 2048
    // bf16: 15.1 us; a CTA a row 16.7), then a CTA of 4 warps (8192 x 4096: 25.0 us, 4.0 TB/s of
    // rows and codes; a warp a row 28.6, whose few warps load and compute in step; 8 warps
    // 31.3).  Few rows, and rows that 4 warps would have to read twice (2000 x 8192: 18.7 us,
    // 13.9 with 8), get 8 warps each.
    const bool many = m >= 16 * sm_count();
    if (many && k <= (sizeof(T) == 2 ? 2048 : 1024)) {
        const dim3 grid((unsigned)((m + 3) / 4));
        auto go = [&](auto kern) {
            return ops_cuda(ops_launch(kern, grid, 128, 0, st, true, 1, static_cast<const T *>(x), ldx, (int)m, (int)k, vec, codes, ldc, scales));
        };
        if (turns <= 2 * 32) return go(k_quantize_rows_warp<T, 2>);
        if constexpr (sizeof(T) == 2)   // fp32 rows of this branch have 4 turns at most
            if (turns > 4 * 32) return go(k_quantize_rows_warp<T, 8>);
        return go(k_quantize_rows_warp<T, 4>);
    }
    const int most = many && k <= kQuantThreads / 2 * 8 * kHeld ? kQuantThreads / 2 : kQuantThreads;
    const int threads = turns >= most ? most : (int)((turns + 31) / 32 * 32);
    return ops_cuda(ops_launch(k_quantize_rows<T>, dim3((unsigned)m), threads, 0, st, true, 1, static_cast<const T *>(x), ldx,
                               k, vec, codes, ldc, scales));
}

int quantize_any(const void *x, int dtype, int64_t ldx, int64_t m, int64_t k, int8_t *codes, int64_t ldc, float *scales,
                 cudaStream_t st) {
    if (dtype == CZG_F32) return quantize<float>(x, ldx, m, k, codes, ldc, scales, st);
    if (dtype == CZG_BF16) return quantize<__nv_bfloat16>(x, ldx, m, k, codes, ldc, scales, st);
    return quantize<__half>(x, ldx, m, k, codes, ldc, scales, st);
}

template <typename T>
int linear(const int8_t *x, int64_t ldx, const float *xs, const int8_t *w, int64_t ldw, const float *ws, const float *bias,
           int64_t m, int64_t n, int64_t k, void *out, int64_t ldo, bool after_quantise, cudaStream_t st) {
    LinearArgs p{xs, ws, bias, out, ldo, (int)m, (int)n, (int)((k + TC_BK - 1) / TC_BK), (int)((n + LT - 1) / LT), 0, 0, 1,
                 aligned(out, 4 * sizeof(T)) && ldo % 4 == 0};
    LinearShape shape = linear_shape(m, n, p.steps);

    p.split = shape.split;
    if (shape.nt == 16) return launch_linear<16, T, void>(x, ldx, w, ldw, k, p, after_quantise, st);
    if (shape.nt == 32) return launch_linear<32, T, void>(x, ldx, w, ldw, k, p, after_quantise, st);
    if (shape.nt == 64) return launch_linear<64, T, void>(x, ldx, w, ldw, k, p, after_quantise, st);
    if (shape.nt == 512) return launch_pair<T>(x, ldx, w, ldw, k, p, after_quantise, st);
    if (shape.nt == 128) return launch_linear<128, T, void>(x, ldx, w, ldw, k, p, after_quantise, st);
    return launch_linear<256, T, void>(x, ldx, w, ldw, k, p, after_quantise, st);
}

int linear_any(const int8_t *x, int64_t ldx, const float *xs, const int8_t *w, int64_t ldw, const float *ws, const float *bias,
               int64_t m, int64_t n, int64_t k, void *out, int dtype, int64_t ldo, bool after_quantise, cudaStream_t st) {
    if (dtype == CZG_F32) return linear<float>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, after_quantise, st);
    if (dtype == CZG_BF16) return linear<__nv_bfloat16>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, after_quantise, st);
    return linear<__half>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, after_quantise, st);
}

template <typename T, typename TX>
int linear_small(const void *x, int64_t ldx, const int8_t *w, int64_t ldw, const float *ws, const float *bias, int64_t m,
                 int64_t n, int64_t k, void *out, int64_t ldo, cudaStream_t st) {
    LinearArgs p{nullptr, ws, bias, out, ldo, (int)m, (int)n, (int)((k + TC_BK - 1) / TC_BK), (int)((n + LT - 1) / LT), 0, 0, 1,
                 aligned(out, 4 * sizeof(T)) && ldo % 4 == 0, x, ldx, (int)k, aligned(x, 16) && (m == 1 || ldx * sizeof(TX) % 16 == 0)};
    p.split = small_split(p.tiles_n, p.steps);
    return launch_linear<kSmallRows, T, TX>(nullptr, 0, w, ldw, k, p, false, st);
}

template <typename T>
int linear_small_of(int dtype, const void *x, int64_t ldx, const int8_t *w, int64_t ldw, const float *ws, const float *bias,
                    int64_t m, int64_t n, int64_t k, void *out, int64_t ldo, cudaStream_t st) {
    if (dtype == CZG_F32) return linear_small<T, float>(x, ldx, w, ldw, ws, bias, m, n, k, out, ldo, st);
    if (dtype == CZG_BF16) return linear_small<T, __nv_bfloat16>(x, ldx, w, ldw, ws, bias, m, n, k, out, ldo, st);
    return linear_small<T, __half>(x, ldx, w, ldw, ws, bias, m, n, k, out, ldo, st);
}

const char *check_codes(const int8_t *p, int64_t ld, int64_t rows, int64_t k) {
    if (!aligned(p, 16) || ld % 16 != 0) return "rows of codes must begin on 16-byte boundaries";
    if (rows > 1 && ld < k) return "rows of codes overlap";
    return nullptr;
}

int check_linear(const int8_t *w, int64_t ldw, const float *ws, int64_t m, int64_t n, int64_t k, const void *out,
                 int out_dtype, int64_t ldo) {
    if (!w || !ws || !out) return ops_fail(CZG_E_ARG, "null pointer");
    if (!dtype_ok(out_dtype)) return ops_fail(CZG_E_ARG, "unknown out_dtype");
    if (const char *why = check_codes(w, ldw, n, k)) return ops_fail(CZG_E_ARG, why);
    if (!aligned(out, (uintptr_t)elem_bytes(out_dtype))) return ops_fail(CZG_E_ARG, "out is not aligned to its type");
    if (m > 1 && ldo < n) return ops_fail(CZG_E_ARG, "rows of out overlap");
    return CZG_OK;
}

// out must not lie over an operand, whose rows other CTAs may still read: ranges that
// meet are refused, but for columns side by side in rows of one stride.
int check_apart(const void *out, int64_t out_ld, int64_t out_row, const void *in, int64_t in_ld, int64_t in_row, int64_t out_rows,
                int64_t in_rows, const char *why) {   // in bytes
    const intptr_t a = reinterpret_cast<intptr_t>(out), b = reinterpret_cast<intptr_t>(in);
    if (a + (out_rows - 1) * out_ld + out_row <= b || b + (in_rows - 1) * in_ld + in_row <= a) return CZG_OK;
    if (out_ld == in_ld && out_ld > 0) {
        const int64_t d = ((b - a) % out_ld + out_ld) % out_ld;   // where in's columns begin, counted from out's
        if (d >= out_row && d + in_row <= out_ld) return CZG_OK;
    }
    return ops_fail(CZG_E_ARG, why);
}

constexpr int64_t kMaxRows = 0x7FFFFE00;   // a tile behind the last row is still an int

int check_sizes(int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 0 || k < 1) return ops_fail(CZG_E_ARG, "m and n must not be negative, k must be at least 1");
    if (k > CZG_LINEAR_MAX_K) return ops_fail(CZG_E_LIMIT, "k is beyond CZG_LINEAR_MAX_K");
    if (m > kMaxRows || n > kMaxRows) return ops_fail(CZG_E_LIMIT, "m and n must be at most 2^31 - 512");
    return CZG_OK;
}

int check_x(const void *x, int dtype, int64_t ldx, int64_t m, int64_t k) {
    if (!x) return ops_fail(CZG_E_ARG, "null pointer");
    if (!dtype_ok(dtype)) return ops_fail(CZG_E_ARG, "unknown dtype");
    if (!aligned(x, (uintptr_t)elem_bytes(dtype))) return ops_fail(CZG_E_ARG, "x is not aligned to its type");
    if (m > 1 && ldx < 0) return ops_fail(CZG_E_ARG, "ld_x is negative");
    return CZG_OK;
}

int64_t codes_ld(int64_t k) { return (k + 15) & ~(int64_t)15; }

}  // namespace
}  // namespace czg

using namespace czg;

extern "C" const char *czg_ops_last_error(void) { return g_ops_error; }

extern "C" int czg_ops_check(void) {
    int a = 0, b = 0;
    if (int st = ops_cuda(cudaDeviceSynchronize())) return st;
    if (int st = take_timeouts(&a)) return st;
    if (int st = kv4_timeouts(&b)) return st;
    return a || b ? ops_fail(CZG_E_TIMEOUT, "a bounded wait of a kernel ran out; its results are incomplete") : CZG_OK;
}

extern "C" int czg_quantize_rows(const void *x, int dtype, int64_t ld_x, int64_t m, int64_t k, int8_t *codes,
                                 int64_t ld_codes, float *scales, void *stream) {
    if (m < 0 || k < 1) return ops_fail(CZG_E_ARG, "m must not be negative, k must be at least 1");
    if (m > kMaxRows) return ops_fail(CZG_E_LIMIT, "m must be at most 2^31 - 512");
    if (m == 0) return CZG_OK;
    if (int st = check_x(x, dtype, ld_x, m, k)) return st;
    if (!codes || !scales) return ops_fail(CZG_E_ARG, "null pointer");
    if (const char *why = check_codes(codes, ld_codes, m, codes_ld(k))) return ops_fail(CZG_E_ARG, why);
    return quantize_any(x, dtype, ld_x, m, k, codes, ld_codes, scales, static_cast<cudaStream_t>(stream));
}

extern "C" int czg_linear_i8(const int8_t *x, int64_t ld_x, const float *x_scale, const int8_t *w, int64_t ld_w,
                             const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k, void *out,
                             int out_dtype, int64_t ld_out, void *stream) {
    if (int st = check_sizes(m, n, k)) return st;
    if (m == 0 || n == 0) return CZG_OK;
    if (!x || !x_scale) return ops_fail(CZG_E_ARG, "null pointer");
    if (const char *why = check_codes(x, ld_x, m, k)) return ops_fail(CZG_E_ARG, why);
    if (int st = check_linear(w, ld_w, w_scale, m, n, k, out, out_dtype, ld_out)) return st;
    const int eb = elem_bytes(out_dtype);
    if (int st = check_apart(out, ld_out * eb, n * eb, x, ld_x, k, m, m, "out lies over x")) return st;
    if (int st = check_apart(out, ld_out * eb, n * eb, w, ld_w, k, m, n, "out lies over w")) return st;
    return linear_any(x, ld_x, x_scale, w, ld_w, w_scale, bias, m, n, k, out, out_dtype, ld_out, false,
                      static_cast<cudaStream_t>(stream));
}

static uint64_t rows_workspace(int64_t m, int64_t k) { return (uint64_t)m * (uint64_t)codes_ld(k) + (((uint64_t)m * 4 + 15) & ~15ull); }

extern "C" uint64_t czg_linear_i8_workspace(int64_t m, int64_t k) {
    return m <= 0 || k <= 0 || small_call(m, k) ? 0 : rows_workspace(m, k);
}

extern "C" uint64_t czg_linear_i8_dynamic_workspace(int64_t m, int64_t n, int64_t k) {
    return m <= 0 || n <= 0 || k <= 0 || (small_call(m, k) && small_pays(n, k)) ? 0 : rows_workspace(m, k);
}

extern "C" int czg_linear_i8_dynamic(const void *x, int dtype, int64_t ld_x, const int8_t *w, int64_t ld_w,
                                     const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k,
                                     void *out, int out_dtype, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream) {
    if (int st = check_sizes(m, n, k)) return st;
    if (m == 0 || n == 0) return CZG_OK;
    if (int st = check_x(x, dtype, ld_x, m, k)) return st;
    if (int st = check_linear(w, ld_w, w_scale, m, n, k, out, out_dtype, ld_out)) return st;
    const int eb = elem_bytes(out_dtype), xb = elem_bytes(dtype);
    if (int st = check_apart(out, ld_out * eb, n * eb, x, ld_x * xb, k * xb, m, m, "out lies over x")) return st;
    if (int st = check_apart(out, ld_out * eb, n * eb, w, ld_w, k, m, n, "out lies over w")) return st;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (small_call(m, k) && (!ws || ws_bytes < rows_workspace(m, k) || small_pays(n, k))) {
        if (out_dtype == CZG_F32) return linear_small_of<float>(dtype, x, ld_x, w, ld_w, w_scale, bias, m, n, k, out, ld_out, st);
        if (out_dtype == CZG_BF16)
            return linear_small_of<__nv_bfloat16>(dtype, x, ld_x, w, ld_w, w_scale, bias, m, n, k, out, ld_out, st);
        return linear_small_of<__half>(dtype, x, ld_x, w, ld_w, w_scale, bias, m, n, k, out, ld_out, st);
    }
    if (!ws || !aligned(ws, 16)) return ops_fail(CZG_E_ARG, "the workspace must begin on a 16-byte boundary");
    if (ws_bytes < czg_linear_i8_workspace(m, k)) return ops_fail(CZG_E_ARG, "the workspace is too small");
    int8_t *codes = static_cast<int8_t *>(ws);
    float *scales = reinterpret_cast<float *>(codes + m * codes_ld(k));
    if (int e = quantize_any(x, dtype, ld_x, m, k, codes, codes_ld(k), scales, st)) return e;
    return linear_any(codes, codes_ld(k), scales, w, ld_w, w_scale, bias, m, n, k, out, out_dtype, ld_out, true, st);
}
