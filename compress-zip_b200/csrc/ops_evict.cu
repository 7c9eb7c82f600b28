// ops_evict.cu -- eviction from the 4-bit cache by accumulated attention weight
// (include/czg_ops.h).
#include "ops_kv4.cuh"

namespace czg {
namespace {

constexpr int kThreads = 512;

// Order of the weights as unsigned numbers: larger weight, larger key; NaN above all.
__device__ __forceinline__ uint32_t rank_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.0f);   // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the CTA of x, and the sum over the threads before this one.
__device__ __forceinline__ int scan(int x, int *before, int *part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    __syncthreads();   // part's readers of the last call are done
    if (lane == 31) part[warp] = y;
    __syncthreads();
    int sum = 0, below = 0;
    for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) below += part[w];
        sum += part[w];
    }
    *before = below + y - x;
    return sum;
}

// One CTA a sequence and head.  The weight that divides the kept from the others is
// found digit by digit, 8 bits at a time from the top, by counting; then the entries
// are walked in order, kThreads at a time: what stays is read, the CTA waits, and it is
// written to its place.  No place is written before it was read: the i-th kept entry
// lies at i or behind it.
template <int D>
__global__ void __launch_bounds__(kThreads) k_kv4_evict(czg_kv4 c, const int32_t *__restrict__ slots,
                                                        const int32_t *__restrict__ lengths, int b, int max_len, int budget,
                                                        int recent, int32_t *__restrict__ kept, int32_t *__restrict__ new_len) {
    __shared__ int hist[256], part[kThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    if (s == b) {   // one more sequence's worth of CTAs: the first looks for repeated slots
        if (h == 0) kv4_check_distinct(c, slots, b);
        return;
    }
    const bool first = tid == 0 && h == 0;
    const int slot = kv4_slot(c, slots, s, first);
    const int n = slot < 0 ? 0 : kv4_length(c, lengths, s, min(max_len, c.capacity), first);
    if (new_len && first) new_len[s] = min(n, budget);
    int32_t *kp = kept ? kept + ((int64_t)s * c.n_heads + h) * budget : nullptr;
    if (n <= budget) {
        if (kp)
            for (int i = tid; i < budget; i += kThreads) kp[i] = i < n ? i : -1;
        return;
    }
    const int64_t base = kv4_row(c, slot, h, 0);
    float *w = c.weights + base;
    const int old = n - recent;           // entries that are ranked
    if (tid == 0) {
        s_prefix = 0;
        s_need = budget - recent;         // how many of them stay
    }
    __syncthreads();
    for (int shift = 24; shift >= 0 && budget > recent; shift -= 8) {
        for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int i = tid; i < old; i += kThreads) {
            const uint32_t key = rank_key(w[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[key >> shift & 255u], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int need = s_need, d = 255;
            while (d > 0 && hist[d] < need) need -= hist[d--];   // d > 0: weights that another call changes meanwhile
            s_need = need;
            s_prefix = prefix | (uint32_t)d << shift;
        }
        __syncthreads();
    }
    // keys above the threshold stay, and the first s_need of those equal to it
    const uint32_t threshold = s_prefix;
    const int equal = budget > recent ? s_need : 0;
    int done = 0, met = 0;   // kept so far, equal keys met so far
    for (int i0 = 0; i0 < n; i0 += kThreads) {
        const int i = i0 + tid;
        const float wi = i < n ? w[i] : 0.0f;
        const uint32_t key = rank_key(wi);
        const bool ranked = i < old && budget > recent;
        const bool same = ranked && key == threshold;
        int before_same, before;
        const int all_same = scan(same, &before_same, part);
        const bool stay = i < n && (i >= old || (ranked && key > threshold) || (same && met + before_same < equal));
        const int count = scan(stay, &before, part);
        uint4 rk[D / 32], rv[D / 32];
        KvScale sc = {};
        if (stay) {
            const uint4 *pk = reinterpret_cast<const uint4 *>(c.k + (base + i) * (D / 2));
            const uint4 *pv = reinterpret_cast<const uint4 *>(c.v + (base + i) * (D / 2));
#pragma unroll
            for (int x = 0; x < D / 32; x++) {
                rk[x] = pk[x];
                rv[x] = pv[x];
            }
            sc = static_cast<const KvScale *>(c.scales)[base + i];
        }
        __syncthreads();   // all of this stretch is read
        const int to = done + before;
        if (stay && to < budget) {
            if (to != i) {
                uint4 *pk = reinterpret_cast<uint4 *>(c.k + (base + to) * (D / 2));
                uint4 *pv = reinterpret_cast<uint4 *>(c.v + (base + to) * (D / 2));
#pragma unroll
                for (int x = 0; x < D / 32; x++) {
                    pk[x] = rk[x];
                    pv[x] = rv[x];
                }
                static_cast<KvScale *>(c.scales)[base + to] = sc;
                w[to] = wi;
            }
            if (kp) kp[to] = i;
        }
        done += count;
        met += all_same;
    }
}

}  // namespace
}  // namespace czg

using namespace czg;

extern "C" int czg_kv4_evict(const czg_kv4 *cache, const int32_t *slots, const int32_t *lengths, int32_t b, int32_t max_len,
                             int32_t budget, int32_t recent, int32_t *kept, int32_t *new_lengths, void *stream) {
    if (b < 0 || max_len < 0) return ops_fail(CZG_E_ARG, "b and max_len must not be negative");
    if (const char *why = check_kv4(cache)) return ops_fail(CZG_E_ARG, why);
    if (cache->head_dim != 64 && cache->head_dim != 128) return ops_fail(CZG_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (!cache->weights) return ops_fail(CZG_E_ARG, "the cache keeps no weights to rank entries by");
    if (budget < 1 || recent < 0 || recent > budget) return ops_fail(CZG_E_ARG, "1 <= budget and 0 <= recent <= budget are needed");
    if (b > 65534) return ops_fail(CZG_E_LIMIT, "more than 65,534 sequences in a call");
    if (max_len > CZG_KV4_EVICT_MAX) return ops_fail(CZG_E_LIMIT, "max_len is beyond CZG_KV4_EVICT_MAX");
    if (!slots || !lengths) return ops_fail(CZG_E_ARG, "null pointer");
    if (new_lengths == lengths) return ops_fail(CZG_E_ARG, "new_lengths must not be the array of lengths");
    if (b == 0) return CZG_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto kern = cache->head_dim == 64 ? k_kv4_evict<64> : k_kv4_evict<128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)cache->n_heads, (unsigned)b + 1), kThreads, 0, st, false, 1, *cache, slots,
                               lengths, b, max_len, budget, recent, kept, new_lengths));
}
