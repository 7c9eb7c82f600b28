// ops_evict.cu -- eviction from the 4-bit cache by accumulated attention weight
// (include/czg_ops.h).
#include "common.cuh"
#include "ops_kv4.cuh"

namespace czg {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kDigit = 11, kBins = 1 << kDigit;   // three digits: 11, 11 and 10 bits
constexpr int kStretch = 8 * kThreads;            // entries sorted out at a time
constexpr int kTasks = 8;                         // 16-byte pieces a thread holds between reading and writing

// Order of the weights as unsigned numbers: larger weight, larger key; NaN above all.
__device__ __forceinline__ uint32_t rank_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.0f);   // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of x over the CTA (returned) and over the threads before this one.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t *before, uint32_t *part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    __syncthreads();   // the readers of part's last contents are done
    if (lane == 31) part[warp] = y;
    __syncthreads();
    uint32_t sum = 0, below = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        const uint32_t p = part[w];
        below += w < warp ? p : 0;
        sum += p;
    }
    *before = below + y - x;
    return sum;
}

// One CTA a sequence and head.
// 1. The weight that divides the kept from the others, digit by digit from the top, by
//    counting: each pass counts the next digit of the weights that share the digits found
//    so far, and a scan over the counts finds the digit that the last one kept has.
// 2. Stretch by stretch, in order: who stays (keys above the threshold, the first ones
//    equal to it, the recent entries), numbered by a scan.
// 3. A stretch's entries move, kThreads * kTasks pieces of 16 bytes at a time: all are read,
//    the CTA waits, all are written.  The i-th kept entry lies at place i or behind it, so
//    no place is written before it was read.
// Bound by reading and writing what moves: 48 x 8 heads of up to 4096 entries cut to 1024
// (D = 128, 114 MB moved) take 23.5 us, 4.9 TB/s; one head from 1024 to 700 takes 6.5 us of
// latency (three passes of counting, two scans, one move).  256 threads a CTA took 4 us
// more on the batch, one CTA an SM (119 registers) 10 us more.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_evict(czg_kv4 c, const int32_t *slots,
                                                        const int32_t *lengths, int b, int max_len, int budget,
                                                        int recent, int32_t *__restrict__ kept, int32_t *__restrict__ new_len) {
    __shared__ uint32_t hist[kBins], part[kWarps];
    __shared__ int stay_list[kStretch];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();
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
    for (int shift = 32 - kDigit; budget > recent; shift = max(shift - kDigit, 0)) {
        const int bits = shift == 0 ? 32 - 2 * kDigit : kDigit;
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = bits + shift == 32 ? 0u : 0xFFFFFFFFu << (bits + shift);
#pragma unroll 8
        for (int i = tid; i < old; i += kThreads) {
            const uint32_t key = rank_key(w[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[key >> shift & (kBins - 1u) & ~(~0u << bits)], 1u);
        }
        __syncthreads();
        // bins from the top: thread i has the four below 4 i, so the scan counts larger keys
        constexpr int EACH = kBins / kThreads;
        uint32_t mine[EACH], sum = 0, above;
#pragma unroll
        for (int i = 0; i < EACH; i++) sum += mine[i] = hist[kBins - 1 - (tid * EACH + i)];
        const uint32_t need = (uint32_t)s_need;
        scan(sum, &above, part);
        if (above < need && need <= above + sum) {   // one thread, as long as the weights hold still
            int i = 0;
            uint32_t left = need - above;
            while (i < EACH - 1 && mine[i] < left) left -= mine[i++];
            s_need = (int)left;
            s_prefix = prefix | (uint32_t)(kBins - 1 - (tid * EACH + i)) << shift;
        }
        __syncthreads();
        if (shift == 0) break;
    }
    // keys above the threshold stay, and the first s_need of those equal to it
    const uint32_t threshold = s_prefix;
    const int equal = budget > recent ? s_need : 0;
    int done = 0, met = 0;   // kept so far, equal keys met so far
    for (int i0 = 0; i0 < n; i0 += kStretch) {
        constexpr int EACH = kStretch / kThreads;
        const int t0 = i0 + tid * EACH;   // this thread's entries, side by side
        uint32_t flags = 0, same = 0;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int i = t0 + j;
            if (i < old && budget > recent) {
                const uint32_t key = rank_key(w[i]);
                if (key > threshold) flags |= 1u << j;
                if (key == threshold) same |= 1u << j;
            } else if (i >= old && i < n) {
                flags |= 1u << j;
            }
        }
        uint32_t before;   // both counts at once: a stretch's fit 16 bits
        const uint32_t all = scan((uint32_t)__popc(flags) | (uint32_t)__popc(same) << 16, &before, part);
        const int same_before = met + (int)(before >> 16);
        int at = (int)(before & 0xFFFFu) + min(same_before, equal) - min(met, equal);   // within the stretch
        int may = equal - same_before;   // equal keys that may still stay
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            bool stay = flags >> j & 1u;
            if (same >> j & 1u) stay = may-- > 0;
            if (stay) stay_list[at++] = t0 + j;
        }
        const int same_all = (int)(all >> 16);
        const int count = min((int)(all & 0xFFFFu) + min(met + same_all, equal) - min(met, equal), max(budget - done, 0));
        met += same_all;
        __syncthreads();
        if (kp)
            for (int i = tid; i < count; i += kThreads) kp[done + i] = stay_list[i];
        // a row's pieces: D / 32 of keys and as many of values; ranges and weights go a thread a row
        constexpr int PIECES = D / 16, ROWS = kThreads * kTasks / PIECES, OWN = ROWS / kThreads;
        for (int r0 = 0; r0 < count; r0 += ROWS) {
            uint4 piece[kTasks];
            KvScale sc[OWN];
            float weight[OWN];
#pragma unroll
            for (int k = 0; k < kTasks; k++) {
                const int task = k * kThreads + tid, r = r0 + task / PIECES, p = task % PIECES;
                if (r < count && stay_list[r] != done + r)
                    piece[k] = reinterpret_cast<const uint4 *>((p < PIECES / 2 ? c.k : c.v) + (base + stay_list[r]) * (D / 2))[p % (PIECES / 2)];
            }
#pragma unroll
            for (int k = 0; k < OWN; k++) {
                const int r = r0 + k * kThreads + tid;
                if (r < count && stay_list[r] != done + r) {
                    sc[k] = static_cast<const KvScale *>(c.scales)[base + stay_list[r]];
                    weight[k] = w[stay_list[r]];
                }
            }
            __syncthreads();   // all of these are read
#pragma unroll
            for (int k = 0; k < kTasks; k++) {
                const int task = k * kThreads + tid, r = r0 + task / PIECES, p = task % PIECES;
                if (r < count && stay_list[r] != done + r)
                    reinterpret_cast<uint4 *>((p < PIECES / 2 ? c.k : c.v) + (base + done + r) * (D / 2))[p % (PIECES / 2)] = piece[k];
            }
#pragma unroll
            for (int k = 0; k < OWN; k++) {
                const int r = r0 + k * kThreads + tid;
                if (r < count && stay_list[r] != done + r) {
                    static_cast<KvScale *>(c.scales)[base + done + r] = sc[k];
                    w[done + r] = weight[k];
                }
            }
        }
        done += count;
        __syncthreads();   // stay_list is read; and this stretch's writes are done before the next weights are read
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
    return ops_cuda(ops_launch(kern, dim3((unsigned)cache->n_heads, (unsigned)b + 1), kThreads, 0, st, true, 1, *cache, slots,
                               lengths, b, max_len, budget, recent, kept, new_lengths));
}
