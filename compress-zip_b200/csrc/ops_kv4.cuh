// ops_kv4.cuh -- what the kernels of the 4-bit key/value cache share (include/czg_ops.h).
#pragma once
#include "ops_common.cuh"

namespace czg {

const char *check_kv4(const czg_kv4 *c);   // ops_kv4.cu

namespace {

struct KvScale {   // one entry of one head
    __nv_bfloat16 k_step, k_lo, v_step, v_lo;
};
static_assert(sizeof(KvScale) == 8, "the layout of czg_kv4.scales");

// The slot of sequence b, or -1 for a padded place (a slot beyond the cache counts as one).
__device__ __forceinline__ int kv4_slot(const czg_kv4 &c, const int32_t *slots, int b, bool report) {
    const int s = slots[b];
    if (s >= c.n_slots) {
        if (report) atomicOr(c.status, CZG_KV4_BAD_SLOT);
        return -1;
    }
    return s < 0 ? -1 : s;
}

// The entries of sequence b, cut to [0, most].
__device__ __forceinline__ int kv4_length(const czg_kv4 &c, const int32_t *lengths, int b, int most, bool report) {
    const int n = lengths[b];
    if (n < 0 || n > most) {
        if (report) atomicOr(c.status, CZG_KV4_BAD_LENGTH);
        return n < 0 ? 0 : most;
    }
    return n;
}

__device__ __forceinline__ int64_t kv4_row(const czg_kv4 &c, int slot, int head, int entry) {
    return ((int64_t)slot * c.n_heads + head) * c.capacity + entry;
}

// Reports a slot that two sequences of a writing call name.  One CTA; a bit a slot, in
// ranges of kDistinctBits slots.
constexpr int kDistinctBits = 32768;
__host__ __device__ constexpr int distinct_ranges(int n_slots) { return (n_slots - 1) / kDistinctBits + 1; }
__host__ __device__ constexpr int distinct_base(int range) { return range * kDistinctBits; }
static_assert(distinct_ranges(1) == 1 && distinct_ranges(kDistinctBits) == 1 && distinct_ranges(kDistinctBits + 1) == 2 &&
              distinct_base(distinct_ranges(0x7FFFFFFF) - 1) == 0x7FFFFFFF / kDistinctBits * kDistinctBits,
              "the last range of the most slots still begins at an int");
__device__ __forceinline__ void kv4_check_distinct(const czg_kv4 &c, const int32_t *slots, int b) {
    __shared__ uint32_t seen[kDistinctBits / 32];
    for (int range = 0, ranges = distinct_ranges(c.n_slots); range < ranges; range++) {   // counted: the next base may pass an int
        const int base = distinct_base(range), bits = min(kDistinctBits, c.n_slots - base);
        for (int i = threadIdx.x; i < (bits + 31) / 32; i += blockDim.x) seen[i] = 0;
        __syncthreads();
#pragma unroll 8
        for (int i = threadIdx.x; i < b; i += blockDim.x) {
            const int slot = slots[i], s = slot - base;
            if (slot >= 0 && s >= 0 && s < bits && (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u))
                atomicOr(c.status, CZG_KV4_TWICE);
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace czg
