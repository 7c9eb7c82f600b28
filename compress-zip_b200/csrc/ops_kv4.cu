// ops_kv4.cu -- the key/value cache held in 4 bits (include/czg_ops.h): append, read
// and attention.
#include <cmath>

#include "ops_kv4.cuh"

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

// One warp a row of one head: the row's range by shuffles, then lane i's D / 32 values
// (dimensions i D/32 ..) as codes.  lo is rounded down and step up (each operation with
// the same direction), so every quotient lies in [0, 15].
template <typename T, int D>
__device__ __forceinline__ void quantise_row(const T *row, uint8_t *codes, __nv_bfloat16 *step_out, __nv_bfloat16 *lo_out) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    float x[N], lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = to_f32(row[lane * N + i]);
        bad |= !(fabsf(x[i]) <= 3.402823466e38f);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    bad = __any_sync(0xffffffffu, bad);
    lo = bf16_down(lo);
    float step = bf16_up(__fdiv_ru(__fsub_ru(hi, lo), 15.0f));
    if (bad || !(fabsf(lo) <= 3.402823466e38f) || !(step <= 3.402823466e38f)) step = lo = NAN;
    uint32_t byte[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        int c0 = 0, c1 = 0;
        if (step > 0.0f) {
            c0 = (int)rintf(__fdiv_rn(__fsub_rn(x[i], lo), step));
            c1 = (int)rintf(__fdiv_rn(__fsub_rn(x[i + 1], lo), step));
        }
        byte[i / 2] = (uint32_t)(c0 | c1 << 4);
    }
    if (N == 4)
        *reinterpret_cast<uint16_t *>(codes + 2 * lane) = (uint16_t)(byte[0] | byte[N / 2 - 1] << 8);
    else
        codes[lane] = (uint8_t)byte[0];
    if (lane == 0) {
        *step_out = __float2bfloat16_rn(step);
        *lo_out = __float2bfloat16_rn(lo);
    }
}

// Two warps a row, one for its key and one for its value; CTA 0 looks for repeated slots.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv4_append(czg_kv4 c, const T *__restrict__ k, Strides ks, const T *__restrict__ v,
                                                    Strides vs, const int32_t *__restrict__ slots,
                                                    const int32_t *__restrict__ lengths, int b, int t) {
    if (blockIdx.x == 0) {
        kv4_check_distinct(c, slots, b);
        return;
    }
    const int64_t id = ((int64_t)blockIdx.x - 1) * 8 + (threadIdx.x >> 5);
    const int64_t row = id >> 1;
    if (row >= (int64_t)b * t * c.n_heads) return;
    const int h = (int)(row % c.n_heads), i = (int)(row / c.n_heads % t), s = (int)(row / c.n_heads / t);
    const bool first = (threadIdx.x & 31) == 0 && h == 0 && (id & 1) == 0;
    const int slot = kv4_slot(c, slots, s, first);
    if (slot < 0) return;
    const int64_t entry = (int64_t)lengths[s] - t + i;
    if (entry < 0 || entry >= c.capacity) {
        if (first && (lengths[s] < 0 || entry >= c.capacity)) atomicOr(c.status, CZG_KV4_BAD_LENGTH);
        return;
    }
    const int64_t at = kv4_row(c, slot, h, (int)entry);
    KvScale *sc = static_cast<KvScale *>(c.scales) + at;
    if (id & 1) {
        quantise_row<T, D>(v + s * vs.b + i * vs.t + h * vs.h, c.v + at * (D / 2), &sc->v_step, &sc->v_lo);
    } else {
        quantise_row<T, D>(k + s * ks.b + i * ks.t + h * ks.h, c.k + at * (D / 2), &sc->k_step, &sc->k_lo);
        if (c.weights && (threadIdx.x & 31) == 0) c.weights[at] = 0.0f;
    }
}

// A thread reads 8 codes of one row and writes their values.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv4_read(czg_kv4 c, const int32_t *__restrict__ slots,
                                                  const int32_t *__restrict__ starts, int b, int count,
                                                  T *__restrict__ k_out, T *__restrict__ v_out) {
    constexpr int P = D / 8;   // threads a row
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = id / P;
    if (row >= (int64_t)b * count * c.n_heads) return;
    const int p = (int)(id % P);
    const int h = (int)(row % c.n_heads), s = (int)(row / c.n_heads / count);
    const int64_t entry = (int64_t)starts[s] + row / c.n_heads % count;
    const int slot = kv4_slot(c, slots, s, p == 0 && h == 0);
    const bool there = slot >= 0 && entry >= 0 && entry < c.capacity;
    if (slot >= 0 && !there && p == 0 && h == 0) atomicOr(c.status, CZG_KV4_BAD_LENGTH);
    const int64_t at = there ? kv4_row(c, slot, h, (int)entry) : 0;
    KvScale sc = {};
    if (there) sc = static_cast<const KvScale *>(c.scales)[at];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        T *out = w ? v_out : k_out;
        if (!out) continue;
        const float step = to_f32(w ? sc.v_step : sc.k_step), lo = to_f32(w ? sc.v_lo : sc.k_lo);
        const uint32_t codes = there ? *reinterpret_cast<const uint32_t *>((w ? c.v : c.k) + at * (D / 2) + 4 * p) : 0u;
        __align__(16) T y[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            y[i] = from_f32<T>(there ? __fmaf_rn(step, (float)(codes >> (4 * i) & 15u), lo) : 0.0f);
        uint4 *dst = reinterpret_cast<uint4 *>(out + row * D + 8 * p);
        const uint4 *src = reinterpret_cast<const uint4 *>(y);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) dst[i] = src[i];
    }
}

// One CTA a sequence and key head, its query rows one after the other: a chunk of 128
// keys at a time, a thread a key for the scores, a thread a dimension for the sums.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_kv4_attend(czg_kv4 c, const T *__restrict__ q, Strides qs,
                                                    const int32_t *__restrict__ slots, const int32_t *__restrict__ lengths,
                                                    int t, int g, int max_len, float scale, T *__restrict__ out, Strides os) {
    __shared__ float sq[D], sp[128], red[4];
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int slot = kv4_slot(c, slots, s, tid == 0 && h == 0);
    const int n = slot < 0 ? 0 : kv4_length(c, lengths, s, min(max_len, c.capacity), tid == 0 && h == 0);
    const int64_t base = kv4_row(c, slot < 0 ? 0 : slot, h, 0);
    const KvScale *sc = static_cast<const KvScale *>(c.scales) + base;
    auto score = [&](int j) {
        float a = 0.0f, z = 0.0f;
        for (int i = 0; i < D / 2; i++) {
            const uint32_t byte = c.k[(base + j) * (D / 2) + i];
            a += sq[2 * i] * (float)(byte & 15u) + sq[2 * i + 1] * (float)(byte >> 4);
            z += sq[2 * i] + sq[2 * i + 1];
        }
        return scale * (to_f32(sc[j].k_step) * a + to_f32(sc[j].k_lo) * z);
    };
    auto reduce = [&](float x, bool is_max) {
        for (int o = 16; o > 0; o >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, x, o);
            x = is_max ? fmaxf(x, y) : x + y;
        }
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = x;
        __syncthreads();
        return is_max ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
    };
    for (int row = 0; row < t * g; row++) {
        const int i = row / g, hq = h * g + row % g;
        __syncthreads();
        if (tid < D) sq[tid] = to_f32(q[s * qs.b + i * qs.t + hq * qs.h + tid]);
        __syncthreads();
        const int seen = max(0, n - (t - 1 - i));
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int j0 = 0; j0 < seen; j0 += 128) {
            const int j = j0 + tid;
            const float x = j < seen ? score(j) : -INFINITY;
            const float m1 = fmaxf(m, reduce(x, true));
            const float p = j < seen ? expf(x - m1) : 0.0f;
            const float f = expf(m - m1);
            l = l * f + reduce(p, false);
            o *= f;
            m = m1;
            sp[tid] = p;
            __syncthreads();
            if (tid < D)
                for (int e = 0; e < min(128, seen - j0); e++) {
                    const uint32_t byte = c.v[(base + j0 + e) * (D / 2) + tid / 2];
                    const float code = (float)(tid & 1 ? byte >> 4 : byte & 15u);
                    o += sp[e] * (to_f32(sc[j0 + e].v_step) * code + to_f32(sc[j0 + e].v_lo));
                }
        }
        if (tid < D) out[s * os.b + i * os.t + hq * os.h + tid] = from_f32<T>(seen > 0 ? o / l : 0.0f);
        if (c.weights)
            for (int j = tid; j < seen; j += 128) c.weights[base + j] += expf(score(j) - m) / l;
    }
    if (c.weights && h == 0 && s == 0) kv4_check_distinct(c, slots, gridDim.y);
}

template <typename T>
int append(const czg_kv4 &c, const void *k, Strides ks, const void *v, Strides vs, const int32_t *slots,
           const int32_t *lengths, int b, int t, cudaStream_t st) {
    const int64_t blocks = ((int64_t)b * t * c.n_heads * 2 + 7) / 8 + 1;
    if (blocks > 0x7FFFFFFF) return ops_fail(CZG_E_LIMIT, "too many rows");
    auto kern = c.head_dim == 64 ? k_kv4_append<T, 64> : k_kv4_append<T, 128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)blocks), 256, 0, st, false, 1, c, static_cast<const T *>(k), ks,
                               static_cast<const T *>(v), vs, slots, lengths, b, t));
}

template <typename T>
int read(const czg_kv4 &c, const int32_t *slots, const int32_t *starts, int b, int count, void *k, void *v, cudaStream_t st) {
    const int64_t blocks = ((int64_t)b * count * c.n_heads * (c.head_dim / 8) + 255) / 256;
    if (blocks > 0x7FFFFFFF) return ops_fail(CZG_E_LIMIT, "too many entries");
    auto kern = c.head_dim == 64 ? k_kv4_read<T, 64> : k_kv4_read<T, 128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)blocks), 256, 0, st, false, 1, c, slots, starts, b, count,
                               static_cast<T *>(k), static_cast<T *>(v)));
}

template <typename T>
int attend(const czg_kv4 &c, const void *q, Strides qs, const int32_t *slots, const int32_t *lengths, int b, int t, int hq,
           int max_len, float scale, void *out, Strides os, cudaStream_t st) {
    auto kern = c.head_dim == 64 ? k_kv4_attend<T, 64> : k_kv4_attend<T, 128>;
    return ops_cuda(ops_launch(kern, dim3((unsigned)c.n_heads, (unsigned)b), 128, 0, st, false, 1, c,
                               static_cast<const T *>(q), qs, slots, lengths, t, hq / c.n_heads, max_len, scale,
                               static_cast<T *>(out), os));
}

}  // namespace

const char *check_kv4(const czg_kv4 *c) {
    if (!c || !c->k || !c->v || !c->scales || !c->status) return "null pointer in the cache";
    if (c->n_slots < 1 || c->n_heads < 1 || c->capacity < 1) return "a cache has at least one slot, head and entry";
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
    (void)cache, (void)b, (void)t, (void)hq, (void)max_len;
    return 0;
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
    if ((int64_t)t * hq > 0x7FFFFFFF) return ops_fail(CZG_E_LIMIT, "too many rows");
    if (ws_bytes < czg_kv4_attend_workspace(cache, b, t, hq, max_len) || !aligned(ws, 16))
        return ops_fail(CZG_E_ARG, "the workspace is too small or not 16-byte aligned");
    const Strides qs{q_sb, q_st, q_sh}, os{o_sb, o_st, o_sh};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CZG_BF16) return attend<__nv_bfloat16>(*cache, q, qs, slots, lengths, b, t, hq, max_len, scale, out, os, st);
    return attend<__half>(*cache, q, qs, slots, lengths, b, t, hq, max_len, scale, out, os, st);
}
