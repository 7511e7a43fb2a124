// Expert routing: the k largest logits of each token, their softmax weights, the order that puts the rows of one expert
// together, and the weighted sum that takes the experts' results back to the tokens.
//
// Selection: one warp per token, logits in registers as order-preserving 32-bit keys; every choice is one maximum and one
// minimum over the warp (redux): the largest key, then the lowest index that has it. -inf and NaN are never chosen.
// Order: a counting sort by expert that keeps the tokens' order. A CTA takes 32 tokens per "word": an expert's tokens
// are one bit mask per word in shared memory, set with OR -- no order of arrival can change it --, a token's rank inside the CTA
// is a population count. One CTA does a small batch alone; a large one is three launches: selection with a count per CTA and expert,
// prefix sums over the CTAs, placement. Bound by launches up to ~10^4 tokens, by the logits' bytes beyond.
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

constexpr int kRouteWarps = 32;
constexpr int kRouteTokens = 128;                // tokens of a CTA
constexpr int kRouteWords = kRouteTokens / 32;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;

// Order-preserving key of a logit; 0 = never chosen (-inf, NaN). -0 and +0 are the same number.
template <int DT>
__device__ __forceinline__ float logit_at(const void* base, long long at) {
    if (DT == BGEMM_DT_F32) return static_cast<const float*>(base)[at];
    if (DT == BGEMM_DT_F16) return W4Type<__half>::to_float(static_cast<const uint16_t*>(base)[at]);
    return W4Type<__nv_bfloat16>::to_float(static_cast<const uint16_t*>(base)[at]);
}
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key); }

// The choices of one token by one warp. V: logits per lane (expert i * 32 + lane).
template <int DT, int V>
__device__ __forceinline__ void route_token(const void* logits, long long at, int E, int top_k, int renormalize, float* weights, int32_t* experts,
                                            uint32_t* mask /*[E][words]*/, int words, int word, uint32_t bit) {
    const int lane = threadIdx.x & 31;
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = i * 32 + lane;
        key[i] = e < E ? logit_key(logit_at<DT>(logits, at + e)) : 0u;
    }
    uint32_t mine = 0;                           // lane j keeps choice j
    int chosen = -1;
    float total = 0.f, best = 0.f;
    for (int j = 0; j < top_k; j++) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < V; i++) m = max(m, key[i]);
        m = __reduce_max_sync(0xffffffffu, m);
        if (j == 0) {
            best = key_logit(m);
            if (!renormalize && m != 0u) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float v = key_logit(key[i]);
                    total += key[i] == 0u ? 0.f : (key[i] == m ? 1.f : expf(v - best));
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            }
        }
        if (m == 0u) break;
        uint32_t e = 0xffffffffu;
#pragma unroll
        for (int i = V - 1; i >= 0; i--)
            if (key[i] == m) e = i * 32 + lane;
        e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i * 32 + lane == e) key[i] = 0u;
        if (lane == j) {
            mine = m;
            chosen = (int)e;
        }
    }
    // +inf: equal keys have difference 0
    const float w = chosen < 0 ? 0.f : (key_logit(mine) == best ? 1.f : expf(key_logit(mine) - best));
    if (renormalize) {
        total = w;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    if (lane < top_k) {
        weights[lane] = chosen < 0 ? 0.f : __fdiv_rn(w, total);
        experts[lane] = chosen;
    }
    if (chosen >= 0) atomicOr(&mask[chosen * words + word], bit);
}

// Rank of a token among the earlier tokens of the CTA that chose the same expert.
__device__ __forceinline__ int mask_rank(const uint32_t* m, int word, int bit) {
    int r = 0;
    for (int i = 0; i < word; i++) r += __popc(m[i]);
    return r + __popc(m[word] & ((1u << bit) - 1u));
}

// Exclusive prefix sums of n values in shared memory by one warp; returns the sum of all.
__device__ __forceinline__ int warp_prefix(int* v, int n) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
    for (int base = 0; base < n; base += 32) {
        const int x = base + lane < n ? v[base + lane] : 0;
        int s = x;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += up;
        }
        if (base + lane < n) v[base + lane] = carry + s - x;
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    return carry;
}

// LAST: the CTA is the only one, and finishes the order itself. Otherwise `slots` gets the rank inside the CTA and
// counts[e * gridDim.x + CTA] the CTA's number of rows for expert e.
template <int DT, int V, bool LAST>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_select_kernel(const void* __restrict__ logits, long long T, int E, long long ld, int top_k,
                                                                       int renormalize, float* __restrict__ weights, int32_t* __restrict__ experts,
                                                                       int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots,
                                                                       int32_t* __restrict__ counts) {
    __shared__ uint32_t mask[V * 32 * kRouteWords];
    __shared__ int start[V * 32];
    __shared__ int s_total;
    __shared__ int chosen[kRouteTokens * kRouteMaxTopK];
    grid_dependency_wait();
    const int tid = threadIdx.x, warp = tid >> 5, nthreads = blockDim.x;
    for (int i = tid; i < E * kRouteWords; i += nthreads) mask[i] = 0u;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * kRouteTokens;
    const int n = (int)(T - t0 < kRouteTokens ? T - t0 : kRouteTokens);
    for (int i = warp; i < n; i += nthreads >> 5) {
        const long long t = t0 + i;
        route_token<DT, V>(logits, t * ld, E, top_k, renormalize, weights + t * top_k, chosen + i * top_k, mask, kRouteWords, i >> 5, 1u << (i & 31));
    }
    __syncthreads();
    for (int e = tid; e < E; e += nthreads) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < kRouteWords; i++) c += __popc(mask[e * kRouteWords + i]);
        if (LAST) start[e] = c;
        else counts[(long long)e * gridDim.x + blockIdx.x] = c;
    }
    if (LAST) {
        __syncthreads();
        if (warp == 0) {
            const int total = warp_prefix(start, E);
            if (tid == 0) s_total = total;
        }
        __syncthreads();
        for (int e = tid; e <= E; e += nthreads) offsets[e] = e < E ? start[e] : s_total;
        for (int i = s_total + tid; i < n * top_k; i += nthreads) rows[i] = -1;
    }
    for (int i = tid; i < n * top_k; i += nthreads) {
        const int e = chosen[i], token = i / top_k;
        int slot = -1;
        if (e >= 0) {
            slot = mask_rank(mask + e * kRouteWords, token >> 5, token & 31);
            if (LAST) {
                slot += start[e];
                rows[slot] = token;
            }
        }
        experts[t0 * top_k + i] = e;
        slots[t0 * top_k + i] = slot;
    }
}

// One warp per expert: exclusive prefix sums of its counts over the CTAs (in place), the sum in totals[e].
__global__ void __launch_bounds__(256) moe_prefix_kernel(int32_t* __restrict__ counts, int32_t* __restrict__ totals, int E, int blocks) {
    grid_dependency_wait();
    const int e = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (e >= E) return;
    const int total = warp_prefix(counts + (long long)e * blocks, blocks);
    if ((threadIdx.x & 31) == 0) totals[e] = total;
}

__global__ void __launch_bounds__(kRouteWarps * 32) moe_place_kernel(const int32_t* __restrict__ counts, const int32_t* __restrict__ totals,
                                                                      const int32_t* __restrict__ experts, long long T, int E, int top_k,
                                                                      int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    __shared__ int start[kRouteMaxExperts];
    __shared__ int s_total;
    grid_dependency_wait();
    const int tid = threadIdx.x, nthreads = blockDim.x;
    for (int e = tid; e < E; e += nthreads) start[e] = totals[e];
    __syncthreads();
    if (tid < 32) {
        const int total = warp_prefix(start, E);
        if (tid == 0) s_total = total;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = tid; e <= E; e += nthreads) offsets[e] = e < E ? start[e] : s_total;
    const long long pairs = T * top_k;
    for (long long i = s_total + (long long)blockIdx.x * nthreads + tid; i < pairs; i += (long long)gridDim.x * nthreads) rows[i] = -1;
    const long long p0 = (long long)blockIdx.x * kRouteTokens * top_k;
    const long long p1 = p0 + (long long)kRouteTokens * top_k < pairs ? p0 + (long long)kRouteTokens * top_k : pairs;
    for (long long i = p0 + tid; i < p1; i += nthreads) {
        const int e = experts[i];
        if (e >= 0) {
            const int slot = start[e] + counts[(long long)e * gridDim.x + blockIdx.x] + slots[i];
            slots[i] = slot;
            rows[slot] = (int)(i / top_k);
        }
    }
}

static long long route_blocks(long long T) { return (T + kRouteTokens - 1) / kRouteTokens; }

size_t moe_route_workspace(long long T, int E) {
    const long long blocks = route_blocks(T);
    return blocks > 1 ? (size_t)(blocks + 1) * (size_t)E * 4 : 0;
}

template <int DT, int V>
static int route_variant(cudaStream_t stream, const void* logits, long long T, int E, long long ld, int top_k, int renormalize, float* weights,
                         int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, int32_t* ws) {
    const long long blocks = route_blocks(T);
    cudaError_t e;
    if (blocks <= 1) {
        int warps = (int)T;
        warps = warps < 4 ? 4 : (warps > kRouteWarps ? kRouteWarps : warps);
        e = launch_pdl(moe_select_kernel<DT, V, true>, dim3(1), dim3((unsigned)warps * 32), stream, logits, T, E, ld, top_k, renormalize, weights, experts,
                       offsets, rows, slots, (int32_t*)nullptr);
        count_launch();
        return (int)(e != cudaSuccess ? e : cudaGetLastError());
    }
    int32_t* totals = ws + blocks * E;
    e = launch_pdl(moe_select_kernel<DT, V, false>, dim3((unsigned)blocks), dim3(kRouteWarps * 32), stream, logits, T, E, ld, top_k, renormalize, weights,
                   experts, offsets, rows, slots, ws);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(moe_prefix_kernel, dim3((unsigned)((E + 7) / 8)), dim3(256), stream, ws, totals, E, (int)blocks);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(moe_place_kernel, dim3((unsigned)blocks), dim3(kRouteWarps * 32), stream, ws, totals, experts, T, E, top_k, offsets, rows, slots);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

template <int DT>
static int route_dtype(cudaStream_t stream, const void* logits, long long T, int E, long long ld, int top_k, int renormalize, float* weights,
                       int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, int32_t* ws) {
#define BGEMM_ROUTE(V) return route_variant<DT, V>(stream, logits, T, E, ld, top_k, renormalize, weights, experts, offsets, rows, slots, ws)
    if (E <= 64) BGEMM_ROUTE(2);
    if (E <= 128) BGEMM_ROUTE(4);
    if (E <= 256) BGEMM_ROUTE(8);
    if (E <= 512) BGEMM_ROUTE(16);
    BGEMM_ROUTE(32);
#undef BGEMM_ROUTE
}

int launch_moe_route(cudaStream_t stream, const void* logits, int dtype, long long T, int E, long long ld, int top_k, int renormalize,
                     float* weights, int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, int32_t* ws) {
    if (dtype == BGEMM_DT_F16) return route_dtype<BGEMM_DT_F16>(stream, logits, T, E, ld, top_k, renormalize, weights, experts, offsets, rows, slots, ws);
    if (dtype == BGEMM_DT_BF16) return route_dtype<BGEMM_DT_BF16>(stream, logits, T, E, ld, top_k, renormalize, weights, experts, offsets, rows, slots, ws);
    return route_dtype<BGEMM_DT_F32>(stream, logits, T, E, ld, top_k, renormalize, weights, experts, offsets, rows, slots, ws);
}

// out[t, m] = sum_j weights[t, j] * y[slots[t, j], m], j in ascending order in 32 bits, rounded once; a slot outside
// [0, slots_total) adds nothing. A thread owns 8 columns of a token (one 16-byte load per slot, four in flight).
template <typename T>
__global__ void __launch_bounds__(256) moe_combine_kernel(const uint16_t* __restrict__ y, long long slots_total, int M, long long y_ld,
                                                          const int32_t* __restrict__ slots, const float* __restrict__ weights, long long tokens, int top_k,
                                                          uint16_t* __restrict__ out, long long out_ld, int vec) {
    grid_dependency_wait();
    const int chunks = (M + 7) / 8;
    const long long total = tokens * chunks, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const long long t = i / chunks;
        const int m0 = (int)(i - t * chunks) * 8, valid = M - m0;
        float acc[8];
#pragma unroll
        for (int c = 0; c < 8; c++) acc[c] = 0.f;
        for (int j0 = 0; j0 < top_k; j0 += 4) {
            uint4 v[4];
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int s = -1;
                if (j0 + j < top_k) s = __ldg(slots + t * top_k + j0 + j);
                const bool in = s >= 0 && s < slots_total;
                w[j] = in ? __ldg(weights + t * top_k + j0 + j) : 0.f;
                v[j] = make_uint4(0, 0, 0, 0);
                if (in) {
                    const uint16_t* src = y + (long long)s * y_ld + m0;
                    if (vec) {
                        v[j] = __ldg(reinterpret_cast<const uint4*>(src));
                    } else {
                        uint32_t e[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            if (c < valid) e[c >> 1] |= (uint32_t)__ldg(src + c) << (16 * (c & 1));
                        v[j] = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float2 f = W4Type<T>::unpack2(e[c]);
                    acc[2 * c] = fmaf(w[j], f.x, acc[2 * c]);
                    acc[2 * c + 1] = fmaf(w[j], f.y, acc[2 * c + 1]);
                }
            }
        }
        uint16_t* dst = out + t * out_ld + m0;
        if (vec) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(W4Type<T>::pack2(acc[0], acc[1]), W4Type<T>::pack2(acc[2], acc[3]), W4Type<T>::pack2(acc[4], acc[5]),
                                                        W4Type<T>::pack2(acc[6], acc[7]));
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (c < valid) dst[c] = W4Type<T>::from_float(acc[c]);
        }
    }
}

int launch_moe_combine(cudaStream_t stream, const void* y, int dtype, long long slots_total, long long M, long long y_ld, const int32_t* slots,
                       const float* weights, long long T, int top_k, void* out, long long out_ld) {
    const int vec = M % 8 == 0 && y_ld % 8 == 0 && out_ld % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    long long blocks = (T * ((M + 7) / 8) + 255) / 256;
    const long long most = (long long)sm_count() * 64;
    if (blocks > most) blocks = most;
    const cudaError_t e =
        dtype == BGEMM_DT_F16
            ? launch_pdl(moe_combine_kernel<__half>, dim3((unsigned)blocks), dim3(256), stream, static_cast<const uint16_t*>(y), slots_total, (int)M, y_ld,
                         slots, weights, T, top_k, static_cast<uint16_t*>(out), out_ld, vec)
            : launch_pdl(moe_combine_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), stream, static_cast<const uint16_t*>(y), slots_total, (int)M,
                         y_ld, slots, weights, T, top_k, static_cast<uint16_t*>(out), out_ld, vec);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace bgemm
