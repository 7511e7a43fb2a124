// Expert routing: the k largest logits of each token, their softmax weights, the order that puts the rows of one expert
// together, and the weighted sum that takes the experts' results back to the tokens.
//
// Selection: a warp takes two tokens at a time (their chains of dependent steps hide each other), logits in registers as
// order-preserving keys. A choice is one maximum over the warp (redux): 16-bit logits carry their expert in the low bits of
// the key, so that equal logits are already in order and no key comes twice; 32-bit ones are followed by ballots that find the lowest
// expert with that key. -inf and NaN have key 0 and are never chosen.
// Order: a counting sort by expert that keeps the tokens' order. A CTA's tokens are bits of one mask per expert and 32 tokens in
// shared memory, set with OR -- no order of arrival can change it --; a token's rank inside the CTA is a population count. One CTA does
// up to 128 tokens alone; more take three launches: selection with a count per CTA and expert, prefix sums over the CTAs, placement.
// Bound by launches and the length of the selection's chain (64 x 64, 8 chosen: 6.3 us) and its instructions (16000 x 256: 23.6), not by the logits' bytes.
#include <cuda_runtime.h>

#include <type_traits>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

constexpr int kRouteAlone = 128;                 // tokens one CTA does by itself
constexpr int kRouteTokens = 32;                 // tokens of a CTA otherwise
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;

// Order-preserving key of a logit; 0 = never chosen (-inf, NaN). `f` has had 0 added, which makes one number of -0 and +0. A
// 16-bit logit fills the upper 19 bits of its 32-bit form at most: the expert goes below, the lowest one largest.
template <int DT>
__device__ __forceinline__ uint32_t logit_key(float f, int expert) {
    const uint32_t u = __float_as_uint(f), k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
    if (!(f > -INFINITY)) return 0u;
    return DT == BGEMM_DT_F32 ? k : ((k & ~0x1FFFu) | (uint32_t)(0x1FFF - expert));
}
template <int DT>
__device__ __forceinline__ float key_logit(uint32_t key) {
    const uint32_t u = (key & 0x80000000u) ? (key ^ 0x80000000u) : ~key;
    return __uint_as_float(DT == BGEMM_DT_F32 ? u : (u & ~0x1FFFu));
}

// The choices of P tokens (row0, row0 + step, ..; those below `rows`) by one warp. V: logits per lane (expert i * 32 + lane).
// weights and chosen have top_k entries a token.
template <int DT, int V, int P>
__device__ __forceinline__ void route_tokens(const void* logits, long long ld, long long token0, int row0, int step, int rows, int E, int top_k, int renormalize,
                                             float* weights, int32_t* chosen, uint32_t* mask /*[E][words]*/, int words) {
    const int lane = threadIdx.x & 31;
    uint32_t key[P][V];
    float value[P][V];                           // for the sum over all experts
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int row = row0 + p * step;
        const long long at = (token0 + (row < rows ? row : row0)) * ld;
#pragma unroll
        for (int i = 0; i < V; i++) {            // all loads first: a key's conditions must not hold the next load up
            const int e = i * 32 + lane < E ? i * 32 + lane : E - 1;
            key[p][i] = DT == BGEMM_DT_F32 ? __ldg(static_cast<const uint32_t*>(logits) + at + e) : (uint32_t)__ldg(static_cast<const uint16_t*>(logits) + at + e);
        }
    }
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float f = (DT == BGEMM_DT_F32 ? __uint_as_float(key[p][i]) : W4Type<typename W4OfDtype<DT>::type>::to_float((uint16_t)key[p][i])) + 0.f;
            const bool in = i * 32 + lane < E;
            key[p][i] = in ? logit_key<DT>(f, i * 32 + lane) : 0u;
            value[p][i] = key[p][i] ? f : -INFINITY;
        }
    // 16-bit logits: every lane keeps its keys in descending order (they are all different, 0 aside), so a choice only looks at
    // the heads and moves one lane's row up
    constexpr bool SORTED = DT != BGEMM_DT_F32;
    if (SORTED) {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int k = 2; k <= V; k *= 2)      // bitonic
#pragma unroll
                for (int d = k / 2; d > 0; d /= 2)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const int o = i ^ d;
                        if (o > i) {
                            const uint32_t hi = max(key[p][i], key[p][o]), lo = min(key[p][i], key[p][o]);
                            const bool down = (i & k) == 0;
                            key[p][i] = down ? hi : lo;
                            key[p][o] = down ? lo : hi;
                        }
                    }
    }
    uint32_t mine[P];                            // lane j keeps choice j
    int pick[P];
    float total[P], best[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        mine[p] = 0u;
        pick[p] = -1;
        total[p] = best[p] = 0.f;
    }
    for (int j = 0; j < top_k; j++) {
        uint32_t top[P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            uint32_t m = key[p][0];
            if (!SORTED) {
#pragma unroll
                for (int i = 1; i < V; i++) m = max(m, key[p][i]);
            }
            top[p] = m;
        }
#pragma unroll
        for (int p = 0; p < P; p++) top[p] = __reduce_max_sync(0xffffffffu, top[p]);
        if (j == 0) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                best[p] = key_logit<DT>(top[p]);
                if (!renormalize && top[p] != 0u) {
                    if (best[p] < INFINITY) {
#pragma unroll
                        for (int i = 0; i < V; i++) total[p] += expf(value[p][i] - best[p]);      // the function of the numerators
                    } else {                     // +inf: equal logits differ by 0
#pragma unroll
                        for (int i = 0; i < V; i++) total[p] += value[p][i] == best[p] ? 1.f : 0.f;
                    }
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) total[p] += __shfl_xor_sync(0xffffffffu, total[p], d);
                }
            }
        }
#pragma unroll
        for (int p = 0; p < P; p++) {
            int e;
            if (DT == BGEMM_DT_F32) {
                e = -1;
#pragma unroll
                for (int i = V - 1; i >= 0; i--) {
                    const uint32_t has = __ballot_sync(0xffffffffu, key[p][i] == top[p]);
                    if (has) e = i * 32 + __ffs(has) - 1;
                }
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (i * 32 + lane == e) key[p][i] = 0u;
            } else {
                e = 0x1FFF - (int)(top[p] & 0x1FFFu);
                const bool mine_goes = key[p][0] == top[p];
#pragma unroll
                for (int i = 0; i < V; i++) key[p][i] = mine_goes ? (i + 1 < V ? key[p][i + 1 < V ? i + 1 : 0] : 0u) : key[p][i];
            }
            if (lane == j && top[p] != 0u) {
                mine[p] = top[p];
                pick[p] = e;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int row = row0 + p * step;
        const float v = key_logit<DT>(mine[p]);
        const float w = pick[p] < 0 ? 0.f : (v == best[p] ? 1.f : expf(v - best[p]));
        if (renormalize) {
            total[p] = w;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) total[p] += __shfl_xor_sync(0xffffffffu, total[p], d);
        }
        if (lane < top_k && row < rows) {
            weights[(token0 + row) * top_k + lane] = pick[p] < 0 ? 0.f : __fdiv_rn(w, total[p]);
            chosen[row * top_k + lane] = pick[p];
        }
        if (pick[p] >= 0 && row < rows) atomicOr(&mask[pick[p] * words + (row >> 5)], 1u << (row & 31));
    }
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

// ALONE: the CTA is the only one, and finishes the order itself. Otherwise `slots` gets the rank inside the CTA and
// counts[e * gridDim.x + CTA] the CTA's number of rows for expert e.
template <int DT, int V, bool ALONE>
__global__ void __launch_bounds__(ALONE ? 1024 : 512) moe_select_kernel(const void* __restrict__ logits, long long T, int E, long long ld, int top_k,
                                                                         int renormalize, float* __restrict__ weights, int32_t* __restrict__ experts,
                                                                         int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots,
                                                                         int32_t* __restrict__ counts) {
    constexpr int TOKENS = ALONE ? kRouteAlone : kRouteTokens, WORDS = TOKENS / 32, P = V <= 8 ? 2 : 1;
    __shared__ uint32_t mask[V * 32 * WORDS];
    __shared__ int start[V * 32];
    __shared__ int s_total;
    __shared__ int chosen[TOKENS * kRouteMaxTopK];
    grid_launch_dependents();                    // the next kernel waits for this one's end, not for its launch
    grid_dependency_wait();
    const int tid = threadIdx.x, warp = tid >> 5, nthreads = blockDim.x, warps = nthreads >> 5;
    for (int i = tid; i < E * WORDS; i += nthreads) mask[i] = 0u;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * TOKENS;
    const int n = (int)(T - t0 < TOKENS ? T - t0 : TOKENS);
    for (int i = warp; i < n; i += warps * P)
        route_tokens<DT, V, P>(logits, ld, t0, i, warps, n, E, top_k, renormalize, weights, chosen, mask, WORDS);
    __syncthreads();
    for (int e = tid; e < E; e += nthreads) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < WORDS; i++) c += __popc(mask[e * WORDS + i]);
        if (ALONE) start[e] = c;
        else counts[(long long)e * gridDim.x + blockIdx.x] = c;
    }
    if (ALONE) {
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
            slot = mask_rank(mask + e * WORDS, token >> 5, token & 31);
            if (ALONE) {
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
    grid_launch_dependents();
    grid_dependency_wait();
    const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (e >= E) return;
    int32_t* row = counts + (long long)e * blocks;
    int carry = 0;
    for (int base = 0; base < blocks; base += 256) {                // eight loads of a lane on their way
        int x[8];
#pragma unroll
        for (int q = 0; q < 8; q++) x[q] = base + q * 32 + lane < blocks ? row[base + q * 32 + lane] : 0;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            int s = x[q];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += up;
            }
            if (base + q * 32 + lane < blocks) row[base + q * 32 + lane] = carry + s - x[q];
            carry += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    if (lane == 0) totals[e] = carry;
}

__global__ void __launch_bounds__(256) moe_place_kernel(const int32_t* __restrict__ counts, const int32_t* __restrict__ totals,
                                                                      const int32_t* __restrict__ experts, long long T, int E, int top_k,
                                                                      int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    constexpr int Q = kRouteMaxExperts / 256;
    __shared__ int start[kRouteMaxExperts];
    __shared__ int warp_sum[8];
    grid_dependency_wait();
    const int tid = threadIdx.x, nthreads = blockDim.x, lane = tid & 31, warp = tid >> 5;
    // exclusive prefix sums of the experts' totals: four experts a thread
    int x[Q], mine = 0;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        x[q] = tid * Q + q < E ? totals[tid * Q + q] : 0;
        mine += x[q];
    }
    int s = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += up;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int s_total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        if (w < warp) before += warp_sum[w];
        s_total += warp_sum[w];
    }
    before += s - mine;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        start[tid * Q + q] = before;
        before += x[q];
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

size_t moe_route_workspace(long long T, int E) { return T > kRouteAlone ? (size_t)(route_blocks(T) + 1) * (size_t)E * 4 : 0; }

template <int DT, int V>
static int route_variant(cudaStream_t stream, const void* logits, long long T, int E, long long ld, int top_k, int renormalize, float* weights,
                         int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, int32_t* ws) {
    cudaError_t e;
    if (T <= kRouteAlone) {
        int warps = V <= 8 ? (int)(T + 1) / 2 : (int)T;
        warps = warps < 4 ? 4 : (warps > 32 ? 32 : warps);
        e = launch_pdl(moe_select_kernel<DT, V, true>, dim3(1), dim3((unsigned)warps * 32), stream, logits, T, E, ld, top_k, renormalize, weights, experts,
                       offsets, rows, slots, (int32_t*)nullptr);
        count_launch();
        return (int)(e != cudaSuccess ? e : cudaGetLastError());
    }
    const long long blocks = route_blocks(T);
    int32_t* totals = ws + blocks * E;
    e = launch_pdl(moe_select_kernel<DT, V, false>, dim3((unsigned)blocks), dim3(512), stream, logits, T, E, ld, top_k, renormalize, weights, experts, offsets,
                   rows, slots, ws);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(moe_prefix_kernel, dim3((unsigned)((E + 7) / 8)), dim3(256), stream, ws, totals, E, (int)blocks);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(moe_place_kernel, dim3((unsigned)blocks), dim3(256), stream, ws, totals, experts, T, E, top_k, offsets, rows, slots);
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
// [0, slots_total) adds nothing. A thread owns 8 columns of a token, the loads of four slots in flight. ALIGNED: whole octets on 16-byte
// boundaries everywhere (8000 x 4104, 4 slots: 55.3 us; 8000 x 4097 by octets of any alignment 78.5, value by value 107).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) moe_combine_kernel(const uint16_t* __restrict__ y, long long slots_total, int M, long long y_ld,
                                                          const int32_t* __restrict__ slots, const float* __restrict__ weights, long long tokens, int top_k,
                                                          uint16_t* __restrict__ out, long long out_ld) {
    grid_dependency_wait();
    const int chunks = (M + 7) / 8;
    const long long total = tokens * chunks, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const long long t = total < (1LL << 32) ? (long long)((unsigned)i / (unsigned)chunks) : i / chunks;
        const int m0 = (int)(i - t * chunks) * 8, valid = M - m0;
        float acc[8];
#pragma unroll
        for (int c = 0; c < 8; c++) acc[c] = 0.f;
        for (int j0 = 0; j0 < top_k; j0 += 4) {
            std::conditional_t<ALIGNED, uint4, Octet> v[4];
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int s = -1;
                if (j0 + j < top_k) s = __ldg(slots + t * top_k + j0 + j);
                const bool in = s >= 0 && s < slots_total;
                w[j] = in ? __ldg(weights + t * top_k + j0 + j) : 0.f;
                const uint16_t* src = y + (long long)s * y_ld + m0;
                if constexpr (ALIGNED) {
                    v[j] = make_uint4(0, 0, 0, 0);
                    if (in) v[j] = __ldg(reinterpret_cast<const uint4*>(src));
                } else {
                    v[j] = Octet{};
                    if (in) load_octet(v[j], src, valid);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t e[4];
                if constexpr (ALIGNED) {
                    e[0] = v[j].x; e[1] = v[j].y; e[2] = v[j].z; e[3] = v[j].w;
                } else {
                    octet_values(v[j], e);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float2 f = W4Type<T>::unpack2(e[c]);
                    acc[2 * c] = fmaf(w[j], f.x, acc[2 * c]);
                    acc[2 * c + 1] = fmaf(w[j], f.y, acc[2 * c + 1]);
                }
            }
        }
        uint16_t* dst = out + t * out_ld + m0;
        const uint32_t e[4] = {W4Type<T>::pack2(acc[0], acc[1]), W4Type<T>::pack2(acc[2], acc[3]), W4Type<T>::pack2(acc[4], acc[5]), W4Type<T>::pack2(acc[6], acc[7])};
        if (ALIGNED) *reinterpret_cast<uint4*>(dst) = make_uint4(e[0], e[1], e[2], e[3]);
        else store_octet(dst, valid, e);
    }
}

int launch_moe_combine(cudaStream_t stream, const void* y, int dtype, long long slots_total, long long M, long long y_ld, const int32_t* slots,
                       const float* weights, long long T, int top_k, void* out, long long out_ld) {
    const bool aligned = M % 8 == 0 && y_ld % 8 == 0 && out_ld % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    long long blocks = (T * ((M + 7) / 8) + 255) / 256;
    const long long most = (long long)sm_count() * 64;
    if (blocks > most) blocks = most;
    const auto kernel = dtype == BGEMM_DT_F16 ? (aligned ? moe_combine_kernel<__half, true> : moe_combine_kernel<__half, false>)
                                              : (aligned ? moe_combine_kernel<__nv_bfloat16, true> : moe_combine_kernel<__nv_bfloat16, false>);
    const cudaError_t e = launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), stream, static_cast<const uint16_t*>(y), slots_total, (int)M, y_ld, slots, weights, T,
                                     top_k, static_cast<uint16_t*>(out), out_ld);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace bgemm
