// 4-bit weights x a few rows of 16-bit activations: y[n, m] = sum_g s[m, g] * (sum_{k in g} q[m, k] x[n, k] - z[m, g] sum_{k in g} x[n, k]).
//
// Bound by the weights' bytes (M K / 2 per matrix; a B200 moves ~23 bytes a clock and SM), so everything is laid out to turn
// four bits into a product with few instructions: the codes go to mma.sync m16n8k16 as they are -- one AND (two, and an OR,
// for bf16) makes a register of two operands --, the tensor cores add them up in 32 bits, and scale and zero point are
// applied once per group and row to the 32-bit sums. No weight is ever rounded.
//   fp16: a 4-bit field in the low mantissa bits IS the subnormal number q 2^-24, in the next four bits q 2^-20; the two
//         kinds go to two accumulators and 2^24 / 2^20 joins the scale.
//   bf16: the product q 2^-133 x would leave the 32-bit range, so the field is OR-ed into 128.0 (128 + q, exact) and
//         128 joins the zero point.
//   The sums of x over a group, which the zero point needs, come from one more product with a matrix of ones.
//
// A CTA of eight warps owns 16 or 32 weight rows; its warps take the 128-column blocks of the rows in turn (adjacent warps
// read adjacent 64-byte pieces of a row) and their sums meet in shared memory, in a fixed order. Activations are read straight
// from L1 / L2 in fragment order: there is nothing to stage, no limit on K, and a row index costs nothing.
// Experts: blockIdx.y counts the experts that have rows; a CTA finds its own in the offsets.
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

constexpr int kW4Warps = 8;

__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight consecutive activations of one row; columns at or beyond `valid` read as zero.
__device__ __forceinline__ uint4 load_x8(const uint16_t* at, int valid, bool vec) {
    if (vec && valid >= 8) return __ldg(reinterpret_cast<const uint4*>(at));
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < valid) v[i >> 1] |= (uint32_t)__ldg(at + i) << (16 * (i & 1));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// One 128-column block of the warp's rows in flight: the codes and, packed, the block's scales and zero points of each row.
template <int MT, int GW>
struct W4Slot {
    static constexpr int G = 4 / GW;                               // scale groups of a block
    uint4 w[2 * MT];
    uint32_t s[2 * MT][G == 4 ? 2 : 1], z[2 * MT];
};

// MT: 16-row tiles of a CTA, NTL: 8-column tiles of activation rows per pass, GW: 32-column words per scale group (1, 2, 4).
template <typename T, int MT, int NTL, int GW>
__global__ void __launch_bounds__(kW4Warps * 32, MT * NTL == 4 ? 1 : 2) w4_stream_kernel(const W4Gemm p) {
    constexpr bool kHalf = W4Type<T>::kMagicValue == 1024.f;
    constexpr int G = 4 / GW;
    __shared__ float red[kW4Warps][NTL * 8][MT * 16 + 4];
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

    int expert = 0, first, count;
    if (p.offsets) {                                               // the blockIdx.y-th expert that has rows
        int want = blockIdx.y;
        bool found = false;
        for (int base = 0; base < p.E && !found; base += 32) {
            int f = 0, c = 0;
            if (base + lane < p.E) w4_expert_range(p, base + lane, f, c);
            const uint32_t has = __ballot_sync(0xffffffffu, c > 0);
            const int n = __popc(has);
            if (want < n) {
                expert = base + (int)__fns(has, 0, want + 1);
                found = true;
            }
            want -= n;
        }
        if (!found) return;
    }
    w4_expert_range(p, expert, first, count);

    const int row0 = blockIdx.x * (MT * 16);
    const int nblocks = (p.K + kW4Block - 1) / kW4Block;
    const int full_blocks = p.x_vec ? p.K / kW4Block : 0;          // blocks whose activations are whole 16-byte pieces
    const bool packed = p.groups % G == 0;                         // a block's scales of a row are one aligned load
    const long long base_row = (long long)expert * p.M + row0;
    const uint8_t* wbase = p.plane + base_row * p.row_bytes + t * 16;
    const uint16_t* sbase = p.scales + base_row * p.groups;
    const uint8_t* zbase = p.zeros ? p.zeros + base_row * p.groups : nullptr;
    uint32_t woff[2 * MT], soff[2 * MT];
#pragma unroll
    for (int r = 0; r < 2 * MT; r++) {
        const int m = row0 + r * 8 + g < p.M ? r * 8 + g : p.M - 1 - row0;     // rows behind the matrix repeat the last one and are not stored
        woff[r] = (uint32_t)m * (uint32_t)p.row_bytes;
        soff[r] = (uint32_t)m * (uint32_t)p.groups;
    }
    auto fetch = [&](W4Slot<MT, GW>& slot, int kb) {
        const uint8_t* at = wbase + (long long)kb * kW4BlockBytes;
#pragma unroll
        for (int r = 0; r < 2 * MT; r++) slot.w[r] = ld_stream(at + woff[r]);
        const int grp = kb * G;
#pragma unroll
        for (int r = 0; r < 2 * MT; r++) {
            const uint16_t* sp = sbase + soff[r] + grp;
            const uint8_t* zp = zbase + soff[r] + grp;
            slot.z[r] = 0x08080808u;
            if (G == 1) {
                slot.s[r][0] = __ldg(sp);
                if (zbase) slot.z[r] = __ldg(zp);
            } else if (packed) {
                if (G == 2) {
                    slot.s[r][0] = __ldg(reinterpret_cast<const uint32_t*>(sp));
                    if (zbase) slot.z[r] = __ldg(reinterpret_cast<const uint16_t*>(zp));
                } else {
                    const uint2 v = __ldg(reinterpret_cast<const uint2*>(sp));
                    slot.s[r][0] = v.x;
                    slot.s[r][G == 4 ? 1 : 0] = v.y;
                    if (zbase) slot.z[r] = __ldg(reinterpret_cast<const uint32_t*>(zp));
                }
            } else {                                               // groups behind K: every activation there is zero, any scale will do
#pragma unroll
                for (int q = 0; q < G; q++) {
                    const int o = grp + q < p.groups ? q : p.groups - 1 - grp;
                    const uint32_t v = __ldg(sp + o);
                    if (q & 1) slot.s[r][q >> 1] |= v << 16;
                    else slot.s[r][q >> 1] = v;
                    if (zbase) slot.z[r] = (slot.z[r] & ~(255u << (8 * q))) | (uint32_t)__ldg(zp + o) << (8 * q);
                }
            }
        }
    };

    for (int c0 = 0; c0 < count; c0 += NTL * 8) {
        const uint16_t* xrow[NTL];
#pragma unroll
        for (int j = 0; j < NTL; j++) {
            // columns behind the expert's rows and rows outside x repeat a row that exists; the former are not stored, the
            // latter stored as zeros (a column of the product sees nothing of the others)
            const int n = c0 + j * 8 + g < count ? c0 + j * 8 + g : count - 1;
            const long long src = p.rows ? (long long)p.rows[first + n] : (long long)first + n;
            xrow[j] = static_cast<const uint16_t*>(p.x) + (src >= 0 && src < p.x_rows ? src : 0) * p.x_ld + t * 8;
        }
        float y[MT][NTL][4];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NTL; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) y[i][j][e] = 0.f;

        // One block: products, then the slot is filled with the block after the next.
        auto block = [&](W4Slot<MT, GW>& slot, int kb) {
            uint4 b[4][NTL];
            if (kb < full_blocks) {
#pragma unroll
                for (int word = 0; word < 4; word++)
#pragma unroll
                    for (int j = 0; j < NTL; j++) b[word][j] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + kb * kW4Block + word * 32));
            } else {
#pragma unroll
                for (int word = 0; word < 4; word++) {
                    const int k0 = kb * kW4Block + word * 32;
#pragma unroll
                    for (int j = 0; j < NTL; j++) b[word][j] = load_x8(xrow[j] + k0, p.K - k0 - t * 8, p.x_vec != 0);
                }
            }
            float acc[MT][NTL][4], acc_hi[MT][NTL][4], gs[NTL][4];
#pragma unroll
            for (int word = 0; word < 4; word++) {
                if (word % GW == 0) {
#pragma unroll
                    for (int j = 0; j < NTL; j++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            gs[j][e] = 0.f;
#pragma unroll
                            for (int i = 0; i < MT; i++) acc[i][j][e] = acc_hi[i][j][e] = 0.f;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const uint4 u = slot.w[2 * i], v = slot.w[2 * i + 1];
                    const uint32_t wa = word == 0 ? u.x : (word == 1 ? u.y : (word == 2 ? u.z : u.w));
                    const uint32_t wb = word == 0 ? v.x : (word == 1 ? v.y : (word == 2 ? v.z : v.w));
                    if (kHalf) {
                        const uint32_t ha = wa >> 8, hb = wb >> 8;
#pragma unroll
                        for (int j = 0; j < NTL; j++) {
                            mma16816<T>(acc[i][j], wa & 0x000f000fu, wb & 0x000f000fu, ha & 0x000f000fu, hb & 0x000f000fu, b[word][j].x, b[word][j].z);
                            mma16816<T>(acc_hi[i][j], wa & 0x00f000f0u, wb & 0x00f000f0u, ha & 0x00f000f0u, hb & 0x00f000f0u, b[word][j].y, b[word][j].w);
                        }
                    } else {
                        uint32_t a[4], c[4];
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            a[q] = ((wa >> (4 * q)) & 0x000f000fu) | W4Type<T>::kMagic;
                            c[q] = ((wb >> (4 * q)) & 0x000f000fu) | W4Type<T>::kMagic;
                        }
#pragma unroll
                        for (int j = 0; j < NTL; j++) {
                            mma16816<T>(acc[i][j], a[0], c[0], a[1], c[1], b[word][j].x, b[word][j].y);
                            mma16816<T>(acc_hi[i][j], a[2], c[2], a[3], c[3], b[word][j].z, b[word][j].w);
                        }
                    }
                }
                constexpr uint32_t one = W4Type<T>::kOnes;
#pragma unroll
                for (int j = 0; j < NTL; j++) {
                    mma16816<T>(gs[j], one, one, one, one, b[word][j].x, b[word][j].y);
                    mma16816<T>(gs[j], one, one, one, one, b[word][j].z, b[word][j].w);
                }
                if ((word + 1) % GW == 0) {                        // the end of a scale group
                    const int q = word / GW;
#pragma unroll
                    for (int i = 0; i < MT; i++) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float s = W4Type<T>::to_float((uint16_t)(slot.s[2 * i + h][q >> 1] >> (16 * (q & 1))));
                            float z = (float)((slot.z[2 * i + h] >> (8 * q)) & 15u);
                            if (!kHalf) z += W4Type<T>::kMagicValue;
#pragma unroll
                            for (int j = 0; j < NTL; j++) {
#pragma unroll
                                for (int e = 0; e < 2; e++) {
                                    const int k = 2 * h + e;
                                    const float sum = kHalf ? fmaf(acc[i][j][k], 16777216.f, acc_hi[i][j][k] * 1048576.f) : acc[i][j][k] + acc_hi[i][j][k];
                                    y[i][j][k] = fmaf(s, fmaf(-z, gs[j][e], sum), y[i][j][k]);
                                }
                            }
                        }
                    }
                }
            }
            if (kb + 2 * kW4Warps < nblocks) fetch(slot, kb + 2 * kW4Warps);
        };
        W4Slot<MT, GW> even, odd;
        if (warp < nblocks) fetch(even, warp);
        if (warp + kW4Warps < nblocks) fetch(odd, warp + kW4Warps);
#pragma unroll 1
        for (int kb = warp; kb < nblocks; kb += 2 * kW4Warps) {
            block(even, kb);
            if (kb + kW4Warps < nblocks) block(odd, kb + kW4Warps);
        }
        // the eight warps' sums, in a fixed order
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NTL; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) red[warp][j * 8 + 2 * t + (e & 1)][i * 16 + g + 8 * (e >> 1)] = y[i][j][e];
        __syncthreads();
        for (int o = threadIdx.x; o < NTL * 8 * MT * 16; o += kW4Warps * 32) {
            const int n = o / (MT * 16), m = o % (MT * 16);
            if (c0 + n < count && row0 + m < p.M) {
                float v = 0.f;
#pragma unroll
                for (int q = 0; q < kW4Warps; q++) v += red[q][n][m];
                if (p.rows) {
                    const int src = p.rows[first + c0 + n];
                    if (src < 0 || src >= p.x_rows) v = 0.f;
                }
                static_cast<uint16_t*>(p.out)[(long long)(first + c0 + n) * p.out_ld + row0 + m] = W4Type<T>::from_float(v);
            }
        }
        if (c0 + NTL * 8 < count) __syncthreads();
    }
}

template <typename T, int MT, int NTL>
static int stream_groups(cudaStream_t stream, const W4Gemm& p, dim3 grid) {
    cudaError_t e;
    if (p.group == 32) e = launch_pdl(w4_stream_kernel<T, MT, NTL, 1>, grid, dim3(kW4Warps * 32), stream, p);
    else if (p.group == 64) e = launch_pdl(w4_stream_kernel<T, MT, NTL, 2>, grid, dim3(kW4Warps * 32), stream, p);
    else e = launch_pdl(w4_stream_kernel<T, MT, NTL, 4>, grid, dim3(kW4Warps * 32), stream, p);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

template <typename T>
static int stream_variant(cudaStream_t stream, const W4Gemm& p) {
    const long long experts = p.offsets ? (p.slots < p.E ? p.slots : p.E) : 1;
    const bool wide = (p.M + 31) / 32 * experts >= 2 * sm_count();
    const bool two = p.slots > 8 * experts;
    const dim3 grid((unsigned)((p.M + (wide ? 31 : 15)) / (wide ? 32 : 16)), (unsigned)experts);
    if (wide) return two ? stream_groups<T, 2, 2>(stream, p, grid) : stream_groups<T, 2, 1>(stream, p, grid);
    return two ? stream_groups<T, 1, 2>(stream, p, grid) : stream_groups<T, 1, 1>(stream, p, grid);
}

int launch_w4_stream(cudaStream_t stream, const W4Gemm& p, int dtype) {
    return dtype == BGEMM_DT_F16 ? stream_variant<__half>(stream, p) : stream_variant<__nv_bfloat16>(stream, p);
}

}  // namespace bgemm
