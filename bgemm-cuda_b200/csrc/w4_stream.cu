// 4-bit weights x a few rows of 16-bit activations: y[n, m] = sum_g s[m, g] * (sum_{k in g} q[m, k] x[n, k] - z[m, g] sum_{k in g} x[n, k]).
//
// Bound by the weights' bytes (M K / 2 per matrix; a B200 moves ~23 bytes a clock and SM), so everything is laid out to turn
// four bits into a product with few instructions: the codes go to mma.sync m16n8k16 as they are -- one AND (two, and an OR,
// for bf16) makes a register of two operands --, the tensor cores add them up in 32 bits, and scale and zero point are
// applied once per group and row to the 32-bit sums. No weight is ever rounded.
//   fp16: a 4-bit field in the low mantissa bits IS the subnormal number q 2^-24, in the next four bits q 2^-20; the two
//         kinds go to two accumulators and 2^24 / 2^20 joins the scale.
//   bf16: the product q 2^-133 x would leave the 32-bit range, so the field is OR-ed into 128.0 (128 + q, exact) and
//         128 joins the zero point. (143 |x| over 128 columns must stay below 3.4e38: |x| up to 1e34.)
//   The sums of x over a group, which the zero point needs, come from one more product with a matrix of ones.
//
// A CTA owns 16, 32 or 40 weight rows; its warps take the 128-column blocks of the rows in turn (adjacent warps
// read adjacent 64-byte pieces of a row) and their sums meet in shared memory, in a fixed order. Activations are read straight
// from L1 / L2 in fragment order: there is nothing to stage, no limit on K, and a row index costs nothing.
// blockIdx.y counts the groups of eight rows, of all experts in turn; a CTA finds its own in the offsets.
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

// 16 bytes from global to shared memory, past L1, waited for by groups.
__device__ __forceinline__ void copy16(uint32_t dst_smem, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst_smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

// c = a b (first) or c += a b; `first` is a constant wherever this is inlined.
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
    if (first)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
    if (first)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
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

// Columns of one pass over the scales, which wait in shared memory as pairs (scale, zero point) of the 16-bit type.
constexpr int kW4ChunkBlocks = 64;
constexpr long long kW4MaxOctets = 65535;                                           // of a launch: blockIdx.y
constexpr int kW4Depth = 3;                                                         // blocks of a warp on their way, the one at work included
template <int GW>
__host__ __device__ constexpr int w4_pitch() { return kW4ChunkBlocks * (4 / GW) + 4; }                  // 4 mod 32, 16-byte rows: the eight rows of a read meet eight banks

// Warps an SM is meant to hold. Registers spill at what 24 leave each with five octets of fp16 rows (28672 x 8192 on 8 rows in
// groups of 64: 47 us, 40 with 20 warps; bf16 31.1 and 32.3), with four scale groups a block (in groups of 32: 58 us, 49 with 16; fp16
// 73 and 56), and with two where eight warps share K (8192 x 8192 on 4 rows 14.6 us, 12.4 with 16, on two tiles an SM anyway). In groups of
// 32 most variants still spill with 16 (up to 92 bytes stored and 120 loaded a thread).
template <typename T>
__host__ __device__ constexpr int w4_resident_warps(int W, int H, int GW) { return H > 2 && (GW == 1 || (GW == 2 && W == 8)) ? 16 : (H > 4 && W4Type<T>::kMagicValue == 1024.f ? 20 : 24); }

// W: warps of a CTA (K is divided among them), H: its weight rows in octets (two make a 16-row product, an odd one a product
// whose other half is zero), GW: 32-column words per scale group (1, 2, 4).
template <typename T, int W, int H, int GW>
__global__ void __launch_bounds__(W * 32, w4_resident_warps<T>(W, H, GW) / W) w4_stream_kernel(const W4Gemm p) {
    constexpr bool kHalf = W4Type<T>::kMagicValue == 1024.f;
    constexpr int MT = (H + 1) / 2, G = 4 / GW, PITCH = w4_pitch<GW>(), ROWS = H * 8, STEP_BYTES = ROWS * kW4BlockBytes;
    // Per warp a ring of blocks that every lane fills and reads back itself (no barrier anywhere near it), then the scales
    // [ROWS][PITCH], where the warps' sums meet afterwards.
    extern __shared__ __align__(16) uint32_t smem[];
    uint32_t* s_sz = smem + W * kW4Depth * (STEP_BYTES / 4);
    float(*red)[8][ROWS + 4] = reinterpret_cast<float(*)[8][ROWS + 4]>(s_sz);
    grid_dependency_wait();
    // the shuffle tells the compiler that the warp's number is uniform: block addresses are then computed by the uniform unit
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, t = lane & 3;

    // This CTA's expert and its eight rows: the octet-th group of eight, experts in order.
    const int octet = p.octet0 + (int)blockIdx.y;
    int expert = 0, first = 0, count;
    if (p.offsets) {
        // lane l looks at experts [l q, (l + 1) q): all loads are on their way at once, one prefix sum over the warp
        const int q = (p.E + 31) / 32;
        int mine = 0;
        for (int i = 0; i < q; i++) {
            int f = 0, c = 0;
            if (lane * q + i < p.E) w4_expert_range(p, lane * q + i, f, c);
            mine += (c + 7) / 8;
        }
        int before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += up;
        }
        before -= mine;
        const int want = octet;
        const uint32_t has = __ballot_sync(0xffffffffu, want >= before && want < before + mine);
        if (!has) return;
        int found = 0, skip = 0;
        if (want >= before && want < before + mine) {
            int at = want - before;
            for (int i = 0; i < q; i++) {
                int f = 0, c = 0;
                if (lane * q + i < p.E) w4_expert_range(p, lane * q + i, f, c);
                const int n = (c + 7) / 8;
                if (at >= 0 && at < n) {
                    found = lane * q + i;
                    skip = at * 8;
                }
                at -= n;
            }
        }
        const int owner = __ffs(has) - 1;
        expert = __shfl_sync(0xffffffffu, found, owner);
        skip = __shfl_sync(0xffffffffu, skip, owner);
        w4_expert_range(p, expert, first, count);
        first += skip;
        count -= skip;
    } else {
        first = octet * 8;
        count = (int)p.slots - first;
    }

    const int row0 = blockIdx.x * ROWS;
    const int nblocks = (p.K + kW4Block - 1) / kW4Block;
    const long long base_row = (long long)expert * p.M + row0;
    const uint8_t* wbase = p.plane + base_row * p.row_bytes;
    uint32_t woff[H];
#pragma unroll
    for (int r = 0; r < H; r++) {
        const int m = row0 + r * 8 + g < p.M ? r * 8 + g : p.M - 1 - row0;     // rows behind the matrix repeat the last one and are not stored
        woff[r] = (uint32_t)m * (uint32_t)p.row_bytes + t * 16;
    }
    const uint32_t ring = smem_u32(smem) + warp * (kW4Depth * STEP_BYTES) + lane * 16;
    auto fetch = [&](int slot, int kb) {                           // a group is committed whether there is such a block or not
        if (kb < nblocks) {
            const uint8_t* at = wbase + (long long)kb * kW4BlockBytes;
#pragma unroll
            for (int r = 0; r < H; r++) copy16(ring + slot * STEP_BYTES + r * 512, at + woff[r]);
        }
        copy_commit();
    };
#pragma unroll
    for (int d = 0; d < kW4Depth - 1; d++) fetch(d, warp + d * W);

    // Scales and zero points of the blocks [kb0, kb0 + 64), coalesced along the rows, two groups of a row a lane (one where the rows
    // are not aligned to two). The zero point (bf16: 128 + z) is put together from bits: a conversion costs four times an addition.
    const auto pack_sz = [&](uint32_t s16, uint32_t z) {
        uint32_t v = (W4Type<T>::kMagic & 0xffffu) | (z & 15u);
        if (kHalf) v = (uint32_t)__half_as_ushort(__hsub(__ushort_as_half((uint16_t)v), __ushort_as_half(0x6400)));
        return s16 | v << 16;
    };
    const bool two = ((p.groups & 1) | (reinterpret_cast<uintptr_t>(p.scales) & 3) | (reinterpret_cast<uintptr_t>(p.zeros) & 1)) == 0;
    auto stage_scales = [&](int kb0) {
        const int g0 = kb0 * G, n = p.groups - g0 < kW4ChunkBlocks * G ? p.groups - g0 : kW4ChunkBlocks * G;
        const int want = (n + G - 1) / G * G;                      // groups behind K: every activation there is zero, any scale will do
        constexpr int RW = (ROWS + W - 1) / W;
        if (G > 1 && two) {                                        // (a path more in groups of 128 cost 4096 x 4096 on one row 0.2 us of 5.2)
            for (int i = lane * 2; i < want; i += 64) {
                const int c = i < n ? i : n - 2;
                uint32_t sv[RW], zv[RW];
#pragma unroll
                for (int q = 0; q < RW; q++) {
                    const int r = warp + q * W;
                    const long long at = (base_row + (row0 + r < p.M ? r : p.M - 1 - row0)) * p.groups + g0 + c;
                    sv[q] = __ldg(reinterpret_cast<const uint32_t*>(p.scales + at));
                    zv[q] = p.zeros ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p.zeros + at)) : 0x0808u;
                }
#pragma unroll
                for (int q = 0; q < RW; q++)
                    if (warp + q * W < ROWS)
                        *reinterpret_cast<uint2*>(&s_sz[(warp + q * W) * PITCH + i]) = make_uint2(pack_sz(sv[q] & 0xffffu, zv[q]), pack_sz(sv[q] >> 16, zv[q] >> 8));
            }
            return;
        }
        for (int i = lane; i < want; i += 32) {
            const int c = i < n ? i : n - 1;
            uint32_t sv[RW], zv[RW];
#pragma unroll
            for (int q = 0; q < RW; q++) {
                const int r = warp + q * W;
                const long long at = (base_row + (row0 + r < p.M ? r : p.M - 1 - row0)) * p.groups + g0 + c;
                sv[q] = __ldg(p.scales + at);
                zv[q] = p.zeros ? (uint32_t)__ldg(p.zeros + at) : 8u;
            }
#pragma unroll
            for (int q = 0; q < RW; q++)
                if (warp + q * W < ROWS) s_sz[(warp + q * W) * PITCH + i] = pack_sz(sv[q], zv[q]);
        }
    };

    // columns behind the expert's rows and rows outside x repeat a row that exists; the former are not stored, the latter
    // stored as zeros (a column of the product sees nothing of the others)
    const uint16_t* xrow;
    {
        const int n = g < count ? g : count - 1;
        const long long src = p.rows ? (long long)p.rows[first + n] : (long long)first + n;
        xrow = static_cast<const uint16_t*>(p.x) + (src >= 0 && src < p.x_rows ? src : 0) * p.x_ld + t * 8;
    }
    const int full_blocks = p.x_vec ? p.K / kW4Block : 0;          // blocks whose activations are whole 16-byte pieces
    const uint32_t magic = w4_opaque(W4Type<T>::kMagic);
    constexpr uint32_t one = W4Type<T>::kOnes;
    float y[MT][4];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) y[i][e] = 0.f;

    auto load_b = [&](uint4 (&b)[4], int kb) {
        if (kb < full_blocks) {
#pragma unroll
            for (int word = 0; word < 4; word++) b[word] = __ldg(reinterpret_cast<const uint4*>(xrow + kb * kW4Block + word * 32));
        } else {
#pragma unroll
            for (int word = 0; word < 4; word++) {
                const int k0 = kb * kW4Block + word * 32;
                b[word] = load_x8(xrow + k0, p.K - k0 - t * 8, p.x_vec != 0);
            }
        }
    };
    // The products of one block; sz: its first group of row g in the staged scales.
    auto block = [&](uint32_t at, const uint4 (&b)[4], const uint32_t* sz) {
        uint2 slot[H];                                             // two words of each row at a time: registers are what limits the warps
        float acc[MT][4], acc_hi[MT][4], gs[4];
#pragma unroll
        for (int word = 0; word < 4; word++) {
            const bool start = word % GW == 0;
            if (word % 2 == 0) {
#pragma unroll
                for (int r = 0; r < H; r++) slot[r] = lds8(at + r * 512 + word * 4);
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const bool both = 2 * i + 1 < H;                   // a constant after unrolling
                const uint2 u = slot[2 * i], v = both ? slot[both ? 2 * i + 1 : 0] : make_uint2(0, 0);
                const uint32_t wa = word % 2 ? u.y : u.x, wb = word % 2 ? v.y : v.x;
                if (kHalf) {
                    const uint32_t ha = wa >> 8, hb = wb >> 8;
                    mma16816<T>(acc[i], wa & 0x000f000fu, wb & 0x000f000fu, ha & 0x000f000fu, hb & 0x000f000fu, b[word].x, b[word].z, start);
                    mma16816<T>(acc_hi[i], wa & 0x00f000f0u, wb & 0x00f000f0u, ha & 0x00f000f0u, hb & 0x00f000f0u, b[word].y, b[word].w, start);
                } else {
                    uint32_t a[4], c[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        a[q] = w4_field(wa >> (4 * q), 0x000f000fu, magic);
                        c[q] = both ? w4_field(wb >> (4 * q), 0x000f000fu, magic) : 0u;
                    }
                    mma16816<T>(acc[i], a[0], c[0], a[1], c[1], b[word].x, b[word].y, start);
                    mma16816<T>(acc[i], a[2], c[2], a[3], c[3], b[word].z, b[word].w, false);
                }
            }
            mma16816<T>(gs, one, one, one, one, b[word].x, b[word].y, start);
            mma16816<T>(gs, one, one, one, one, b[word].z, b[word].w, false);
            if ((word + 1) % GW == 0) {                            // the end of a scale group
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (2 * i + h >= H) continue;
                        const float2 f = W4Type<T>::unpack2(sz[(i * 16 + h * 8) * PITCH + word / GW]);       // scale, zero point (+ magic)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int k = 2 * h + e;
                            const float sum = kHalf ? fmaf(acc[i][k], 16777216.f, acc_hi[i][k] * 1048576.f) : acc[i][k];
                            y[i][k] = fmaf(f.x, fmaf(-f.y, gs[e], sum), y[i][k]);
                        }
                    }
                }
            }
        }
    };
    int at = 0;                                                    // ring slot of the next block
    for (int kc = 0; kc < nblocks; kc += kW4ChunkBlocks) {
        if (kc) __syncthreads();                                   // the last pass over this memory is over
        stage_scales(kc);
        __syncthreads();
        const int end = nblocks - kc < kW4ChunkBlocks ? nblocks : kc + kW4ChunkBlocks;
        const uint32_t* sz = s_sz + g * PITCH + warp * G;
        // a warp's first block of this chunk: kW4ChunkBlocks need not be a multiple of W
        int kb = kc + ((warp - kc) % W + W) % W;
        sz += (kb - kc - warp) * G;
#pragma unroll 1
        for (; kb < end; kb += W, sz += W * G) {
            uint4 b[4];
            load_b(b, kb);
            fetch(at ? at - 1 : kW4Depth - 1, kb + (kW4Depth - 1) * W);                    // into the slot read a step ago
            copy_wait<kW4Depth - 1>();
            block(ring + at * STEP_BYTES, b, sz);
            at = at + 1 == kW4Depth ? 0 : at + 1;
        }
    }
    // the warps' sums, in a fixed order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (2 * i + (e >> 1) < H) red[warp][2 * t + (e & 1)][i * 16 + g + 8 * (e >> 1)] = y[i][e];
    __syncthreads();
    for (int o = threadIdx.x; o < 8 * ROWS; o += W * 32) {
        const int n = o / ROWS, m = o % ROWS;
        if (n < count && row0 + m < p.M) {
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < W; q++) v += red[q][n][m];
            if (p.rows) {
                const int src = p.rows[first + n];
                if (src < 0 || src >= p.x_rows) v = 0.f;
            }
            static_cast<uint16_t*>(p.out)[(long long)(first + n) * p.out_ld + row0 + m] = W4Type<T>::from_float(v);
        }
    }
}

template <typename T, int W, int H, int GW>
static int stream_launch(cudaStream_t stream, W4Gemm p, long long octets) {
    constexpr int ROWS = H * 8;
    constexpr int scale_bytes = ROWS * w4_pitch<GW>() * 4, sum_bytes = W * 8 * (ROWS + 4) * 4;
    constexpr int bytes = W * kW4Depth * ROWS * kW4BlockBytes + (scale_bytes > sum_bytes ? scale_bytes : sum_bytes);
    static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(w4_stream_kernel<T, W, H, GW>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return (int)e;
        if (dev < 64) configured[dev] = true;
    }
    // more groups of eight rows than a grid has places for (half a million rows that TMA cannot take) go in several launches
    for (long long o = 0; o < octets; o += kW4MaxOctets) {
        const dim3 grid((unsigned)((p.M + ROWS - 1) / ROWS), (unsigned)(octets - o < kW4MaxOctets ? octets - o : kW4MaxOctets));
        p.octet0 = (int)o;
        const cudaError_t e = launch_pdl_smem(w4_stream_kernel<T, W, H, GW>, grid, dim3(W * 32), (size_t)bytes, stream, p);
        count_launch();
        if (e != cudaSuccess) return (int)e;
    }
    return (int)cudaGetLastError();
}

// Groups of eight rows at most: each expert may end in a partial one.
static long long w4_octets(const W4Gemm& p) {
    if (!p.offsets) return (p.slots + 7) / 8;
    const long long experts = p.slots < p.E ? p.slots : p.E;
    return experts + (p.slots - experts) / 8;
}

template <typename T, int W, int H>
static int stream_groups(cudaStream_t stream, const W4Gemm& p) {
    const long long octets = w4_octets(p);
    if (p.group == 32) return stream_launch<T, W, H, 1>(stream, p, octets);
    if (p.group == 64) return stream_launch<T, W, H, 2>(stream, p, octets);
    return stream_launch<T, W, H, 4>(stream, p, octets);
}

// Warps and rows of a CTA. The launch lasts as long as the SM with the most rows (a tile more than an SM's share is a seventh
// more time at six tiles an SM: 28672 x 8192 on one row took 32.3 us in tiles of 32 rows, 896 of them, and 28.4 in tiles of
// 40, 717), so of 32 and 40 rows the one with the lower maximum is taken. Few tiles: smaller ones, and more warps to share
// their K. Measured against the others (us, one row): 1024 x 4096 12 warps x 16 rows 3.33, 8 x 16 3.44, 4 x 32 5.19; 4096 x
// 4096 8 x 16 5.52, 8 x 32 5.98, 4 x 32 6.90; 8192 x 8192 8 x 32 12.4, 8 x 16 13.6, 4 x 32 13.1; 11008 x 4096 8 x 40 8.98,
// 4 x 40 9.24, 8 x 16 10.3; 14336 x 4096 4 x 40 11.0, 4 x 32 11.2, 8 x 40 13.1.
template <typename T>
static int stream_variant(cudaStream_t stream, const W4Gemm& p) {
    const long long octets = p.offsets ? (p.slots < p.E ? p.slots : p.E) : (p.slots + 7) / 8, sms = sm_count();
    const auto tiles = [&](int rows) { return (p.M + rows - 1) / rows * octets; };
    const auto most_rows = [&](int rows) { return (tiles(rows) + sms - 1) / sms * rows; };
    if (tiles(16) <= sms) return stream_groups<T, 12, 2>(stream, p);
    if (tiles(16) <= 2 * sms) return stream_groups<T, 8, 2>(stream, p);
    const bool forty = most_rows(40) < most_rows(32), shared = 2 * tiles(32) <= 5 * sms;
    if (shared) return forty ? stream_groups<T, 8, 5>(stream, p) : stream_groups<T, 8, 4>(stream, p);
    return forty ? stream_groups<T, 4, 5>(stream, p) : stream_groups<T, 4, 4>(stream, p);
}

int launch_w4_stream(cudaStream_t stream, const W4Gemm& p, int dtype) {
    return dtype == BGEMM_DT_F16 ? stream_variant<__half>(stream, p) : stream_variant<__nv_bfloat16>(stream, p);
}

}  // namespace bgemm
