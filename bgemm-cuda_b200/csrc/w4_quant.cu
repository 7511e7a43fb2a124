// Quantisation of weight matrices to 4 bits with a scale (and zero point) per row and group of columns, and back.
//
//   asymmetric: lo = min(0, min w), hi = max(0, max w), s = r16((hi - lo) * fl(1/15)), z = clamp(rint(-lo / s), 0, 15)
//   symmetric:  s = r16(max |w| * fl(1/7)), z = 8
//   q = clamp(rint(w / s) + z, 0, 15);  s = 0 (an all-zero group): q = z (0 or 8);  value = r16((q - z) * s)
// r16 rounds to the scales' 16-bit type (nearest even), everything else is 32-bit arithmetic, rint rounds ties to even.
//
// Both kernels are bound by memory: 2 (4) bytes in and half a byte out per weight, or the reverse. A lane owns 8 consecutive
// columns -- one 16-byte load and one word of codes -- sixteen lanes a storage block; the group's extremes are exchanged
// with 2 to 4 shuffles.
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

template <int DT>
__device__ __forceinline__ void load8(const void* src, long long at, int valid, bool vec, float (&v)[8]) {
    if (valid >= 8 && vec) {
        if (DT == BGEMM_DT_F32) {
            const float4 a = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(src) + at));
            const float4 b = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(src) + at + 4));
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = DT == BGEMM_DT_F16 ? W4Type<__half>::unpack2(w[i]) : W4Type<__nv_bfloat16>::unpack2(w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float f = 0.f;
        if (i < valid) {
            if (DT == BGEMM_DT_F32) f = static_cast<const float*>(src)[at + i];
            else if (DT == BGEMM_DT_F16) f = W4Type<__half>::to_float(static_cast<const uint16_t*>(src)[at + i]);
            else f = W4Type<__nv_bfloat16>::to_float(static_cast<const uint16_t*>(src)[at + i]);
        }
        v[i] = f;
    }
}

// rint(w / s) for |w / s| < 2^20, without a division per element. r = rint(w * (1 / s)) can only be wrong where w / s lies
// next to a half: e = w - r s is exact there (r s has few bits, and e is a multiple of w's last place no smaller than
// 2^-24 s), so |e| clearly below s / 2 proves r; the rest (ties, mostly) takes the division.
__device__ __forceinline__ float quotient_rint(float w, float s, float inv, float near_half) {
    const float magic = 12582912.f;                                // 1.5 * 2^23: adding it rounds to a whole number, ties to even
    float r = __fsub_rn(__fadd_rn(__fmul_rn(w, inv), magic), magic);
    const float e = __fmaf_rn(-r, s, w);
    if (!(fabsf(e) < near_half)) r = rintf(__fdiv_rn(w, s));
    return r;
}

template <int DT, typename S>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const void* __restrict__ src, long long M, int K, long long ld, int lanes_log2 /*lanes per group: 4, 8, 16*/,
                                                          int symmetric, uint32_t* __restrict__ plane, uint16_t* __restrict__ scales,
                                                          uint8_t* __restrict__ zeros, long long batch_stride, int vec) {
    grid_dependency_wait();
    const int chunks = (K + 127) / 128 * 16;                       // 8-column chunks per row, whole blocks
    const int half_warps = (chunks + 31) / 32;                     // warp steps per row
    const int groups = (K + (8 << lanes_log2) - 1) / (8 << lanes_log2);
    const int lane = threadIdx.x & 31;
    const long long batch = blockIdx.y;
    const long long steps = M * half_warps, nwarps = (long long)gridDim.x * (blockDim.x >> 5);
    const char* base = static_cast<const char*>(src) + batch * batch_stride * (DT == BGEMM_DT_F32 ? 4 : 2);
    plane += batch * M * chunks;
    scales += batch * M * groups;
    if (zeros) zeros += batch * M * groups;
    for (long long st = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); st < steps; st += nwarps) {
        const long long m = st / half_warps;
        const int chunk = (int)(st - m * half_warps) * 32 + lane;
        const int k0 = chunk * 8;
        float v[8];
        load8<DT>(base, m * ld + k0, K - k0, vec != 0, v);
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            lo = fminf(lo, v[i]);
            hi = fmaxf(hi, v[i]);
        }
        for (int d = 1; d < (1 << lanes_log2); d <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        const float range = symmetric ? __fmul_rn(fmaxf(-lo, hi), 1.f / 7.f) : __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f);
        const uint16_t s16 = W4Type<S>::from_float(range);
        const float s = W4Type<S>::to_float(s16);
        float z = symmetric ? 8.f : 0.f, inv = 0.f;
        if (s > 0.f) {
            inv = __fdiv_rn(1.f, s);
            if (!symmetric) z = fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f);
        }
        uint32_t word = 0;
        const float near_half = s * 0.49999f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float r = s > 0.f ? quotient_rint(v[i], s, inv, near_half) : 0.f;
            r = fminf(fmaxf(r + z, 0.f), 15.f);
            word |= (uint32_t)(int)r << (4 * ((i & 1) ? 4 + i / 2 : i / 2));
        }
        if (k0 >= K) word = 0;                                     // the padding of the last block
        if (chunk < chunks) plane[m * chunks + (chunk >> 4) * 16 + (chunk & 3) * 4 + ((chunk >> 2) & 3)] = word;
        const int g = chunk >> lanes_log2;
        if ((chunk & ((1 << lanes_log2) - 1)) == 0 && g < groups) {
            scales[m * groups + g] = s16;
            if (zeros) zeros[m * groups + g] = (uint8_t)(int)z;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint32_t* __restrict__ plane, long long M, int K, int lanes_log2,
                                                            const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros, uint16_t* __restrict__ out,
                                                            int vec) {
    grid_dependency_wait();
    const int chunks = (K + 127) / 128 * 16, used = (K + 7) / 8;
    const int groups = (K + (8 << lanes_log2) - 1) / (8 << lanes_log2);
    const long long total = M * used, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const long long m = i / used;
        const int chunk = (int)(i - m * used), g = chunk >> lanes_log2, k0 = chunk * 8;
        const uint32_t word = __ldcs(plane + m * chunks + (chunk >> 4) * 16 + (chunk & 3) * 4 + ((chunk >> 2) & 3));
        const auto s2 = w4_splat<T>(scales[m * groups + g]);
        const auto mz = w4_splat<T>(w4_magic_zero_bits<T>(zeros ? zeros[m * groups + g] : 8u));
        uint32_t v[4];
#pragma unroll
        for (int p = 0; p < 4; p++) v[p] = w4_pair<T>(word >> (4 * p), mz, s2);
        uint16_t* dst = out + m * (long long)K + k0;
        if (vec) {
            __stcs(reinterpret_cast<uint4*>(dst), make_uint4(v[0], v[1], v[2], v[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k0 + j < K) dst[j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
        }
    }
}

static int lanes_log2_of(int group) { return group == 32 ? 2 : (group == 64 ? 3 : 4); }

template <int DT, typename S>
static int quantize_variant(cudaStream_t stream, const void* src, long long M, long long K, long long ld, int group, int symmetric, void* plane,
                            void* scales, void* zeros, long long batch, long long batch_stride) {
    const size_t size = DT == BGEMM_DT_F32 ? 4 : 2;
    const int vec = reinterpret_cast<uintptr_t>(src) % 16 == 0 && (ld * size) % 16 == 0 && (batch == 1 || (batch_stride * size) % 16 == 0);
    const long long steps = M * (((K + 127) / 128 * 16 + 31) / 32);
    long long blocks = (steps + 7) / 8;
    const long long most = (long long)sm_count() * 16;
    if (blocks > most) blocks = most;
    const cudaError_t e = launch_pdl(w4_quantize_kernel<DT, S>, dim3((unsigned)blocks, (unsigned)batch), dim3(256), stream, src, M, (int)K, ld,
                                     lanes_log2_of(group), symmetric, static_cast<uint32_t*>(plane), static_cast<uint16_t*>(scales),
                                     static_cast<uint8_t*>(zeros), batch_stride, vec);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_w4_quantize(cudaStream_t stream, const void* src, int dtype, long long M, long long K, long long ld, int group, int symmetric,
                       int scale_dtype, void* plane, void* scales, void* zeros, long long batch, long long batch_stride) {
#define BGEMM_W4_Q(DT, S) return quantize_variant<DT, S>(stream, src, M, K, ld, group, symmetric, plane, scales, zeros, batch, batch_stride)
    if (scale_dtype == BGEMM_DT_F16) {
        if (dtype == BGEMM_DT_F16) BGEMM_W4_Q(BGEMM_DT_F16, __half);
        if (dtype == BGEMM_DT_BF16) BGEMM_W4_Q(BGEMM_DT_BF16, __half);
        BGEMM_W4_Q(BGEMM_DT_F32, __half);
    }
    if (dtype == BGEMM_DT_F16) BGEMM_W4_Q(BGEMM_DT_F16, __nv_bfloat16);
    if (dtype == BGEMM_DT_BF16) BGEMM_W4_Q(BGEMM_DT_BF16, __nv_bfloat16);
    BGEMM_W4_Q(BGEMM_DT_F32, __nv_bfloat16);
#undef BGEMM_W4_Q
}

int launch_w4_dequantize(cudaStream_t stream, const void* plane, long long M, long long K, int group, const void* scales, const void* zeros,
                         int dtype, void* out) {
    const int vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    long long blocks = (M * ((K + 7) / 8) + 255) / 256;
    const long long most = (long long)sm_count() * 32;
    if (blocks > most) blocks = most;
    const cudaError_t e =
        dtype == BGEMM_DT_F16
            ? launch_pdl(w4_dequantize_kernel<__half>, dim3((unsigned)blocks), dim3(256), stream, static_cast<const uint32_t*>(plane), M, (int)K,
                         lanes_log2_of(group), static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), static_cast<uint16_t*>(out), vec)
            : launch_pdl(w4_dequantize_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), stream, static_cast<const uint32_t*>(plane), M, (int)K,
                         lanes_log2_of(group), static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), static_cast<uint16_t*>(out), vec);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace bgemm
