// Quantisation of weight matrices to 4 bits with a scale (and zero point) per row and group of columns, and back.
//
//   asymmetric: lo = min(0, min w), hi = max(0, max w), s = r16((hi - lo) * fl(1/15)), z = clamp(rint(-lo / s), 0, 15)
//   symmetric:  s = r16(max |w| * fl(1/7)), z = 8
//   q = clamp(rint(w / s) + z, 0, 15);  s = 0 (an all-zero group): q = z (0 or 8);  value = r16((q - z) * s)
// r16 rounds to the scales' 16-bit type (nearest even), everything else is 32-bit arithmetic, rint rounds ties to even.
//
// Both kernels are bound by memory: 2 (4) bytes in and half a byte out per weight, or the reverse. A lane owns 8 consecutive
// columns -- one 16-byte load and one word of codes --, sixteen lanes a storage block; the group's extremes are exchanged with
// 2 to 4 shuffles. A warp takes 1024 columns of a row at a time, four loads of a lane on their way (one at a time, with a 64-bit
// division for its place, took 450 us for both kernels on 28672 x 8192 bf16, groups of 64; now 130 + 94, 182 at the copy bandwidth; the way there is bound by its arithmetic, the way back by memory).
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

constexpr int kQSteps = 4;                                         // 8-column chunks of a lane in a unit
constexpr int kQUnit = kQSteps * 32;                               // chunks of a unit: 1024 columns

// Eight columns as they are stored. `piece`: bytes of the widest access that the rows' alignment allows (16, 8, 4 or 2).
template <int DT>
struct Raw8 {
    uint32_t r[DT == BGEMM_DT_F32 ? 8 : 4];
};
template <int DT>
__device__ __forceinline__ void load8(Raw8<DT>& v, const void* src, long long at, int valid, int piece) {
    constexpr int N = DT == BGEMM_DT_F32 ? 8 : 4;
    const uint32_t* p = DT == BGEMM_DT_F32 ? static_cast<const uint32_t*>(src) + at : reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(src) + at);
    if (valid >= 8 && piece == 16) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p + i));
            v.r[i] = a.x; v.r[i + 1] = a.y; v.r[i + 2] = a.z; v.r[i + 3] = a.w;
        }
    } else if (valid >= 8 && piece == 8) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p + i));
            v.r[i] = a.x; v.r[i + 1] = a.y;
        }
    } else if (valid >= 8 && piece == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) v.r[i] = __ldcs(p + i);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v.r[i] = 0u;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < valid) {
                if (DT == BGEMM_DT_F32) v.r[DT == BGEMM_DT_F32 ? i : 0] = p[i];
                else v.r[i >> 1] |= (uint32_t)static_cast<const uint16_t*>(src)[at + i] << (16 * (i & 1));
            }
    }
}
template <int DT>
__device__ __forceinline__ void floats8(const Raw8<DT>& v, float (&f)[8]) {
    if (DT == BGEMM_DT_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = __uint_as_float(v.r[DT == BGEMM_DT_F32 ? i : 0]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 p = DT == BGEMM_DT_F16 ? W4Type<__half>::unpack2(v.r[i]) : W4Type<__nv_bfloat16>::unpack2(v.r[i]);
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
}

// The largest -v and the largest v of eight columns and zero, as floats. 16-bit types are compared two at a time.
template <int DT, int LG>
__device__ __forceinline__ float2 extremes8(const Raw8<DT>& v) {
    float down = 0.f, up = 0.f;
    if (DT == BGEMM_DT_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float f = __uint_as_float(v.r[DT == BGEMM_DT_F32 ? i : 0]);
            down = fmaxf(down, -f);
            up = fmaxf(up, f);
        }
#pragma unroll
        for (int d = 1; d < (1 << LG); d <<= 1) {
            down = fmaxf(down, __shfl_xor_sync(0xffffffffu, down, d));
            up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, d));
        }
        return make_float2(down, up);
    }
    using X = typename W4OfDtype<DT>::type;
    using T2 = typename W4Type<X>::T2;
    const auto as2 = [](uint32_t u) { return *reinterpret_cast<const T2*>(&u); };
    const auto bits = [](T2 h) { return *reinterpret_cast<const uint32_t*>(&h); };
    const T2 m = __hmax2(__hmax2(as2(v.r[0]), as2(v.r[1])), __hmax2(as2(v.r[2]), as2(v.r[3])));
    const T2 n = __hmax2(__hmax2(__hneg2(as2(v.r[0])), __hneg2(as2(v.r[1]))), __hmax2(__hneg2(as2(v.r[2])), __hneg2(as2(v.r[3]))));
    T2 both = __hmax2(as2(__byte_perm(bits(n), bits(m), 0x5410)), as2(__byte_perm(bits(n), bits(m), 0x7632)));      // (-lowest, highest)
    both = __hmax2(both, as2(0u));
#pragma unroll
    for (int d = 1; d < (1 << LG); d <<= 1) both = __hmax2(both, as2(__shfl_xor_sync(0xffffffffu, bits(both), d)));
    return W4Type<X>::unpack2(bits(both));
}

__device__ __forceinline__ float pick8(const float (&v)[8], int i) {
    float f = v[0];
#pragma unroll
    for (int j = 1; j < 8; j++) f = j == i ? v[j] : f;
    return f;
}

// w / s where inv + low = 1 / s: inv to a place or two, low its remainder (1 - s inv) inv -- one step of P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990, taken once for eight columns. The sum of the products is off by
// less than 2^-43 before its own rounding: where w / s is exactly a half it is that half, and a quotient of a number of 24 bits by one of 11 that
// is no midpoint of two floats stays 2^-36 away from one, so this is the division's own result. (A test of |w - r s| against s / 2
// that sends only doubtful octets to a division took 259 us on 28672 x 8192 bf16: two in five warps held a tie. Correcting each quotient
// by its own remainder, and packing the codes as floats, 140; now 130.)
__device__ __forceinline__ float quotient(float w, float inv, float low) { return __fmaf_rn(w, inv, __fmul_rn(w, low)); }
// 1.5 * 2^23: adding it rounds to a whole number, ties to even, whose two's complement is then in the low bits
constexpr float kRound = 12582912.f;
constexpr uint32_t kRoundBits = 0x4B400000u;

// LG: log2 of the lanes (8 columns each) of a group. SYM: symmetric codes. Four CTAs an SM (67 registers, three CTAs: 181 us on 28672 x 8192 bf16 with zero points in groups of 128, 159 with four); fp32 has three.
template <int DT, typename S, int LG, bool SYM>
__global__ void __launch_bounds__(256, DT == BGEMM_DT_F32 ? 3 : 4) w4_quantize_kernel(const void* __restrict__ src, long long M, int K, long long ld, uint32_t* __restrict__ plane,
                                                          uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros, long long batch_stride, int piece) {
    grid_dependency_wait();
    const int chunks = (K + 127) / 128 * 16;                       // 8-column chunks per row, whole blocks
    const unsigned units = (unsigned)(chunks + kQUnit - 1) / kQUnit;
    const int groups = (K + (8 << LG) - 1) / (8 << LG);
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int word_of_lane = (lane >> 4) * 16 + (lane & 3) * 4 + ((lane >> 2) & 3);
    const long long batch = blockIdx.y;
    const long long steps = M * units, nwarps = (long long)gridDim.x * 8;
    const char* base = static_cast<const char*>(src) + batch * batch_stride * (DT == BGEMM_DT_F32 ? 4 : 2);
    plane += batch * M * chunks;
    scales += batch * M * groups;
    if (!SYM) zeros += batch * M * groups;
    for (long long st = (long long)blockIdx.x * 8 + warp; st < steps; st += nwarps) {
        // M <= 2^24 rows of at most 2^14 units
        const long long m = units == 1 ? st : (st < (1LL << 32) ? (long long)((unsigned)st / units) : st / units);
        const int unit = (int)(st - m * units) * kQUnit;
        const bool whole = (unit + kQUnit) * 8 <= K && piece == 16;
        Raw8<DT> raw[kQSteps];
        const long long at = m * ld + (unit + lane) * 8;
        if (whole) {
#pragma unroll
            for (int q = 0; q < kQSteps; q++) load8<DT>(raw[q], base, at + q * 256, 8, 16);
        } else {
#pragma unroll
            for (int q = 0; q < kQSteps; q++) load8<DT>(raw[q], base, at + q * 256, K - (unit + lane + q * 32) * 8, piece);
        }
        uint32_t* out = plane + m * chunks + unit + word_of_lane;
        const int g0 = (unit + lane) >> LG;
        uint16_t* s_out = scales + m * groups + g0;
        uint8_t* z_out = SYM ? nullptr : zeros + m * groups + g0;
#pragma unroll
        for (int q = 0; q < kQSteps; q++) {
            const int chunk = unit + lane + q * 32;
            if (chunk - lane >= chunks) break;                     // the same for the whole warp
            const float2 ext = extremes8<DT, LG>(raw[q]);
            const float range = SYM ? __fmul_rn(fmaxf(ext.x, ext.y), 1.f / 7.f) : __fmul_rn(__fadd_rn(ext.y, ext.x), 1.f / 15.f);
            const uint16_t s16 = W4Type<S>::from_float(range);
            const float s = W4Type<S>::to_float(s16);
            float z = SYM ? 8.f : 0.f;
            uint32_t word;
            if (s > 0.f) {
                const float inv = __fdividef(1.f, s), low = __fmul_rn(__fmaf_rn(-s, inv, 1.f), inv);
                float v[8], zr = 0.f, most = 16.f;                        // most: the largest code, before its bound
                uint32_t r[8];                                     // kRoundBits + rint(w / s)
                floats8<DT>(raw[q], v);
                if (s >= 1.2e-38f && s <= 1.0e30f) {
#pragma unroll
                    for (int i = 0; i < 8; i++) r[i] = __float_as_uint(__fadd_rn(quotient(v[i], inv, low), kRound));
                    if (!SYM) {
                        zr = __fsub_rn(__fadd_rn(quotient(ext.x, inv, low), kRound), kRound);
                        most = zr + __fsub_rn(__fadd_rn(quotient(ext.y, inv, low), kRound), kRound);
                    }
                } else {                                           // 1 / s or its remainder is not a normal number
#pragma unroll 1
                    for (int i = 0; i < 9; i++) {
                        const float w = i == 8 ? ext.x : pick8(v, i), whole_number = rintf(__fdiv_rn(w, s));
                        if (i == 8 && !SYM) zr = whole_number;
                        const uint32_t bits = __float_as_uint(__fadd_rn(whole_number, kRound));
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (j == i) r[j] = bits;
                    }
                }
                if (!SYM) z = fminf(zr, 15.f);
                const uint32_t zi = SYM ? 8u : __float_as_uint(__fadd_rn(z, kRound)) - kRoundBits;
                // q = clamp(r + z, 0, 15). Below, the clamp is void (r(lowest) = -zr, symmetric r >= -7) unless s itself was rounded
                // far, as a subnormal number, or z was cut; above, both roundings can add up to 16 (one group in sixty).
                if (s < 6.2e-5f || (!SYM && (zr > 15.f || most > 15.f))) {
#pragma unroll
                    for (int i = 0; i < 8; i++) r[i] = min(max(r[i], kRoundBits - zi), kRoundBits + 15u - zi);
                }
                // sum of q 16^nibble, modulo 2^32: what kRoundBits and z add is taken off once
                word = (zi - kRoundBits) * 0x11111111u;
#pragma unroll
                for (int i = 0; i < 8; i++) word += r[i] << (4 * ((i & 1) * 4 + (i >> 1)));
            } else {
                word = SYM ? 0x88888888u : 0u;
            }
            if (!whole && chunk * 8 >= K) word = 0;                // the padding of the last block
            if (whole || chunk < chunks) out[q * 32] = word;
            if ((lane & ((1 << LG) - 1)) == 0 && (whole || g0 + (q << (5 - LG)) < groups)) {
                s_out[q << (5 - LG)] = s16;
                if (!SYM) z_out[q << (5 - LG)] = (uint8_t)(int)z;
            }
        }
    }
}

// ALIGNED: every octet of the result lies on a 16-byte boundary (others: 4096 x 4097 15 us; value by value 44).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint32_t* __restrict__ plane, long long M, int K, int lanes_log2,
                                                            const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros, uint16_t* __restrict__ out) {
    grid_dependency_wait();
    const int chunks = (K + 127) / 128 * 16, used = (K + 7) / 8;
    const unsigned units = (unsigned)(chunks + kQUnit - 1) / kQUnit;
    const int groups = (K + (8 << lanes_log2) - 1) / (8 << lanes_log2);
    const int lane = threadIdx.x & 31;
    const uint32_t magic = w4_opaque(W4Type<T>::kMagic);
    const long long steps = M * units, nwarps = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long st = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); st < steps; st += nwarps) {
        const long long m = units == 1 ? st : (st < (1LL << 32) ? (long long)((unsigned)st / units) : st / units);
        const int first = (int)(st - m * units) * kQUnit + lane;
        uint32_t word[kQSteps], s16[kQSteps], z8[kQSteps];
#pragma unroll
        for (int q = 0; q < kQSteps; q++) {
            const int chunk = first + q * 32, g = chunk >> lanes_log2;
            word[q] = s16[q] = 0u;
            z8[q] = 8u;
            if (chunk < used) {
                word[q] = __ldcs(plane + m * chunks + (chunk >> 4) * 16 + (chunk & 3) * 4 + ((chunk >> 2) & 3));
                s16[q] = __ldg(scales + m * groups + g);
                if (zeros) z8[q] = __ldg(zeros + m * groups + g);
            }
        }
#pragma unroll
        for (int q = 0; q < kQSteps; q++) {
            const int chunk = first + q * 32, k0 = chunk * 8;
            if (chunk >= used) break;
            const auto s2 = w4_splat<T>(s16[q]);
            const auto mz = w4_splat<T>(w4_magic_zero_bits<T>(z8[q]));
            uint32_t v[4];
#pragma unroll
            for (int p = 0; p < 4; p++) v[p] = w4_pair<T>(word[q] >> (4 * p), mz, s2, magic);
            uint16_t* dst = out + m * (long long)K + k0;
            if (ALIGNED) __stcs(reinterpret_cast<uint4*>(dst), make_uint4(v[0], v[1], v[2], v[3]));
            else store_octet(dst, K - k0, v);
        }
    }
}

// the widest of 16, 8, 4 and 2 bytes that divides an address and its steps, OR-ed together
static int widest_piece(uintptr_t steps) { return steps % 16 == 0 ? 16 : (steps % 8 == 0 ? 8 : (steps % 4 == 0 ? 4 : 2)); }
static int lanes_log2_of(int group) { return group == 32 ? 2 : (group == 64 ? 3 : 4); }
static unsigned quant_blocks(long long M, long long K) {
    const long long steps = M * (((K + 127) / 128 * 16 + kQUnit - 1) / kQUnit), most = (long long)sm_count() * 32;
    const long long blocks = (steps + 7) / 8;
    return (unsigned)(blocks < most ? blocks : most);
}

template <int DT, typename S, int LG, bool SYM>
static int quantize_launch(cudaStream_t stream, const void* src, long long M, long long K, long long ld, void* plane, void* scales, void* zeros, long long batch,
                           long long batch_stride) {
    const size_t size = DT == BGEMM_DT_F32 ? 4 : 2;
    const int piece = widest_piece(reinterpret_cast<uintptr_t>(src) | (uintptr_t)(M > 1 ? ld * size : 0) | (uintptr_t)(batch > 1 ? batch_stride * size : 0));
    const cudaError_t e = launch_pdl(w4_quantize_kernel<DT, S, LG, SYM>, dim3(quant_blocks(M, K), (unsigned)batch), dim3(256), stream, src, M, (int)K, ld,
                                     static_cast<uint32_t*>(plane), static_cast<uint16_t*>(scales), static_cast<uint8_t*>(zeros), batch_stride, piece);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}
template <int DT, typename S>
static int quantize_variant(cudaStream_t stream, const void* src, long long M, long long K, long long ld, int group, int symmetric, void* plane,
                            void* scales, void* zeros, long long batch, long long batch_stride) {
#define BGEMM_W4_LG(LG) \
    return symmetric ? quantize_launch<DT, S, LG, true>(stream, src, M, K, ld, plane, scales, zeros, batch, batch_stride) \
                     : quantize_launch<DT, S, LG, false>(stream, src, M, K, ld, plane, scales, zeros, batch, batch_stride)
    if (group == 32) BGEMM_W4_LG(2);
    if (group == 64) BGEMM_W4_LG(3);
    BGEMM_W4_LG(4);
#undef BGEMM_W4_LG
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
    const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0 && K % 8 == 0;
    const dim3 grid(quant_blocks(M, K));
    const auto kernel = dtype == BGEMM_DT_F16 ? (aligned ? w4_dequantize_kernel<__half, true> : w4_dequantize_kernel<__half, false>)
                                              : (aligned ? w4_dequantize_kernel<__nv_bfloat16, true> : w4_dequantize_kernel<__nv_bfloat16, false>);
    const cudaError_t e = launch_pdl(kernel, grid, dim3(256), stream, static_cast<const uint32_t*>(plane), M, (int)K, lanes_log2_of(group),
                                     static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), static_cast<uint16_t*>(out));
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace bgemm
