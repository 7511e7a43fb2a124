// 4-bit weight format shared by the w4 kernels: element access, conversions, the rounding rules.
//
// A row of K codes is stored in blocks of 128 columns = 64 bytes = sixteen little-endian 32-bit words; word 4 t + w of a
// block holds columns 32 w + 8 t + i (i = 0..7), column i in nibble i / 2 (even i) or 4 + i / 2 (odd i). So
//   * (word >> 4 p) & 0x000f000f is the column pair (2 p, 2 p + 1) as two 16-bit fields: the pair order that both
//     mma.sync fragments and tensor-memory operands want, without a byte permute;
//   * the 16 bytes that thread t of a quad loads hold one word of every 32-column group, so an mma.sync of the quad stays
//     inside one scale group for every group size (32, 64, 128).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/bgemm_b200.h"

namespace bgemm {

constexpr int kW4Block = 128;                    // columns per storage block
constexpr int kW4BlockBytes = 64;

template <typename T>
struct W4Type;
template <>
struct W4Type<__half> {
    using T2 = __half2;
    static constexpr uint32_t kOnes = 0x3C003C00u;
    static constexpr uint32_t kMagic = 0x64006400u;      // 1024 + q: the ulp of [1024, 2048) is 1
    static constexpr float kMagicValue = 1024.f;
    static __device__ __forceinline__ float to_float(uint16_t b) { return __half2float(__ushort_as_half(b)); }
    static __device__ __forceinline__ uint16_t from_float(float v) { return __half_as_ushort(__float2half_rn(v)); }
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};
template <>
struct W4Type<__nv_bfloat16> {
    using T2 = __nv_bfloat162;
    static constexpr uint32_t kOnes = 0x3F803F80u;
    static constexpr uint32_t kMagic = 0x43004300u;      // 128 + q: the ulp of [128, 256) is 1
    static constexpr float kMagicValue = 128.f;
    static __device__ __forceinline__ float to_float(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ uint16_t from_float(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack2(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};

template <int DT>
struct W4OfDtype {
    using type = __half;
};
template <>
struct W4OfDtype<BGEMM_DT_BF16> {
    using type = __nv_bfloat16;
};

// (v & mask) | magic in ONE logic instruction. Written as C the two constants would be two immediates, of which an
// instruction can hold one, and the compiler splits it.
__device__ __forceinline__ uint32_t w4_field(uint32_t v, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(magic));
    return r;
}
// A constant in a register the compiler does not see through.
__device__ __forceinline__ uint32_t w4_opaque(uint32_t v) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Two values (q - z) * s, each rounded ONCE to 16 bits: the magic number turns the 4-bit fields into exact 16-bit floats
// (magic + q), the subtraction of (magic + z) is exact (|q - z| <= 15), the product rounds.
template <typename T>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word_shifted, typename W4Type<T>::T2 magic_zero, typename W4Type<T>::T2 scale,
                                            uint32_t magic = W4Type<T>::kMagic) {
    uint32_t v = w4_field(word_shifted, 0x000f000fu, magic);
    typename W4Type<T>::T2 h = *reinterpret_cast<typename W4Type<T>::T2*>(&v);
    h = __hmul2(__hsub2(h, magic_zero), scale);
    return *reinterpret_cast<uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ typename W4Type<T>::T2 w4_splat(uint32_t bits16) {
    uint32_t v = bits16 | (bits16 << 16);
    return *reinterpret_cast<typename W4Type<T>::T2*>(&v);
}
// 16-bit pattern of magic + z, z in 0..15
template <typename T>
__device__ __forceinline__ uint32_t w4_magic_zero_bits(uint32_t z) { return (W4Type<T>::kMagic & 0xffffu) + (z & 15u); }

// Eight 16-bit values that start on an even address, loaded as what the address allows: one, two or four pieces, or, on an odd
// 4-byte boundary, a half word, three words and a half word. `v` is put in order by octet_values, so that several are on their way at once.
struct Octet {
    uint32_t v[5];
    bool odd;
};
__device__ __forceinline__ void load_octet(Octet& o, const uint16_t* src, int valid) {
    const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15u;
    o.odd = false;
    if (valid < 8) {
        o.v[0] = o.v[1] = o.v[2] = o.v[3] = 0u;
#pragma unroll
        for (int c = 0; c < 7; c++)
            if (c < valid) o.v[c >> 1] |= (uint32_t)__ldg(src + c) << (16 * (c & 1));
    } else if (low == 0) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
        o.v[0] = a.x; o.v[1] = a.y; o.v[2] = a.z; o.v[3] = a.w;
    } else if (low == 8) {
        const uint2 a = __ldg(reinterpret_cast<const uint2*>(src)), b = __ldg(reinterpret_cast<const uint2*>(src) + 1);
        o.v[0] = a.x; o.v[1] = a.y; o.v[2] = b.x; o.v[3] = b.y;
    } else if (low % 4 == 0) {
#pragma unroll
        for (int c = 0; c < 4; c++) o.v[c] = __ldg(reinterpret_cast<const uint32_t*>(src) + c);
    } else {
        o.odd = true;
        o.v[0] = __ldg(src);
#pragma unroll
        for (int c = 0; c < 3; c++) o.v[1 + c] = __ldg(reinterpret_cast<const uint32_t*>(src + 1) + c);
        o.v[4] = __ldg(src + 7);
    }
}
__device__ __forceinline__ void octet_values(const Octet& o, uint32_t (&e)[4]) {
    e[0] = o.odd ? o.v[0] | o.v[1] << 16 : o.v[0];
    e[1] = o.odd ? __funnelshift_r(o.v[1], o.v[2], 16) : o.v[1];
    e[2] = o.odd ? __funnelshift_r(o.v[2], o.v[3], 16) : o.v[2];
    e[3] = o.odd ? __funnelshift_r(o.v[3], o.v[4], 16) : o.v[3];
}
__device__ __forceinline__ void store_octet(uint16_t* dst, int valid, const uint32_t (&e)[4]) {
    const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(dst) & 15u;
    if (valid < 8) {
#pragma unroll
        for (int c = 0; c < 7; c++)
            if (c < valid) dst[c] = (uint16_t)(e[c >> 1] >> (16 * (c & 1)));
    } else if (low == 0) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(e[0], e[1], e[2], e[3]);
    } else if (low == 8) {
        reinterpret_cast<uint2*>(dst)[0] = make_uint2(e[0], e[1]);
        reinterpret_cast<uint2*>(dst)[1] = make_uint2(e[2], e[3]);
    } else if (low % 4 == 0) {
#pragma unroll
        for (int c = 0; c < 4; c++) reinterpret_cast<uint32_t*>(dst)[c] = e[c];
    } else {
        dst[0] = (uint16_t)e[0];
#pragma unroll
        for (int c = 0; c < 3; c++) reinterpret_cast<uint32_t*>(dst + 1)[c] = __funnelshift_r(e[c], e[c + 1], 16);
        dst[7] = (uint16_t)(e[3] >> 16);
    }
}

// ---- launches (w4_quant.cu, w4_stream.cu, moe.cu) -----------------------------------------------------------------
struct W4Gemm {
    const uint8_t* plane;          // [E][M][row_bytes]
    const uint16_t* scales;        // [E][M][groups]
    const uint8_t* zeros;          // [E][M][groups] or null (all 8)
    const void* x;                 // [x_rows][x_ld] 16-bit
    const int32_t* rows;           // [slots] source row of each slot, or null (slot s reads row s)
    const int32_t* offsets;        // [E + 1], or null: one expert, all slots
    void* out;                     // [slots][out_ld] 16-bit
    long long row_bytes, x_ld, x_rows, out_ld, slots;
    int E, M, K, groups, group;
    int x_vec;                     // rows of x start on 16-byte boundaries
    int octet0;                    // streaming kernel: the launch's first group of eight rows
};

// [first, first + count) of expert e; whatever the offsets hold, the range stays inside [0, slots).
__device__ __forceinline__ void w4_expert_range(const W4Gemm& p, int e, int& first, int& count) {
    if (!p.offsets) {
        first = 0;
        count = (int)p.slots;
        return;
    }
    const int n = (int)p.slots;
    int a = p.offsets[e], b = p.offsets[e + 1];
    a = a < 0 ? 0 : (a > n ? n : a);
    b = b < a ? a : (b > n ? n : b);
    first = a;
    count = b - a;
}

int launch_w4_quantize(cudaStream_t stream, const void* src, int dtype, long long M, long long K, long long ld, int group, int symmetric,
                       int scale_dtype, void* plane, void* scales, void* zeros, long long batch, long long batch_stride);
int launch_w4_dequantize(cudaStream_t stream, const void* plane, long long M, long long K, int group, const void* scales, const void* zeros,
                         int dtype, void* out);
int launch_w4_stream(cudaStream_t stream, const W4Gemm& p, int dtype);
size_t w4_umma_workspace(const W4Gemm& p);       // bytes of partial sums the call wants; 0: none
int launch_w4_umma(cudaStream_t stream, const W4Gemm& p, int dtype, void* workspace);
int launch_moe_route(cudaStream_t stream, const void* logits, int dtype, long long T, int E, long long ld, int top_k, int renormalize,
                     float* weights, int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, int32_t* workspace);
size_t moe_route_workspace(long long T, int E);
int launch_moe_combine(cudaStream_t stream, const void* y, int dtype, long long slots_total, long long M, long long y_ld, const int32_t* slots,
                       const float* weights, long long T, int top_k, void* out, long long out_ld);

}  // namespace bgemm
