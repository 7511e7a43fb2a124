// extern "C" surface of the 4-bit weight products and the expert routing (include/bgemm_b200.h): argument checks and launches.
#include <atomic>
#include <cstdlib>

#include "internal.h"
#include "w4.cuh"

using namespace bgemm;

namespace {
constexpr long long kMaxDim = 1LL << 24;
constexpr long long kMaxSlots = 1LL << 30;       // rows of a grouped product, pairs of a routing call
constexpr int kMaxExperts = 1024, kMaxTopK = 32;

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool group_ok(int g) { return g == 32 || g == 64 || g == 128; }
bool is16(int d) { return d == BGEMM_DT_F16 || d == BGEMM_DT_BF16; }

// bgemm_debug_set_w4_kernel: 0 streaming, 1 tensor cores, -1 the rule below; -2 not set, where BGEMM_W4_TENSOR (read once) says the same.
std::atomic<int> g_w4_kernel{-2};
std::atomic<uint64_t> g_w4_calls[2];             // products that each kernel has taken: streaming, tensor cores

int forced_kernel() {
    static const int env = [] {
        const char* e = std::getenv("BGEMM_W4_TENSOR");
        return e ? std::atoi(e) : -1;
    }();
    const int m = g_w4_kernel.load(std::memory_order_relaxed);
    return m == -2 ? env : m;
}

int check_matrix(int64_t M, int64_t K, int group) {
    if (!group_ok(group)) return BGEMM_ERR_ENUM;
    if (M < 1 || K < 1 || M > kMaxDim || K > kMaxDim) return BGEMM_ERR_SHAPE;
    return BGEMM_OK;
}

int check_gemm(const void* plane, int64_t M, int64_t K, int group, const void* scales, const void* x, int64_t x_ld, int64_t x_rows, int dtype,
               int64_t slots, const void* out, int64_t out_ld) {
    if (!plane || !scales || !x || !out) return BGEMM_ERR_NULL;
    if (!is16(dtype)) return BGEMM_ERR_ENUM;
    const int rc = check_matrix(M, K, group);
    if (rc) return rc;
    if (slots < 1 || slots > kMaxSlots || x_rows < 1 || x_rows > kMaxSlots || x_ld < K || out_ld < M || x_ld > (1LL << 40) || out_ld > (1LL << 40))
        return BGEMM_ERR_SHAPE;
    if (!aligned(plane, 16) || !aligned(scales, 2) || !aligned(x, 2) || !aligned(out, 2)) return BGEMM_ERR_ALIGN;
    return BGEMM_OK;
}

W4Gemm problem(const void* plane, int E, int64_t M, int64_t K, int group, const void* scales, const void* zeros, const void* x, int64_t x_ld,
               int64_t x_rows, int64_t slots, void* out, int64_t out_ld) {
    W4Gemm p{};
    p.plane = static_cast<const uint8_t*>(plane);
    p.scales = static_cast<const uint16_t*>(scales);
    p.zeros = static_cast<const uint8_t*>(zeros);
    p.x = x;
    p.out = out;
    p.row_bytes = bgemm_w4_row_bytes(K);
    p.x_ld = x_ld; p.x_rows = x_rows; p.out_ld = out_ld; p.slots = slots;
    p.E = E; p.M = (int)M; p.K = (int)K; p.group = group; p.groups = (int)((K + group - 1) / group);
    p.x_vec = aligned(x, 16) && (x_rows == 1 || x_ld % 8 == 0);
    return p;
}

// Which kernel. The streaming kernel passes over a matrix once for every eight rows that meet it; the tensor-core kernel takes
// any number of rows in one pass, but needs ~9 us to fill and drain and unpacks codes at less than half the memory's rate.
// Measured (us, streaming / tensor cores): 4096 x 4096 on 16 rows 8 / 15, on 24 10 / 15, on 32 11 / 15; 11008 x 4096 on 16 rows
// 14 / 17, on 24 20 / 17; 8192 x 8192 on 12 rows 19 / 22; 28672 x 8192 on 8 rows 31 / 50, on 16 57 / 50; 177 x 1720 on 709 rows 8 / 16; 64 experts of 2048 x 4096 on 8
// rows each 82 / 104, on 9 133 / 104; 8 of them on 93 rows 24 / 19. So: by the bytes of all passes, a short row counting as
// 1536 columns (a CTA's own start and end; 18 experts of 11964 x 128 on 160 rows: 61 / 33). Rows of x off 16-byte
// boundaries cannot be loaded by TMA and stay on the former.
// One pass always streams, whatever the matrix: no weight is rounded on up to eight rows, or eight slots an expert. The counts of
// more experts than one are on the device, so that is by their average, and an expert's last pass is not full: 0.4 of one more.
// (Eight slots on average, unevenly: 64 x 2048 x 4096 107 / 115, 16 x 4096 x 4096 59 / 65, 64 x 1001 x 2056 51 / 47. All 768 slots of 128 experts
// of 2048 x 2048 on one of them: 70 / 22.)
bool on_tensor_cores(const W4Gemm& p) {
    if (!p.x_vec) return false;
    const int forced = forced_kernel();
    if (forced >= 0) return forced != 0;
    const double matrix = (double)p.M * (p.K > 1536 ? (double)p.K : 1536.0) / 2;
    if (!p.offsets || p.E == 1) {
        const long long passes = (p.slots + 7) / 8;
        return passes > 1 && passes * matrix > (passes == 2 ? 80e6 : 45e6);
    }
    const double experts = (double)(p.slots < p.E ? p.slots : p.E), rows = (double)p.slots / experts;
    return rows > 8 && experts * (rows / 8 + 0.4) * matrix > 45e6;
}

int run(cudaStream_t stream, const W4Gemm& p, int dtype, void* workspace, size_t workspace_bytes, int flags) {
    const bool tensor = !(flags & BGEMM_FLAG_EXACT_WEIGHTS) && on_tensor_cores(p);
    g_w4_calls[tensor].fetch_add(1, std::memory_order_relaxed);
    if (!tensor) return launch_w4_stream(stream, p, dtype);
    const size_t need = w4_umma_workspace(p);
    return launch_w4_umma(stream, p, dtype, need && workspace && workspace_bytes >= need ? workspace : nullptr);
}
}  // namespace

extern "C" {

int64_t bgemm_w4_row_bytes(int64_t K) { return K < 1 ? 0 : (K + kW4Block - 1) / kW4Block * kW4BlockBytes; }

int bgemm_w4_quantize(void* stream, const void* src, int src_dtype, int64_t M, int64_t K, int64_t ld, int group, int symmetric, int scale_dtype,
                      void* plane, void* scales, uint8_t* zeros, int64_t batch, int64_t src_batch_stride) {
    if (!src || !plane || !scales || (!symmetric && !zeros)) return BGEMM_ERR_NULL;
    if (src_dtype < BGEMM_DT_F16 || src_dtype > BGEMM_DT_F32 || !is16(scale_dtype)) return BGEMM_ERR_ENUM;
    const int rc = check_matrix(M, K, group);
    if (rc) return rc;
    if (ld < K || ld > (1LL << 40) || batch < 1 || batch > 65535 || (batch > 1 && src_batch_stride < 0)) return BGEMM_ERR_SHAPE;
    if (!aligned(plane, 16) || !aligned(scales, 2) || !aligned(src, src_dtype == BGEMM_DT_F32 ? 4 : 2)) return BGEMM_ERR_ALIGN;
    return launch_w4_quantize((cudaStream_t)stream, src, src_dtype, M, K, ld, group, symmetric ? 1 : 0, scale_dtype, plane, scales,
                              symmetric ? nullptr : zeros, batch, src_batch_stride);
}

int bgemm_w4_dequantize(void* stream, const void* plane, int64_t M, int64_t K, int group, const void* scales, const uint8_t* zeros, int dtype,
                        void* out) {
    if (!plane || !scales || !out) return BGEMM_ERR_NULL;
    if (!is16(dtype)) return BGEMM_ERR_ENUM;
    if (!group_ok(group)) return BGEMM_ERR_ENUM;
    if (M < 1 || K < 1 || M > (1LL << 40) || K > kMaxDim) return BGEMM_ERR_SHAPE;      // M: all rows of a stack of matrices
    if (!aligned(plane, 16) || !aligned(scales, 2) || !aligned(out, 2)) return BGEMM_ERR_ALIGN;
    return launch_w4_dequantize((cudaStream_t)stream, plane, M, K, group, scales, zeros, dtype, out);
}

size_t bgemm_w4a16_workspace_bytes(int64_t E, int64_t M, int64_t K, int64_t slots) {
    if (E < 1 || M < 1 || K < 1 || slots < 1 || E > kMaxExperts || M > kMaxDim || K > kMaxDim || slots > kMaxSlots) return 0;
    W4Gemm p{};
    static const int32_t some = 0;
    p.E = (int)E; p.M = (int)M; p.K = (int)K; p.slots = slots; p.x_vec = 1;
    const size_t dense = E == 1 && on_tensor_cores(p) ? w4_umma_workspace(p) : 0;
    p.offsets = &some;                            // only whether there are any; one matrix may be called either way, with an index too
    const size_t grouped = on_tensor_cores(p) ? w4_umma_workspace(p) : 0;
    return dense > grouped ? dense : grouped;
}

int bgemm_w4a16_gemm(void* stream, const void* plane, int64_t M, int64_t K, int group, const void* scales, const uint8_t* zeros, const void* x,
                     int64_t x_ld, int dtype, int64_t N, void* out, int64_t out_ld, void* workspace, size_t workspace_bytes) {
    return bgemm_w4a16_gemm_ex(stream, plane, M, K, group, scales, zeros, x, x_ld, dtype, N, out, out_ld, workspace, workspace_bytes, 0);
}

int bgemm_w4a16_gemm_ex(void* stream, const void* plane, int64_t M, int64_t K, int group, const void* scales, const uint8_t* zeros, const void* x,
                        int64_t x_ld, int dtype, int64_t N, void* out, int64_t out_ld, void* workspace, size_t workspace_bytes, int flags) {
    if (flags & ~BGEMM_FLAG_EXACT_WEIGHTS) return BGEMM_ERR_ENUM;
    const int rc = check_gemm(plane, M, K, group, scales, x, x_ld, N, dtype, N, out, out_ld);
    if (rc) return rc;
    const W4Gemm p = problem(plane, 1, M, K, group, scales, zeros, x, x_ld, N, N, out, out_ld);
    if (!aligned(workspace, 256)) return BGEMM_ERR_ALIGN;
    return run((cudaStream_t)stream, p, dtype, workspace, workspace_bytes, flags);
}

int bgemm_w4a16_grouped_gemm(void* stream, const void* plane, int64_t E, int64_t M, int64_t K, int group, const void* scales, const uint8_t* zeros,
                             const void* x, int64_t x_rows, int64_t x_ld, int dtype, const int32_t* offsets, const int32_t* rows, int64_t slots,
                             void* out, int64_t out_ld, void* workspace, size_t workspace_bytes) {
    return bgemm_w4a16_grouped_gemm_ex(stream, plane, E, M, K, group, scales, zeros, x, x_rows, x_ld, dtype, offsets, rows, slots, out, out_ld, workspace,
                                       workspace_bytes, 0);
}

int bgemm_w4a16_grouped_gemm_ex(void* stream, const void* plane, int64_t E, int64_t M, int64_t K, int group, const void* scales, const uint8_t* zeros,
                                const void* x, int64_t x_rows, int64_t x_ld, int dtype, const int32_t* offsets, const int32_t* rows, int64_t slots,
                                void* out, int64_t out_ld, void* workspace, size_t workspace_bytes, int flags) {
    if (flags & ~BGEMM_FLAG_EXACT_WEIGHTS) return BGEMM_ERR_ENUM;
    if (!offsets) return BGEMM_ERR_NULL;
    const int rc = check_gemm(plane, M, K, group, scales, x, x_ld, x_rows, dtype, slots, out, out_ld);
    if (rc) return rc;
    if (E < 1 || E > kMaxExperts || (!rows && x_rows < slots)) return BGEMM_ERR_SHAPE;
    if (!aligned(offsets, 4) || !aligned(rows, 4) || !aligned(workspace, 256)) return BGEMM_ERR_ALIGN;
    W4Gemm p = problem(plane, (int)E, M, K, group, scales, zeros, x, x_ld, x_rows, slots, out, out_ld);
    p.offsets = offsets;
    p.rows = rows;
    return run((cudaStream_t)stream, p, dtype, workspace, workspace_bytes, flags);
}

void bgemm_debug_set_w4_kernel(int mode) { g_w4_kernel.store(mode < -1 || mode > 1 ? -2 : mode, std::memory_order_relaxed); }
uint64_t bgemm_debug_w4_calls(int tensor) { return g_w4_calls[tensor ? 1 : 0].load(std::memory_order_relaxed); }

size_t bgemm_moe_route_workspace_bytes(int64_t T, int64_t E) {
    if (T < 1 || E < 1 || E > kMaxExperts || T > kMaxSlots) return 0;
    return moe_route_workspace(T, (int)E);
}

int bgemm_moe_route(void* stream, const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int top_k, int renormalize, float* weights,
                    int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots, void* workspace, size_t workspace_bytes) {
    if (!logits || !weights || !experts || !offsets || !rows || !slots) return BGEMM_ERR_NULL;
    if (dtype < BGEMM_DT_F16 || dtype > BGEMM_DT_F32) return BGEMM_ERR_ENUM;
    if (T < 1 || E < 1 || E > kMaxExperts || ld < E || ld > (1LL << 40) || top_k < 1 || top_k > kMaxTopK || top_k > E || T > kMaxSlots / top_k)
        return BGEMM_ERR_SHAPE;
    if (!aligned(logits, dtype == BGEMM_DT_F32 ? 4 : 2) || !aligned(weights, 4) || !aligned(experts, 4) || !aligned(offsets, 4) || !aligned(rows, 4) ||
        !aligned(slots, 4) || !aligned(workspace, 4))
        return BGEMM_ERR_ALIGN;
    const size_t need = moe_route_workspace(T, (int)E);
    if (need && (!workspace || workspace_bytes < need)) return BGEMM_ERR_WORKSPACE;
    return launch_moe_route((cudaStream_t)stream, logits, dtype, T, (int)E, ld, top_k, renormalize ? 1 : 0, weights, experts, offsets, rows, slots,
                            static_cast<int32_t*>(workspace));
}

int bgemm_moe_combine(void* stream, const void* y, int dtype, int64_t slots_total, int64_t M, int64_t y_ld, const int32_t* slots, const float* weights,
                      int64_t T, int top_k, void* out, int64_t out_ld) {
    if (!y || !slots || !weights || !out) return BGEMM_ERR_NULL;
    if (!is16(dtype)) return BGEMM_ERR_ENUM;
    if (slots_total < 1 || slots_total > kMaxSlots || M < 1 || M > kMaxDim || y_ld < M || out_ld < M || y_ld > (1LL << 40) || out_ld > (1LL << 40) ||
        top_k < 1 || top_k > kMaxTopK || T < 1 || T > kMaxSlots / top_k)
        return BGEMM_ERR_SHAPE;
    if (!aligned(y, 2) || !aligned(out, 2) || !aligned(slots, 4) || !aligned(weights, 4)) return BGEMM_ERR_ALIGN;
    return launch_moe_combine((cudaStream_t)stream, y, dtype, slots_total, M, y_ld, slots, weights, T, top_k, out, out_ld);
}

}  // extern "C"
