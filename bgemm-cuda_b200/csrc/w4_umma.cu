// 4-bit weights x many rows of 16-bit activations on the tensor cores, dense or grouped by expert with ragged row counts:
// y[n, m] = sum_k x[n, k] r16((q[m, k] - z) s), 32-bit accumulators in tensor memory.
//
// CTA pairs (tcgen05 cta_group::2) walk over tiles of 256 weight rows x up to 256 activation rows. Each CTA streams ITS 128
// weight rows as packed codes (TMA, 64 bytes of a row per 128 columns), unpacks them in registers and writes them to its tensor
// memory as the A operand (".ts" form); it loads half of the activation rows (TMA, 128-byte swizzle; row by row with
// tile::gather4 where an index names the rows), and one thread of the even CTA issues the products for both SMs. Why pairs:
// a weight is 4 bits on its way to the SM and 16 inside, so the activations are what loads the L2 -> SM path; a pair needs
// half a tile's activations per SM (32 bytes a clock at full tensor rate, 64 without the pair: all an SM can take in).
// Why the weights are the M side: a tile's width in activation rows is then free (any multiple of 32), which is what ragged
// groups need: an expert with 40 rows costs 64 columns of tensor work, not 128 or 256.
//
// Work: tiles are (activation tile, weight tile) pairs over all experts; every CTA derives the same list from the offsets, so
// the host never reads them. The tile width is chosen on the device too, from the counts: the width whose number of rounds
// over the pairs, times the time of a tile (tensor work or the weights' bytes, whichever is longer), is least.
// Few tiles (splits > 1): K is divided, the partial sums go to a workspace as 32-bit values and a second kernel adds them up
// in a fixed order.
//
// The weight is rounded once to 16 bits, because the scale changes along K and the accumulator cannot: (q - z) s has up to
// 15 (bf16: 12) significant bits, r16 keeps 11 (8). Sums are 32-bit. Callers that want no weight rounded say so and get the streaming kernel.
//
// Tensor memory: 256 accumulator columns as two halves of 128 (a tile of up to 128 rows takes one of them, so its epilogue
// runs under the next tile's products; a wider one takes both) + 4 operand stages of 64 columns (128 weight columns each).
//   warps 0-15   unpack: set s = warps 4 s .. takes every fourth 128-column block
//   warps 16-23  epilogue: accumulator -> 16-bit staging tile -> 16-byte stores
//   warp 24      tensor-memory allocation; one lane of the even CTA issues the UMMAs
//   warp 25      one lane streams the codes
//   warps 26-27  activations, every second operand stage each: boxes of 16 to 128 rows, or four rows at a time (gather4)
#include <cuda.h>
#include <cuda_runtime.h>

#include "internal.h"
#include "ptx.cuh"
#include "w4.cuh"

namespace bgemm {

constexpr int kUThreads = 896;
constexpr int kUSets = 4;
constexpr int kUWarpEpi = 16, kUWarpMma = 24, kUWarpW = 25, kUWarpB = 26;
constexpr int kUMaxExperts = 1024;
constexpr long long kUCopyDrainClocks = 4000000;  // ~2 ms: far beyond any TMA copy in flight

struct UCfg {
    static constexpr int NT = 256;                          // widest tile
    // An operand stage is 128 weight columns: 64 columns of tensor memory and 256 bytes of each activation row (two swizzled
    // tiles of 128). Unpack set s fills stage s. (Stages of 64 columns, eight of them, measured 505 against 400 ns per 128
    // columns of a 32-row tile: a stage costs its issuer ~330 clocks before the first product.)
    static constexpr int STAGES = 4, A_STAGE_COLS = 64, A_COL0 = NT;
    static constexpr int B_SUB_BYTES = 128 * 128;           // 64 columns of this CTA's half of the activation rows
    static constexpr int B_STAGE_BYTES = 2 * B_SUB_BYTES;
    static constexpr int W_STAGES = 8, W_STAGE_BYTES = 128 * kW4BlockBytes;
    static constexpr int PITCH = 272;                       // bytes of a staged result column: 128 x 2 + 16
    static constexpr int STAGED = 32;                       // result columns staged at a time, per epilogue half
    static constexpr int STAGING_BYTES = 2 * STAGED * PITCH;
    // w_full/w_empty, full/empty, d_full[2], d_empty[2], drained
    static constexpr int NBARS = 2 * W_STAGES + 2 * STAGES + 5;
    static constexpr int MISC_BYTES = 512 + 2 * 4 * (kUMaxExperts + 8);
    static constexpr int SMEM_BYTES = STAGES * B_STAGE_BYTES + W_STAGES * W_STAGE_BYTES + STAGING_BYTES + MISC_BYTES + 1024;
    // A stage and its barriers always meet the same set (and the same producer warp): a set that waits for a phase by its
    // parity has then seen the phase before it complete. With six code stages and four sets it had not, and a code copy that was
    // overtaken by a later one let a set read a stage that was still being filled.
    static_assert(W_STAGES % kUSets == 0 && STAGES % 2 == 0, "stage -> unpack set / producer must stay fixed");
    static_assert(STAGES == kUSets, "an operand stage always meets the same unpack set");
    static_assert(NBARS * 8 <= 320, "barrier area");
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
    static_assert(SMEM_BYTES > 114 * 1024, "one CTA per SM: the tensor-memory allocation never waits");
};

struct W4UmmaParams {
    W4Gemm g;
    float* partial;              // [splits][slots][M] or null
    int* status;
    long long wait_budget;
    int splits;
    int mpairs;                  // tiles of 256 weight rows
    int test_skip_kblock;        // bgemm_debug_set_wait_test; -1: none
};

// kind::f16, both operands K-major, 32-bit accumulator, M = 256 over the pair.
__host__ __device__ constexpr uint32_t umma_idesc_16(bool bf16, int n) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ts_pair(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrival on a barrier of either CTA of the pair, without a release at cluster scope: what is handed over is tensor memory,
// whose accesses tcgen05.wait::st / ::ld have completed before. A cluster-scope release waits for every outstanding access
// of the thread, the prefetched scales among them: ~2300 clocks for each arrival (a set unpacked a block in 5600 clocks instead of 3300).
__device__ __forceinline__ void arrive_pair(uint32_t bar_cluster) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
        "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
// Four rows of a matrix whose tensor map has boxes of one row, to consecutive rows of a swizzled tile.
__device__ __forceinline__ void tma_gather4_pair(uint32_t dst_smem, const CUtensorMap* map, int c0, const int (&row)[4], uint32_t bar_cluster) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            dst_smem),
        "l"(map), "r"(c0), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(bar_cluster)
        : "memory");
}

// Position in a ring of N slots: slot and how often it has come round. (Divisions of a running 64-bit block number by the ring
// sizes cost the unpack warps a fifth of their time.)
template <int N>
struct URing {
    uint32_t slot = 0, lap = 0;
    __device__ __forceinline__ void step(uint32_t by = 1) {
        slot += by;
        if (slot >= N) { slot -= N; lap++; }
    }
    __device__ __forceinline__ uint32_t full_parity() const { return lap & 1; }
    __device__ __forceinline__ uint32_t empty_parity() const { return (lap - 1) & 1; }     // of the previous lap; waited for when lap > 0
};

// Tensor maps of the activations: boxes of 128, 64, 32 and 16 rows, of which a tile's half is put together with as few copies
// as possible (a copy costs its issuing thread ~150 clocks whatever its size); with an index, map 0 has boxes of one row.
struct UXMaps {
    CUtensorMap map[4];
};

struct UTile {
    int expert, first, valid, n;      // slots [first, first + valid), n = valid rounded up to 32
    int m0;                           // first weight row of the pair's tile
    int kb0, kb1, split;              // 128-column blocks
};

// The list of tiles, derived from the offsets by every CTA alike (shared memory, read-only after the prologue).
struct UPlan {
    const int* first;                 // [E + 1]
    const int* tiles;                 // [E + 1] exclusive prefix of activation tiles
    int E, mpairs, splits, nkb;
    __device__ __forceinline__ int total() const { return tiles[E] * mpairs * splits; }
    __device__ __forceinline__ UTile get(int t) const {
        UTile r;
        r.split = 0;
        if (splits > 1) {
            r.split = t % splits;
            t /= splits;
        }
        const int tt = (int)((unsigned)t / (unsigned)mpairs), rt = t - tt * mpairs;
        int lo = 0, hi = E;           // tiles[lo] <= tt < tiles[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tiles[mid] <= tt) lo = mid;
            else hi = mid;
        }
        const int k = tiles[lo + 1] - tiles[lo], count = first[lo + 1] - first[lo];
        const int step = ((count + k - 1) / k + 31) & ~31;      // the expert's rows in equal tiles
        const int at = (tt - tiles[lo]) * step;
        r.expert = lo;
        r.first = first[lo] + at;
        r.valid = count - at < step ? count - at : step;
        r.n = (r.valid + 31) & ~31;
        r.m0 = rt * 256;
        r.kb0 = 0;
        r.kb1 = nkb;
        if (splits > 1) {
            r.kb0 = nkb * r.split / splits;              // nkb <= 2^17, splits <= 8
            r.kb1 = nkb * (r.split + 1) / splits;
        }
        return r;
    }
};

// Which accumulator halves a tile takes, and how often each has been used: every role steps through the same sequence.
struct UHalves {
    int next = 0, used[2] = {0, 0}, led[2] = {0, 0};
    int mask, lead;                   // lead: the half whose d_full barrier announces the tile
    __device__ __forceinline__ void take(int n) {
        if (n > 128) {
            mask = 3;
            lead = 0;
        } else {
            mask = 1 << next;
            lead = next;
            next ^= 1;
        }
    }
    __device__ __forceinline__ void done() {
        if (mask & 1) used[0]++;
        if (mask & 2) used[1]++;
        led[lead]++;
    }
};

// VEC: the result's rows start on 16-byte boundaries, by their first and their pitch. Where they do not, octets go out in as few pieces as their address allows (14340 x 4096 on
// 2000 rows 170 us, 14336 x 4096 from an odd address 165 to 185; value by value 225 to 250); as a branch of one kernel that cost the others up to a tenth (4096 x 256 on 4096 rows 27.7 -> 30.4).
template <typename T, int GW, bool GATHER, bool VEC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kUThreads, 1)
w4_umma_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ UXMaps tmap_x, const W4UmmaParams p) {
    using C = UCfg;
    grid_launch_dependents();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = smem;
    uint8_t* sW = sB + C::STAGES * C::B_STAGE_BYTES;
    uint8_t* sOut = sW + C::W_STAGES * C::W_STAGE_BYTES;
    uint8_t* misc = sOut + C::STAGING_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(misc);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(misc + 320);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    int* s_first = reinterpret_cast<int*>(misc + 512);
    int* s_tiles = s_first + kUMaxExperts + 8;

    const uint32_t w_full = smem_u32(bars);
    const uint32_t w_empty = w_full + 8 * C::W_STAGES;
    const uint32_t full = w_empty + 8 * C::W_STAGES;     // [S] even CTA: operand stage filled in both CTAs
    const uint32_t empty = full + 8 * C::STAGES;         // [S] both CTAs: operand stage consumed
    const uint32_t d_full = empty + 8 * C::STAGES;       // [2] both CTAs: accumulator (half) complete
    const uint32_t d_empty = d_full + 16;                // [2] even CTA: accumulator half read out in both CTAs
    const uint32_t drained = d_empty + 16;               // both CTAs: every UMMA has been executed

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
    const uint32_t full_leader = mapa_shared(full, 0);
    const uint32_t d_empty_leader = mapa_shared(d_empty, 0);
    const int nkb = (p.g.K + kW4Block - 1) / kW4Block;

    if (warp == 0) {
        for (int i = lane; i < C::NBARS; i += 32) {
            const int f0 = 2 * C::W_STAGES, d0 = f0 + 2 * C::STAGES;
            int count = 1;
            if (i >= C::W_STAGES && i < 2 * C::W_STAGES) count = 4;           // w_empty: unpack warps of a set
            else if (i >= f0 && i < f0 + C::STAGES) count = 9;                // full: activation producer + unpack warps of a set in both CTAs
            else if (i == d0 + 2 || i == d0 + 3) count = 16;                  // d_empty: epilogue warps of both CTAs
            mbar_init(w_full + 8 * i, count);
        }
        if (lane == 0) { *abort_flag = 0; set_wait_budget(abort_flag, p.wait_budget); }
        mbar_fence_init();
    } else if (warp == kUWarpMma) {
        tmem_alloc_pair(smem_u32(tmem_holder), 512);
    } else if (warp == kUWarpB && lane == 0) {
        tma_prefetch_desc(&tmap_x.map[0]);
        tma_prefetch_desc(&tmap_w);
    }
    grid_dependency_wait();

    // ---- the plan, by one warp: the experts' ranges, the tile width, prefix sums of the tiles ----
    const int E = p.g.E;
    if (warp == 1) {
        int carry = 0;                                   // ranges are made ascending and kept inside [0, slots]
        for (int base = 0; base <= E; base += 32) {
            const int e = base + lane;
            int v = 0;
            if (e <= E) {
                v = p.g.offsets ? p.g.offsets[e] : (e ? (int)p.g.slots : 0);
                v = v < 0 ? 0 : (v > (int)p.g.slots ? (int)p.g.slots : v);
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) v = max(v, __shfl_up_sync(0xffffffffu, v, d));
            v = max(v, carry);
            if (e <= E) s_first[e] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
        __syncwarp();
        // candidate widths 32, 64 .. 256; lane c of the first eight works out the cost of 32 (c + 1)
        int tiles[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int e = lane; e < E; e += 32) {
            const unsigned n = (unsigned)(s_first[e + 1] - s_first[e]);
#pragma unroll
            for (int c = 0; c < 8; c++) tiles[c] += (int)((n + 32 * c + 31) / (32 * c + 32));
        }
        int mine = 0;
#pragma unroll
        for (int c = 0; c < 8; c++) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) tiles[c] += __shfl_xor_sync(0xffffffffu, tiles[c], d);
            if (lane == c) mine = tiles[c];
        }
        // clocks of a tile, as measured: 620 + 2.3 per column for each 128-column block, and a fixed part for filling the pipeline
        // and draining the accumulator
        const int nt = 32 * (lane + 1);
        const float rounds = ceilf((float)mine * (float)(p.mpairs * p.splits) / (float)ncl);
        const float per_block = 620.f + 2.3f * (float)nt;
        float cost = rounds * (per_block * (float)((nkb + p.splits - 1) / p.splits) + 2000.f + 6.f * (float)nt);
        int best = lane < 8 ? lane : 7;
        if (lane >= 8) cost = 3.0e38f;
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) {                // the least cost; of equal ones the wider tile
            const float oc = __shfl_xor_sync(0xffffffffu, cost, d);
            const int ob = __shfl_xor_sync(0xffffffffu, best, d);
            if (oc < cost || (oc == cost && ob > best)) {
                cost = oc;
                best = ob;
            }
        }
        const unsigned width = 32u * (unsigned)(__shfl_sync(0xffffffffu, best, 0) + 1);
        carry = 0;
        for (int base = 0; base < E; base += 32) {
            const int e = base + lane;
            const int x = e < E ? (int)(((unsigned)(s_first[e + 1] - s_first[e]) + width - 1) / width) : 0;
            int s = x;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += up;
            }
            if (e < E) s_tiles[e] = carry + s - x;
            carry += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) s_tiles[E] = carry;
    }
    tc_fence_before();
    __syncwarp();
    // Both CTAs' barriers exist before anybody signals across the pair; the plan is visible to the CTA.
    cluster_arrive_release();
    cluster_wait_acquire();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    const uint32_t tmem_a = tmem + C::A_COL0;
    const UPlan plan{s_first, s_tiles, E, p.mpairs, p.splits, nkb};
    const int total = plan.total();

    if (warp == kUWarpW) {
        // ---------------- codes: this CTA's 128 rows ----------------
        if (lane == 0) {
            URing<C::W_STAGES> ring;
            bool ok = true;
            for (int t = cid; t < total && ok; t += ncl) {
                const UTile u = plan.get(t);
                const int row = u.m0 + (int)rank * 128;
                for (int i = u.kb0; i < u.kb1; i++, ring.step()) {
                    if (ring.lap) ok = mbar_wait_relaxed(w_empty + 8 * ring.slot, ring.empty_parity(), abort_flag, p.status, 51);
                    if (!ok) break;
                    if (i - u.kb0 == p.test_skip_kblock) continue;    // test hook: this block never arrives, its consumers' waits run out
                    mbar_arrive_expect_tx(w_full + 8 * ring.slot, C::W_STAGE_BYTES);
                    tma_load_3d(smem_u32(sW) + ring.slot * C::W_STAGE_BYTES, &tmap_w, i * kW4BlockBytes, row, u.expert, w_full + 8 * ring.slot);
                }
            }
            if (*abort_flag) {  // copies in flight must land before the CTA may exit: wait for the longest plausible copy time
                const long long t0 = clock64();
                while (clock64() - t0 < kUCopyDrainClocks) {}
            }
        }
    } else if (warp >= kUWarpB) {
        // ---------------- activations: this CTA's half of the tile's rows; warp 26 the even operand stages, warp 27 the odd ones ----------------
        // A wait, the announcement and a copy cost ~600 clocks of one thread, more than a stage's products (448 for 224 rows):
        // one warp alone held the tensor cores to 55 %. As above, the whole warp walks and one elected lane issues.
        const int me = warp - kUWarpB;
        URing<C::STAGES> ring;
        ring.step(me);
        int skip = me;
        bool ok = true;
        for (int t = cid; t < total && ok; t += ncl) {
            const UTile u = plan.get(t);
            const int half = __shfl_sync(0xffffffffu, u.n >> 1, 0);  // a multiple of 16
            const int at = (int)rank * half;
            const int row0 = __shfl_sync(0xffffffffu, u.first + at, 0);
            int row[4] = {0, 0, 0, 0};
            if (GATHER) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int n = at + lane * 4 + q;
                    // rows behind the tile and indices outside x lie outside the tensor map: zeros
                    int r = -1;
                    if (lane * 4 < half && n < u.valid) r = p.g.rows[u.first + n];
                    row[q] = r < 0 || r >= (int)p.g.x_rows ? (int)p.g.x_rows : r;
                }
            }
            const int kb1 = __shfl_sync(0xffffffffu, u.kb1, 0);
            int i = __shfl_sync(0xffffffffu, u.kb0, 0) + skip;
            for (; i < kb1; i += 2, ring.step(2)) {
                const uint32_t s = ring.slot;
                ok = __all_sync(0xffffffffu, ring.lap == 0 || mbar_wait(empty + 8 * s, ring.empty_parity(), abort_flag, p.status, 52));
                if (!ok) break;
                const uint32_t dst = smem_u32(sB) + s * C::B_STAGE_BYTES, bar = full_leader + 8 * s;
                // one arrival for the pair, announcing the bytes of both halves
                if (leader && elect_one()) mbar_arrive_expect_tx(full + 8 * s, 2 * half * 256);
                __syncwarp();
                if (GATHER) {
                    if (lane * 4 < half) {
                        tma_gather4_pair(dst + lane * 512, &tmap_x.map[0], i * kW4Block, row, bar);
                        tma_gather4_pair(dst + C::B_SUB_BYTES + lane * 512, &tmap_x.map[0], i * kW4Block + 64, row, bar);
                    }
                } else if (elect_one()) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t to = dst + h * C::B_SUB_BYTES;
                        const int c = i * kW4Block + h * 64;
                        if (half == 128) {
                            tma_load_3d_pair(to, &tmap_x.map[0], c, row0, 0, bar);
                        } else {
                            if (half & 64) tma_load_3d_pair(to, &tmap_x.map[1], c, row0, 0, bar);
                            if (half & 32) tma_load_3d_pair(to + (half & 64) * 128, &tmap_x.map[2], c, row0 + (half & 64), 0, bar);
                            if (half & 16) tma_load_3d_pair(to + (half & 96) * 128, &tmap_x.map[3], c, row0 + (half & 96), 0, bar);
                        }
                    }
                }
                __syncwarp();
            }
            skip = i - kb1;                                   // 0 or 1 blocks into the next tile
        }
        if (*abort_flag) {
            const long long t0 = clock64();       // as above
            while (clock64() - t0 < kUCopyDrainClocks) {}
        }
    } else if (warp == kUWarpMma) {
        // ---------------- UMMA issuer (even CTA) ----------------
        // The whole warp walks through the loop and one elected lane issues: what the instruction takes from uniform registers
        // (descriptors, addresses) is then computed there. A loop under "if (lane == 0)" moved every operand over for each
        // product and cost its thread ~130 clocks apiece, more than a product of 256 columns takes.
        if (leader) {
            bool ok = true;
            URing<C::STAGES> ring;
            bool peek = false;                        // the next stage is known to be full
            UHalves h;
            const uint32_t bdesc_hi = (uint32_t)(umma_desc_sw128(0) >> 32);
            const uint32_t bdesc_lo = __shfl_sync(0xffffffffu, (uint32_t)umma_desc_sw128(smem_u32(sB)), 0);
            const uint32_t a0 = __shfl_sync(0xffffffffu, tmem_a, 0), d0 = __shfl_sync(0xffffffffu, tmem, 0);
            for (int t = cid; t < total && ok; t += ncl) {
                const UTile u = plan.get(t);
                h.take(u.n);
                // the first product of a tile overwrites its accumulator: the epilogue warps of both CTAs must have read it out
                if ((h.mask & 1) && h.used[0] > 0) ok = mbar_wait(d_empty, (uint32_t)(h.used[0] - 1) & 1, abort_flag, p.status, 55);
                if (ok && (h.mask & 2) && h.used[1] > 0) ok = mbar_wait(d_empty + 8, (uint32_t)(h.used[1] - 1) & 1, abort_flag, p.status, 55);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t idesc = __shfl_sync(0xffffffffu, umma_idesc_16(W4Type<T>::kMagicValue == 128.f, u.n), 0);
                const uint32_t d = d0 + __shfl_sync(0xffffffffu, h.lead, 0) * 128;
                const int steps = __shfl_sync(0xffffffffu, u.kb1 - u.kb0, 0);
                for (int i = 0; i < steps; i++) {
                    const uint32_t s = ring.slot;
                    if (!peek) ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * s, ring.full_parity(), abort_flag, p.status, 53));
                    if (!ok) break;
                    tc_fence_after();
                    ring.step();
                    // the next stage is asked for before this one's products are issued: a probe takes ~100 clocks to answer
                    const bool next = mbar_test(full + 8 * ring.slot, ring.full_parity());
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint64_t bdesc = ((uint64_t)bdesc_hi << 32) | (bdesc_lo + ((s * C::B_STAGE_BYTES + (j >> 2) * C::B_SUB_BYTES + (j & 3) * 32) >> 4));
                            umma_f16_ts_pair(d, a0 + s * C::A_STAGE_COLS + j * 8, bdesc, idesc, (i | j) ? 1u : 0u);
                        }
                        umma_commit_pair_mask(empty + 8 * s, (uint16_t)3);
                        if (i == steps - 1) umma_commit_pair_mask(d_full + 8 * h.lead, (uint16_t)3);
                    }
                    __syncwarp();
                    peek = __all_sync(0xffffffffu, next);
                }
                if (!ok) break;
                h.done();
            }
            if (elect_one()) umma_commit_pair_mask(drained, (uint16_t)3);
        }
    } else if (warp < 4 * kUSets) {
        // ---------------- unpack: set s takes the blocks g of the CTA's stream with g % 4 == s ----------------
        const int set = warp >> 2;
        const int r = (warp & 3) * 32 + lane;                 // weight row of this CTA's half tile == tensor-memory lane
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        constexpr int G = 4 / GW;                             // scale groups of a block
        bool ok = true;
        const uint32_t magic = w4_opaque(W4Type<T>::kMagic);
        URing<C::W_STAGES> wring;                             // of the set's next block
        wring.step(set);
        uint32_t lap = 0;                                     // blocks of the set so far
        int skip = set;                                       // blocks until the set's next one, counted from the tile's first
        for (int t = cid; t < total && ok; t += ncl) {
            const UTile u = plan.get(t);
            int m = u.m0 + (int)rank * 128 + r;
            if (m >= p.g.M) m = p.g.M - 1;                    // rows behind the matrix: zero codes from the tensor map, any scale
            const long long at = ((long long)u.expert * p.g.M + m) * p.g.groups;
            const uint16_t* srow = p.g.scales + at;
            const uint8_t* zrow = p.g.zeros ? p.g.zeros + at : nullptr;
            // The scales (two in a word) and zero points (four) of a block, loaded a block of the set ahead. A lane's row is its own cache
            // line, so it is the number of loads that costs: one of each where the row's alignment allows it (28672 x 8192 on 16 rows in
            // groups of 64: 71 -> 61 us, of 32: 106 -> 67).
            constexpr int SW = (G + 1) / 2;
            struct Raw { uint32_t s[SW], z; };
            const bool wide = reinterpret_cast<uintptr_t>(srow) % (2 * G) == 0 && reinterpret_cast<uintptr_t>(zrow) % G == 0;
            const auto fetch = [&](Raw& v, int kb) {
                if (kb >= u.kb1) return;
                const uint16_t* sp = srow + kb * G;
                const uint8_t* zp = zrow + kb * G;
                v.z = 0x08080808u;
                if (G > 1 && wide && (kb + 1) * G <= p.g.groups) {
                    if constexpr (G == 2) {
                        v.s[0] = __ldg(reinterpret_cast<const uint32_t*>(sp));
                        if (zrow) v.z = __ldg(reinterpret_cast<const uint16_t*>(zp));
                    } else if constexpr (G == 4) {
                        const uint2 s4 = __ldg(reinterpret_cast<const uint2*>(sp));
                        v.s[0] = s4.x; v.s[1] = s4.y;
                        if (zrow) v.z = __ldg(reinterpret_cast<const uint32_t*>(zp));
                    }
                    return;
                }
                uint32_t sv[G], zv[G];
#pragma unroll
                for (int q = 0; q < G; q++) {
                    const int c = kb * G + q < p.g.groups ? q : p.g.groups - 1 - kb * G;      // behind K: the activations there are zero
                    sv[q] = __ldg(sp + c);
                    zv[q] = zrow ? __ldg(zp + c) : 8u;
                }
                v.z = 0u;
#pragma unroll
                for (int q = 0; q < SW; q++) v.s[q] = sv[2 * q] | (2 * q + 1 < G ? sv[2 * q + 1 < G ? 2 * q + 1 : 0] << 16 : 0u);
#pragma unroll
                for (int q = 0; q < G; q++) v.z |= zv[q] << (8 * q);
            };
            int kb = u.kb0 + skip;
            Raw now{};
            fetch(now, kb);
            for (; kb < u.kb1 && ok; kb += kUSets, lap++) {
                const uint32_t ws = wring.slot;
                ok = mbar_wait(w_full + 8 * ws, wring.full_parity(), abort_flag, p.status, 57);
                wring.step(kUSets);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // TMA's 64-byte swizzle: 16-byte piece c of row r sits at piece c ^ (r / 2 % 4)
                const uint8_t* src = sW + ws * C::W_STAGE_BYTES + r * kW4BlockBytes;
                const int x = (r >> 1) & 3;
                const uint4 c0 = *reinterpret_cast<const uint4*>(src + ((0 ^ x) << 4));
                const uint4 c1 = *reinterpret_cast<const uint4*>(src + ((1 ^ x) << 4));
                const uint4 c2 = *reinterpret_cast<const uint4*>(src + ((2 ^ x) << 4));
                const uint4 c3 = *reinterpret_cast<const uint4*>(src + ((3 ^ x) << 4));
                fence_proxy_async_smem();     // generic-proxy reads before the producer's next copy into this stage
                __syncwarp();
                if (lane == 0) mbar_arrive(w_empty + 8 * ws);
                const Raw cur = now;
                fetch(now, kb + kUSets);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    // the first half's arithmetic comes before the wait for the stage
                    uint32_t v[32];
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int w = 2 * half + q;
                        const uint32_t pair = cur.s[w / GW / 2];
                        const auto s2 = w4_splat<T>(w / GW % 2 ? pair >> 16 : pair & 0xffffu);
                        const auto mz = w4_splat<T>(w4_magic_zero_bits<T>(cur.z >> (8 * (w / GW))));
                        const uint32_t word[4] = {w == 0 ? c0.x : (w == 1 ? c0.y : (w == 2 ? c0.z : c0.w)), w == 0 ? c1.x : (w == 1 ? c1.y : (w == 2 ? c1.z : c1.w)),
                                                  w == 0 ? c2.x : (w == 1 ? c2.y : (w == 2 ? c2.z : c2.w)), w == 0 ? c3.x : (w == 1 ? c3.y : (w == 2 ? c3.z : c3.w))};
#pragma unroll
                        for (int e = 0; e < 16; e++) v[16 * q + e] = w4_pair<T>(word[e >> 2] >> (4 * (e & 3)), mz, s2, magic);
                    }
                    // Codes behind K stand for zero: their activations are, but (q - z) s of what they hold may be no number of the type. (The test
                    // costs 0 to 2 % of narrow tiles; once a block, on the codes, 28672 x 8192 on 16 rows in groups of 128 took 57.8 us against 54.4.)
                    const int left = p.g.K - kb * kW4Block - half * 64;
                    if (left < 64) {
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (2 * e + 1 >= left) v[e] = 2 * e < left ? v[e] & 0xffffu : 0u;
                    }
                    if (half == 0) {
                        if (lap) ok = mbar_wait(empty + 8 * set, (lap - 1) & 1, abort_flag, p.status, 58);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    tmem_st32(tmem_a + lane_base + set * C::A_STAGE_COLS + half * 32, v);
                }
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_pair(full_leader + 8 * set);
            }
            skip = kb - u.kb1;                                // 0 .. 3
        }
    } else if (warp >= kUWarpEpi && warp < kUWarpEpi + 8) {
        // ---------------- epilogue: this CTA's 128 weight rows; columns [hw n / 2, (hw + 1) n / 2) per group of four warps ----------------
        const int hw = (warp - kUWarpEpi) >> 2;
        const int et = (warp & 3) * 32 + lane;                // weight row == tensor-memory lane; also the thread's number in its group
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        uint8_t* stage = sOut + hw * C::STAGED * C::PITCH;
        UHalves h;
        for (int t = cid; t < total; t += ncl) {
            const UTile u = plan.get(t);
            h.take(u.n);
            bool ok = mbar_wait_relaxed(d_full + 8 * h.lead, (uint32_t)h.led[h.lead] & 1, abort_flag, p.status, 59);
            if (named_bar_or(1 + hw, 128, !ok)) break;        // one answer for the four warps
            tc_fence_after();
            const int ncols = u.n >> 1, col0 = hw * ncols;    // a multiple of 16
            const uint32_t acc = tmem + h.lead * 128 + lane_base + col0;
            const int m0 = u.m0 + (int)rank * 128;
            for (int c0 = 0; c0 < ncols; c0 += C::STAGED) {
                const int nc = ncols - c0 < C::STAGED ? ncols - c0 : C::STAGED;
                if (c0) named_bar_sync(1 + hw, 128);          // the staging columns have been stored
                for (int c = 0; c < nc; c += 16) {
                    uint32_t v[16];
                    tmem_ld16(acc + c0 + c, v);
                    tmem_wait_ld();
                    if (p.partial) {
#pragma unroll
                        for (int q = 0; q < 16; q++) {
                            const int n = col0 + c0 + c + q;
                            if (n < u.valid && m0 + et < p.g.M)
                                p.partial[((long long)u.split * p.g.slots + u.first + n) * p.g.M + m0 + et] = __uint_as_float(v[q]);
                        }
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; q++)
                            *reinterpret_cast<uint16_t*>(stage + (c + q) * C::PITCH + et * 2) = W4Type<T>::from_float(__uint_as_float(v[q]));
                    }
                }
                if (c0 + C::STAGED >= ncols) {                       // everything is out of the accumulator
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (h.mask & 1) arrive_pair(d_empty_leader);
                        if (h.mask & 2) arrive_pair(d_empty_leader + 8);
                    }
                }
                if (!p.partial) {
                    named_bar_sync(1 + hw, 128);
                    // sixteen threads store the 128 rows of a column: 256 contiguous bytes
                    for (int o = et; o < nc * 16; o += 128) {
                        const int c = o >> 4, m = (o & 15) * 8, n = col0 + c0 + c;
                        if (n < u.valid && m0 + m < p.g.M) {
                            uint16_t* dst = static_cast<uint16_t*>(p.g.out) + (long long)(u.first + n) * p.g.out_ld + m0 + m;
                            const uint4 v = *reinterpret_cast<const uint4*>(stage + c * C::PITCH + m * 2);
                            if constexpr (!VEC) {
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                                store_octet(dst, p.g.M - m0 - m, w);
                            } else if (m0 + m + 8 <= p.g.M) {
                                *reinterpret_cast<uint4*>(dst) = v;
                            } else {
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int q = 0; q < 8; q++)
                                    if (m0 + m + q < p.g.M) dst[q] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
                            }
                        }
                    }
                }
            }
            h.done();
            named_bar_sync(1 + hw, 128);                      // the staging columns are free for the next tile
        }
    }
    tc_fence_before();
    __syncwarp();
    // Both CTAs are done with each other's barriers and tensor memory before either frees it or exits.
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp == kUWarpMma) {
        if (lane == 0) {   // every UMMA has been executed before the columns are freed (immediate unless a wait ran out)
            const long long t0 = clock64();
            while (!mbar_test(drained, 0) && clock64() - t0 < wait_budget_of(abort_flag)) {}
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// out[s, m] = r16(sum over the K partitions, in order), for the slots below offsets[E].
template <typename T>
__global__ void __launch_bounds__(256) w4_sum_kernel(const W4Gemm g, const float* __restrict__ partial, int splits) {
    grid_dependency_wait();
    long long slots = g.slots;
    if (g.offsets) {
        int last = 0;                                         // the largest offset: the ranges are made ascending by the product kernel
        for (int e = threadIdx.x & 31; e <= g.E; e += 32) last = max(last, g.offsets[e]);
        last = __reduce_max_sync(0xffffffffu, last);
        if (last < slots) slots = last;
    }
    int low = 0;
    if (g.offsets) low = g.offsets[0] < 0 ? 0 : g.offsets[0];
    const long long chunks = (g.M + 3) / 4, total = slots * chunks;
    const bool vec = g.M % 4 == 0;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long s = i / chunks;
        const int m = (int)(i - s * chunks) * 4;
        if (s < low) continue;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        for (int q = 0; q < splits; q++) {
            const float* src = partial + ((long long)q * g.slots + s) * g.M + m;
            if (vec) {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(src));
                a[0] += v.x; a[1] += v.y; a[2] += v.z; a[3] += v.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (m + c < g.M) a[c] += src[c];
            }
        }
        uint16_t* dst = static_cast<uint16_t*>(g.out) + s * g.out_ld + m;
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (m + c < g.M) dst[c] = W4Type<T>::from_float(a[c]);
    }
}

// The rows of x that the slots name, in slot order, rows 16 bytes apart or a multiple of it; an index outside x gives zeros.
__global__ void __launch_bounds__(256) w4_gather_kernel(const W4Gemm g, uint16_t* __restrict__ dst, long long dst_ld) {
    grid_dependency_wait();
    const long long chunks = dst_ld / 8, total = g.slots * chunks;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long s = i / chunks;
        const int k = (int)(i - s * chunks) * 8, r = __ldg(g.rows + s);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r >= 0 && r < (int)g.x_rows) {
            const uint16_t* src = static_cast<const uint16_t*>(g.x) + (long long)r * g.x_ld + k;
            if (k + 8 <= g.K) {
                v = __ldg(reinterpret_cast<const uint4*>(src));      // rows of x start on 16-byte boundaries on this path
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
                for (int c = 0; c < 8 && k + c < g.K; c++) w[c >> 1] |= (uint32_t)__ldg(src + c) << (16 * (c & 1));
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        *reinterpret_cast<uint4*>(dst + s * dst_ld + k) = v;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
// K partitions of a launch with few tiles. A 128-column block of a tile costs a pair ~0.4 us (its codes) or 0.54 us times
// its share of 256 columns (its products); the second kernel that adds the partitions up costs ~3.5 us and its bytes.
// (9472 x 1024 on 256 rows, 37 tiles: 11.6 us whole, 22.6 in two.)
static int w4_splits(const W4Gemm& p) {
    const long long pairs = sm_count() / 2, mpairs = (p.M + 255) / 256, nkb = (p.K + kW4Block - 1) / kW4Block;
    const long long experts = p.offsets ? (p.slots < p.E ? p.slots : p.E) : 1;
    const long long rows = (p.slots + experts - 1) / experts;                 // of an expert, on average
    const long long cols = (rows + 255) / 256, width = (rows + cols - 1) / cols;
    const long long tiles = mpairs * experts * cols;
    if (tiles >= pairs) return 1;
    const double block_us = width > 190 ? 0.54 * (double)width / 256.0 : 0.4;
    int best = 1;
    double least = 0;
    for (int s = 1; s <= 8 && s <= nkb; s++) {
        const long long rounds = (tiles * s + pairs - 1) / pairs;
        const double t = (double)rounds * (double)((nkb + s - 1) / s) * block_us + (s > 1 ? 3.5 + (double)s * (double)p.slots * (double)p.M * 8.0 / 3.0e6 : 0.0);
        if (s == 1 || t < least) {
            best = s;
            least = t;
        }
    }
    return best;
}

// With an index: the rows are put together first where experts have more than 24 of them. tile::gather4 costs its issuer a
// copy for every four rows, which holds wide tiles up (8 x 14336 x 4096 on 8192 rows: 1082 us against 694; 64 x 2048 x 4096 on
// 2048 rows: 125 against 115), while narrow ones hide it and save the launch (64 x 1001 x 2056 on 768 rows: 40.8, 39.9 in order).
static long long w4_gathered_ld(const W4Gemm& p, bool indexed) {
    const long long experts = p.slots < p.E ? p.slots : p.E;
    return indexed && p.slots > 24 * experts ? (p.K + 7) / 8 * 8 : 0;
}

static size_t partial_bytes(const W4Gemm& p) {
    const int s = w4_splits(p);
    return s > 1 ? align_up((size_t)s * (size_t)p.slots * (size_t)p.M * 4, 256) : 0;
}
size_t w4_umma_workspace(const W4Gemm& p) { return partial_bytes(p) + (size_t)p.slots * (size_t)w4_gathered_ld(p, p.offsets != nullptr) * 2; }

template <typename T, int GW, bool GATHER, bool VEC>
static int umma_variant(cudaStream_t stream, const CUtensorMap& tw, const UXMaps& tx, const W4UmmaParams& p) {
    using C = UCfg;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(w4_umma_kernel<T, GW, GATHER, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
        if (e != cudaSuccess) return (int)e;
        if (dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count() / 2 * 2), 1, 1);
    cfg.blockDim = dim3(kUThreads, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    if (programmatic_launch_enabled()) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, w4_umma_kernel<T, GW, GATHER, VEC>, tw, tx, p);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    if (p.partial) {
        long long blocks = (p.g.slots * ((p.g.M + 3) / 4) + 255) / 256;
        if (blocks > (long long)sm_count() * 8) blocks = (long long)sm_count() * 8;
        e = launch_pdl(w4_sum_kernel<T>, dim3((unsigned)blocks), dim3(256), stream, p.g, (const float*)p.partial, p.splits);
        count_launch();
        if (e != cudaSuccess) return (int)e;
    }
    return (int)cudaGetLastError();
}

template <typename T, bool GATHER, bool VEC>
static int umma_groups(cudaStream_t stream, const CUtensorMap& tw, const UXMaps& tx, const W4UmmaParams& p) {
    if (p.g.group == 32) return umma_variant<T, 1, GATHER, VEC>(stream, tw, tx, p);
    if (p.g.group == 64) return umma_variant<T, 2, GATHER, VEC>(stream, tw, tx, p);
    return umma_variant<T, 4, GATHER, VEC>(stream, tw, tx, p);
}
template <typename T>
static int umma_dtype(cudaStream_t stream, const CUtensorMap& tw, const UXMaps& tx, const W4UmmaParams& p) {
    const bool vec = p.g.out_ld % 8 == 0 && reinterpret_cast<uintptr_t>(p.g.out) % 16 == 0;
    if (p.g.rows) return vec ? umma_groups<T, true, true>(stream, tw, tx, p) : umma_groups<T, true, false>(stream, tw, tx, p);
    return vec ? umma_groups<T, false, true>(stream, tw, tx, p) : umma_groups<T, false, false>(stream, tw, tx, p);
}

// TMA needs rows of x on 16-byte boundaries. Without a workspace K is not divided and rows are taken by index.
int launch_w4_umma(cudaStream_t stream, const W4Gemm& problem, int dtype, void* workspace) {
    W4UmmaParams q{};
    q.g = problem;
    W4Gemm& p = q.g;
    q.status = device_status_word();
    q.splits = workspace ? w4_splits(p) : 1;
    q.partial = q.splits > 1 ? static_cast<float*>(workspace) : nullptr;
    q.mpairs = (p.M + 255) / 256;
    if (const long long ld = p.rows && workspace ? w4_gathered_ld(p, true) : 0) {
        uint16_t* to = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + partial_bytes(p));
        long long blocks = (p.slots * (ld / 8) + 255) / 256;
        if (blocks > (long long)sm_count() * 32) blocks = (long long)sm_count() * 32;
        const cudaError_t e = launch_pdl(w4_gather_kernel, dim3((unsigned)blocks), dim3(256), stream, p, to, ld);
        count_launch();
        if (e != cudaSuccess) return (int)e;
        p.x = to;
        p.x_ld = ld;
        p.x_rows = p.slots;
        p.rows = nullptr;
    }
    CUtensorMap tw;
    UXMaps tx{};
    const cuuint64_t wdims[3] = {(cuuint64_t)p.row_bytes, (cuuint64_t)p.M, (cuuint64_t)p.E};
    const cuuint64_t wstrides[2] = {(cuuint64_t)p.row_bytes, (cuuint64_t)p.row_bytes * (cuuint64_t)p.M};
    const cuuint32_t wbox[3] = {(cuuint32_t)kW4BlockBytes, 128u, 1u}, ones[3] = {1u, 1u, 1u};
    int rc = encode_tensor_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.plane, wdims, wstrides, wbox, ones, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
    const cuuint64_t pitch = (cuuint64_t)(p.x_rows > 1 ? p.x_ld : (p.K + 7) / 8 * 8) * 2;
    const cuuint64_t xdims[3] = {(cuuint64_t)p.K, (cuuint64_t)p.x_rows, 1u}, xstrides[2] = {pitch, pitch * (cuuint64_t)p.x_rows};
    const CUtensorMapDataType kind = dtype == BGEMM_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int b = 0; b < (p.rows ? 1 : 4); b++) {
        const cuuint32_t xbox[3] = {64u, p.rows ? 1u : 128u >> b, 1u};
        rc = encode_tensor_map(&tx.map[b], kind, p.rows ? 2 : 3, p.x, xdims, xstrides, xbox, ones, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
    }
    GemmParams hooks{};
    apply_test_hooks(hooks);
    q.wait_budget = hooks.wait_budget;
    q.test_skip_kblock = hooks.test_skip_kblock;
    return dtype == BGEMM_DT_F16 ? umma_dtype<__half>(stream, tw, tx, q) : umma_dtype<__nv_bfloat16>(stream, tw, tx, q);
}

}  // namespace bgemm
