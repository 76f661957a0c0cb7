// Products of 8-bit rows with 4-bit weights (both in the microscaling form of mx.cuh), with float sums:
//   out[t, n] = epilogue(sum_k x[t, k] W[n, k]);  the gated epilogues take gate and up rows of W that alternate in groups of 8 and
//   give act(gate) * up, as values or as 8-bit rows for the product behind.
//
// Few rows (decode steps): bound by streaming W from HBM once.
//   * The tensor cores take both forms as they are, with their scales (tcgen05.mma kind::mxf8f6f4): no value is unpacked by a thread.
//     128 rows of W are the M side, one a lane of tensor memory; the rows of x, padded to a multiple of 16, the N side.
//   * A stage is 128 values of K: 8 KB of W (16 KB once the copy engine has spread it), the rows of x, and a block of scales of
//     each, which the thread that issues the products brings to columns of tensor memory of the stage's own.
//   * Where W has few tiles of 128 rows, a cluster of up to 8 CTAs shares K.  Each leaves its sums in shared memory, and each adds up
//     and stores a share of the rows, in the order of the ranks: the result does not depend on timing.
// Every wait is bounded: a CTA that gives up counts it (janis_mx_timeouts_async), waits for its copies, frees its tensor memory
// and leaves without a result.  No load here uses cluster multicast.
#include <cooperative_groups.h>

#include "mx_tc05.cuh"

namespace cg = cooperative_groups;

namespace janis {
namespace mx {

using namespace tc;

enum { EPI_NONE = 0, EPI_GATED_GELU = 1, EPI_GATED_SILU = 3, EPI_GATED_CLAMP = 4 };

__device__ int g_timeouts = 0;

struct Out {
    void* values;          // [T, N or N / 2] of `dtype`, or null
    uint8_t* codes;        // 8-bit rows instead
    uint8_t* scales;
    int dtype;
    int epi;
    float limit, alpha, up_add;
};

__device__ __forceinline__ float gated(float gate, float up, const Out& o) {
    if (o.epi == EPI_GATED_CLAMP) return clamped_gate(gate, up, o.limit, o.alpha, o.up_add);
    return (o.epi == EPI_GATED_GELU ? gelu_tanh(gate) : gate / (1.0f + expf(-gate))) * up;
}

constexpr int TILE = 128;                      // rows of W a CTA
constexpr int A_BYTES = TILE * 128, A_PACKED = A_BYTES / 2;
constexpr int MAX_STAGES = 11;
constexpr int MAX_ROWS = 256;                  // rows of x a CTA
constexpr int SCALE_BYTES = 3 * BLOCK_BYTES;   // of a stage: a block of W's, one or two of x's
constexpr int SCALE_COLS = 12;
constexpr int few_smem(int stages, int NP) { return stages * (A_BYTES + NP * 128 + SCALE_BYTES) + 1024; }

__global__ void __launch_bounds__(128)
few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ ws,
                const uint8_t* __restrict__ xs, const Out o, int T, int N, int kp, int NP, int split, int stages, int tmem_cols) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * MAX_STAGES + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int n0 = blockIdx.x / split * TILE, t0 = blockIdx.y * NP;
    const int blocks = kp / BLOCK;

    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t stage0 = (raw + 1023) & ~1023u;                   // swizzle atoms want 1024-byte alignment
    float* sums = reinterpret_cast<float*>(smem_raw + (stage0 - raw));      // [NP][TILE], once the stages are idle
    const int stage_bytes = A_BYTES + NP * 128;
    const uint32_t scales0 = stage0 + stages * stage_bytes;
    const uint32_t bar_full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t bar_empty = bar_full + 8 * stages, bar_done = bar_full + 16 * stages;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * stages + 1; ++i) mbar_init(bar_full + 8 * i, 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), tmem_cols);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;

    // this CTA's share of K: value blocks rank, rank + split, ...
    const int nk = (blocks - rank + split - 1) / split;
    const int x_blocks = NP > BLOCK && t0 + BLOCK < T ? 2 : 1;       // blocks of x's scales that are there
    // (a tile past W's rows, which only makes the padding of 8-bit rows, finds zeros there whatever their scales)
    const uint8_t* w_scales = ws + (size_t)min(n0 / BLOCK, (N - 1) / BLOCK) * blocks * BLOCK_BYTES;
    const uint8_t* x_scales = xs + (size_t)(t0 / BLOCK) * blocks * BLOCK_BYTES;

    int filled = 0;                                                   // stages that copies were asked for (thread 0)
    grid_dependents_launch();
    if (warp == 0 && lane == 0) {
        // ---- the copies.  The weights are constants of the model: the first tiles of W are on their way before this kernel
        // waits for the one that makes x.
        const int bytes = A_PACKED + NP * 128 + (1 + x_blocks) * BLOCK_BYTES;
        const auto load_w = [&](int i, int s) {
            mbar_expect_tx(bar_full + 8 * s, bytes);
            const int kb = rank + i * split;
            tma_load_2d(stage0 + s * stage_bytes, &map_w, kb * BLOCK, n0, bar_full + 8 * s);
            bulk_load(scales0 + s * SCALE_BYTES, w_scales + (size_t)kb * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const auto load_x = [&](int i, int s) {
            const int kb = rank + i * split;
            tma_load_2d(stage0 + s * stage_bytes + A_BYTES, &map_x, kb * BLOCK, t0, bar_full + 8 * s);
            for (int b = 0; b < x_blocks; ++b)
                bulk_load(scales0 + s * SCALE_BYTES + (1 + b) * BLOCK_BYTES, x_scales + ((size_t)b * blocks + kb) * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const int pre = nk < stages ? nk : stages;
        for (int i = 0; i < pre; ++i) load_w(i, i);
        grid_dependency_wait();
        for (int i = 0; i < pre; ++i) load_x(i, i);
        for (filled = pre; filled < nk; ++filled) {
            const int s = filled % stages;
            if (!mbar_wait(bar_empty + 8 * s, (filled / stages - 1) & 1)) { atomicExch(&failed, 1); break; }
            load_w(filled, s);
            load_x(filled, s);
        }
    } else if (warp == 1 && lane == 0) {
        // ---- the thread that issues the products
        grid_dependency_wait();
        for (int i = 0; i < nk; ++i) {
            const int s = i % stages;
            if (!mbar_wait(bar_full + 8 * s, (i / stages) & 1)) { atomicExch(&failed, 1); break; }
            fence_after_sync();
            const uint32_t a = stage0 + s * stage_bytes, b = a + A_BYTES, sc = scales0 + s * SCALE_BYTES;
            const uint32_t ta = tmem + NP + s * SCALE_COLS, tb = ta + 4;
            scales_to_tmem(ta, sc);
            for (int j = 0; j < x_blocks; ++j) scales_to_tmem(tb + 4 * j, sc + (1 + j) * BLOCK_BYTES);
#pragma unroll
            for (int g = 0; g < 4; ++g)                               // 32 bytes further along the swizzled row
                umma_block(tmem, smem_desc(a + g * 32), smem_desc(b + g * 32), block_desc<WEIGHTS>(TILE, NP, g), ta, tb, (i > 0 || g > 0) ? 1u : 0u);
            umma_commit(bar_empty + 8 * s);                           // the stage is free once these have read it
        }
        umma_commit(bar_done);                                        // all products of this CTA have finished
    } else {
        grid_dependency_wait();
    }
    __syncwarp();
    bool ok = mbar_wait_parked(bar_done, 0, &failed);
    ok = __syncthreads_and(ok ? 1 : 0) && failed == 0;
    fence_after_sync();
    if (!ok && threadIdx.x == 0)                                      // no copy is under way when the CTA leaves
        for (int j = filled > stages ? filled - stages : 0; j < filled; ++j) mbar_wait(bar_full + 8 * (j % stages), (j / stages) & 1);

    // ---- sums of row (32 * warp + lane) of the tile of W
    for (int c = 0; c < NP; c += 16) {
        uint32_t r[16];
        tmem_load16(r, tmem + ((uint32_t)(warp * 32) << 16) + c);
        tmem_wait_load();
#pragma unroll
        for (int j = 0; j < 16; ++j) sums[(c + j) * TILE + threadIdx.x] = __uint_as_float(r[j]);
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_free(tmem, tmem_cols);
    if (!ok && threadIdx.x == 0) atomicAdd(&g_timeouts, 1);
    cg::cluster_group cluster = cg::this_cluster();
    const float* theirs[8];
    if (split > 1) {
        cluster.sync();
        for (int r = 0; r < split; ++r) theirs[r] = cluster.map_shared_rank(sums, r);
    } else {
        theirs[0] = sums;
    }
    const auto sum_at = [&](int m, int row) {
        float v = theirs[0][m * TILE + row];
        for (int r = 1; r < split; ++r) v += theirs[r][m * TILE + row];
        return v;
    };
    // ---- this CTA's share: rows [row0, row0 + share) of the tile, all rows of x
    const int rows = T - t0 < NP ? T - t0 : NP, share = TILE / split, row0 = rank * share;
    if (ok) {
        if (o.epi == EPI_NONE) {
            for (int i = threadIdx.x; i < rows * share; i += 128) {
                const int m = i / share, row = row0 + i % share, n = n0 + row;
                if (n >= N) continue;
                const float v = sum_at(m, row);
                if (o.dtype == JANIS_BF16) reinterpret_cast<bf16*>(o.values)[(size_t)(t0 + m) * N + n] = from_float<bf16>(v);
                else reinterpret_cast<float*>(o.values)[(size_t)(t0 + m) * N + n] = v;
            }
        } else {
            // a gate's up stands 8 rows behind it; for 8-bit rows a warp has the 32 columns of a group (the share is 64 rows at least)
            const int cols = share / 2, c0 = n0 / 2 + row0 / 2, all = N / 2, wide = o.codes != nullptr ? padded(all) : all;
            for (int i = threadIdx.x; i < rows * cols; i += 128) {
                const int m = i / cols, j = i % cols, c = c0 + j, row = row0 + j / 8 * 16 + j % 8;
                const float v = c < all ? gated(sum_at(m, row), sum_at(m, row + 8), o) : 0.f;
                if (o.codes != nullptr) {
                    if (c - lane >= wide) continue;                   // (the whole warp)
                    float big = fabsf(v);
#pragma unroll
                    for (int s = 16; s > 0; s >>= 1) big = larger(big, __shfl_xor_sync(0xffffffffu, big, s));
                    const uint32_t byte = scale_byte_e4m3(big);
                    o.codes[(size_t)(t0 + m) * wide + c] = byte == 255u ? 0 : (uint8_t)two_e4m3(v * inverse_scale(byte), 0.f);
                    if (lane == 0) o.scales[scale_at(t0 + m, c / BLOCK, wide / BLOCK) + c % BLOCK / GROUP] = (uint8_t)byte;
                } else if (c < all) {
                    if (o.dtype == JANIS_BF16) reinterpret_cast<bf16*>(o.values)[(size_t)(t0 + m) * all + c] = from_float<bf16>(v);
                    else reinterpret_cast<float*>(o.values)[(size_t)(t0 + m) * all + c] = v;
                }
            }
        }
    }
    if (split > 1) cluster.sync();                                    // nobody leaves while its sums are read
}

static int sm_count() {
    static int sms = 0;
    if (sms == 0) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
            sms = 148;
    }
    return sms;
}

static int few_rows(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                    int split, int stages, cudaStream_t stream) {
    const int NP = T >= MAX_ROWS ? MAX_ROWS : (T + 15) / 16 * 16;
    // (8-bit rows are padded to whole blocks of 128 columns: 256 rows of gates and ups)
    const int tiles = o.codes != nullptr ? padded(N / 2) / (TILE / 2) : (N + TILE - 1) / TILE, blocks = kp / BLOCK, t_tiles = (T + NP - 1) / NP;
    const int most_split = o.codes != nullptr ? 2 : 8;                // (a group of 8-bit rows lies within a CTA's share)
    if (split == 0) {
        split = 1;
        while (split < most_split && tiles * t_tiles * split * 2 <= sm_count() && blocks >= split * 2) split *= 2;
    }
    if (split > most_split || split > blocks) return fail("mx_product: a split of %d is not possible here", split);
    if (stages == 0) {
        const int per_sm = (tiles * t_tiles * split + sm_count() - 1) / sm_count();
        stages = (227 * 1024 / (per_sm >= 2 ? 2 : 1) - 2048) / (A_BYTES + NP * 128 + SCALE_BYTES);
        if (NP > 128 && stages < 4) stages = 4;                       // (the sums of 256 rows leave through four stages)
        const int share = (blocks + split - 1) / split;
        if (stages > share) stages = share;
        while (few_smem(stages, NP) < NP * TILE * 4 + 1024) ++stages;
    }
    if (stages < 1 || stages > MAX_STAGES || few_smem(stages, NP) > 227 * 1024 - 512 || few_smem(stages, NP) < NP * TILE * 4 + 1024)
        return fail("mx_product: %d stages of %d rows do not fit", stages, NP);
    int cols = 32;
    while (cols < NP + stages * SCALE_COLS) cols *= 2;
    CUtensorMap mw, mx;
    if (!make_map(&mw, WEIGHTS, wc, N, kp, TILE) || !make_map(&mx, ROWS, xc, T, kp, NP))
        return fail("mx_product: cuTensorMapEncodeTiled is not available or refused the operands");
    static std::once_flag once;
    static cudaError_t e = cudaSuccess;
    std::call_once(once, [] { e = cudaFuncSetAttribute(few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 512); });
    if (e != cudaSuccess) return fail("mx_product: shared memory refused: %s", cudaGetErrorString(e));
    return launch_kernel("mx_product", few_rows_kernel, dim3(tiles * split, t_tiles), dim3(128), few_smem(stages, NP), stream, split, mw, mx, ws,
                         xs, o, T, N, kp, NP, split, stages, cols);
}

}  // namespace mx
}  // namespace janis

using namespace janis;

static int g_split = 0, g_stages = 0;

// Fixes the CTAs that share K (1, 2, 4, 8) and the depth of the ring of stages (0: chosen).  For tests and tuning.
JANIS_EXPORT void janis_mx_set_few(int split, int stages) {
    g_split = split;
    g_stages = stages;
}

// x: codes [T, padded K], W: codes [N, padded K / 2]; out [T, N] (N / 2 with a gated epilogue) of out_dtype, or 8-bit rows
JANIS_EXPORT int janis_mx_product(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, void* out, int out_dtype,
                                  uint8_t* out_codes, uint8_t* out_scales, int T, int N, int K, int epi, float limit, float alpha,
                                  float up_add, cudaStream_t stream) {
    if (T <= 0 || N <= 0) return 0;
    if (K <= 0) return fail("mx_product: a row has no values");
    if (epi != mx::EPI_NONE && epi != mx::EPI_GATED_GELU && epi != mx::EPI_GATED_SILU && epi != mx::EPI_GATED_CLAMP)
        return fail("mx_product: unknown epilogue %d", epi);
    if (epi != mx::EPI_NONE && N % 16) return fail("mx_product: gates and ups alternate in groups of 8, found %d rows of weights", N);
    if (out_codes == nullptr && out_dtype != JANIS_BF16 && out_dtype != JANIS_F32) return fail("mx_product: unknown dtype %d", out_dtype);
    if (K > 1 << 30) return fail("mx_product: a row has at most 2^30 values, found %d", K);
    const mx::Out o = {out, out_codes, out_scales, out_dtype, epi, limit, alpha, up_add};
    return mx::few_rows(xc, xs, wc, ws, o, T, N, mx::padded(K), g_split, g_stages, stream);
}

// The count of given-up waits copied into `host` (pinned memory, two ints, the second always 0) in the order of `stream`.
JANIS_EXPORT int janis_mx_timeouts_async(int* host, cudaStream_t stream) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(host, mx::g_timeouts, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
    if (e != cudaSuccess) return fail("mx_timeouts_async: %s", cudaGetErrorString(e));
    return 0;
}
