// Products of 8-bit rows with 4-bit weights (both in the microscaling form of mx.cuh), with float sums:
//   out[t, n] = epilogue(sum_k x[t, k] W[n, k]);  the gated epilogues take gate and up rows of W that alternate in groups of 8 and
//   give act(gate) * up, as values or as 8-bit rows for the product behind.
//
// Few rows (decode steps): bound by streaming W from HBM once.
//   * The tensor cores take both forms as they are, with their scales (tcgen05.mma kind::mxf8f6f4): no value is unpacked by a thread.
//     128 rows of W are the M side, one a lane of tensor memory; the rows of x, padded to a multiple of 16, the N side.
//   * A stage is 128 values of K: 8 KB of W (16 KB once the copy engine has spread it), the rows of x, and a block of scales of
//     each, which the thread that issues the products brings to columns of tensor memory of the stage's own.
//   * Where W has few tiles of 128 rows, a cluster of up to 8 CTAs shares K.  Each sends its sums to the CTAs that add them up, a share
//     of the rows each, in the order of the ranks: the result does not depend on timing.  The sums are counted in by an mbarrier; nobody
//     waits for anybody else at the end.
//
// Many rows (prompts): bound by the tensor cores.
//   * 128 rows of x are the M side, 128 rows of W the N side (256 and 256 of a pair of CTAs, which share one product), so that a thread of the
//     epilogue has a row of x and a run of columns: gates beside their ups, whole groups of 32 for 8-bit rows, whole sectors to store.
//   * A CTA an SM takes tile after tile.  One thread asks for the copies, one issues the products, eight warps drain: they take the sums
//     into registers at once (half of the columns each four warps), give the tensor memory back and work while the next tile is multiplied.
//
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

// gelu's tanh form as v / (1 + e^(-2 y)), y = sqrt(2 / pi) (v + 0.044715 v^3): 1 + tanh(y) is 2 / (1 + e^(-2 y)), which loses nothing where
// tanh comes near -1.  __fdividef is within 2 units in the last place here (and 0 where the divisor has passed 2^126).
__device__ __forceinline__ float gated(float gate, float up, int epi, const Out& o) {
    if (epi == EPI_GATED_CLAMP) return clamped_gate(gate, up, o.limit, o.alpha, o.up_add);
    const float y = epi == EPI_GATED_GELU ? 1.5957691216057308f * fmaf(0.044715f * gate * gate, gate, gate) : gate;
    return __fdividef(gate, 1.0f + expf(-y)) * up;
}

constexpr int TILE = 128;                      // rows of W a CTA
constexpr int A_BYTES = TILE * 128, A_PACKED = A_BYTES / 2;
constexpr int MAX_STAGES = 11;
constexpr int FEW = 64;                        // rows of x at most
constexpr int SCALE_BYTES = 2 * BLOCK_BYTES;   // of a stage: a block of W's, a block of x's
constexpr int SCALE_COLS = 8;                  // of tensor memory
constexpr int FEW_ROOM = 225 * 1024;           // of shared memory, beside what has a fixed place
constexpr int few_smem(int stages, int NP, int split) {
    return stages * (A_BYTES + NP * 128 + SCALE_BYTES) + 1024 + (split > 1 ? NP * TILE * 4 : 0);
}

// The end of a tile of few rows: sums [SPLIT][rows][128 / SPLIT] of rows of W from row0 on, by the CTA's 128 threads.
template <int SPLIT>
__device__ __forceinline__ void store_rows(const float* sums, int rows, int row0, int N, const Out& o) {
    constexpr int SHARE = TILE / SPLIT;
    const int id = threadIdx.x;
    const auto sum_at = [&](int m, int row) {                         // in the order of the ranks
        float v = sums[m * SHARE + row];
#pragma unroll
        for (int r = 1; r < SPLIT; ++r) v += sums[(r * rows + m) * SHARE + row];
        return v;
    };
    if (o.epi == EPI_NONE) {
        const int row = id % SHARE, n = row0 + row;
        if (n >= N) return;
        for (int m = id / SHARE; m < rows; m += SPLIT) {
            const float v = sum_at(m, row);
            if (o.dtype == JANIS_BF16) reinterpret_cast<bf16*>(o.values)[(size_t)m * N + n] = from_float<bf16>(v);
            else reinterpret_cast<float*>(o.values)[(size_t)m * N + n] = v;
        }
        return;
    }
    // a gate's up stands 8 rows behind it; for 8-bit rows (SHARE is 64 at least) a warp has the 32 columns of a group
    constexpr int COLS = SHARE / 2;
    const int j = id % COLS, c = row0 / 2 + j, row = j / 8 * 16 + j % 8;
    const int all = N / 2, wide = o.codes != nullptr ? padded(all) : all;
    if (c >= wide) return;                                            // (for 8-bit rows a whole warp)
    constexpr int AT_ONCE = 4, STEP = 128 / COLS;                     // rows of x whose latencies (two loads, an exponential, a quotient, shuffles) overlap
    for (int m0 = id / COLS; m0 < rows; m0 += AT_ONCE * STEP) {
        float v[AT_ONCE], big[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int m = m0 + u * STEP;
            v[u] = c < all && m < rows ? gated(sum_at(m, row), sum_at(m, row + 8), o.epi, o) : 0.f;
            big[u] = fabsf(v[u]);
        }
        if (o.codes == nullptr) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int m = m0 + u * STEP;
                if (m >= rows) break;
                if (o.dtype == JANIS_BF16) reinterpret_cast<bf16*>(o.values)[(size_t)m * all + c] = from_float<bf16>(v[u]);
                else reinterpret_cast<float*>(o.values)[(size_t)m * all + c] = v[u];
            }
            continue;
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1)
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) big[u] = larger(big[u], __shfl_xor_sync(0xffffffffu, big[u], s));
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int m = m0 + u * STEP;
            if (m >= rows) break;
            const uint32_t byte = scale_byte_e4m3(big[u]);
            o.codes[(size_t)m * wide + c] = byte == 255u ? 0 : (uint8_t)two_e4m3(v[u] * inverse_scale(byte), 0.f);
            if ((id & 31) == 0) o.scales[scale_at(m, c / BLOCK, wide / BLOCK) + c % BLOCK / GROUP] = (uint8_t)byte;
        }
    }
}

// The same for 8-bit rows where a CTA's share is half (SPLIT 4) or a quarter (SPLIT 8) of the 64 rows of W behind a group: the CTAs of a group tell
// each other their largest magnitudes, one for each row of x, counted in by `bar`.  False: they did not come.
template <int SPLIT>
__device__ __forceinline__ bool store_group_shares(const float* sums, float* largest, uint32_t bar, int rank, int rows, int row0, int N, const Out& o) {
    constexpr int SHARE = TILE / SPLIT, COLS = SHARE / 2, STEP = 128 / COLS, CTAS = 32 / COLS, MOST = FEW / STEP;
    const int id = threadIdx.x, j = id % COLS, c = row0 / 2 + j, row = j / 8 * 16 + j % 8, all = N / 2, wide = padded(all);
    const int place = rank % CTAS, first = rank - place;
    float v[MOST];
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
        const int m = id / COLS + u * STEP;
        v[u] = 0.f;
        if (m < rows && c < all) {
            float gate = sums[m * SHARE + row], up = sums[m * SHARE + row + 8];
#pragma unroll
            for (int r = 1; r < SPLIT; ++r) {                         // in the order of the ranks
                gate += sums[(r * rows + m) * SHARE + row];
                up += sums[(r * rows + m) * SHARE + row + 8];
            }
            v[u] = gated(gate, up, o.epi, o);
        }
        float big = fabsf(v[u]);
#pragma unroll
        for (int s = COLS / 2; s > 0; s >>= 1) big = larger(big, __shfl_xor_sync(0xffffffffu, big, s));
        if (m < rows && j < CTAS) {                                   // lane j tells CTA j of the group
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(largest + place * FEW + m);
            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];\n" ::"r"(in_cta(at, first + j)),
                         "r"(__float_as_uint(big)), "r"(in_cta(bar, first + j))
                         : "memory");
        }
    }
    bool there = false;
    for (int i = 0; i < 8 && !there; ++i) there = mbar_wait_cluster(bar, 0);
    if (!__syncthreads_and(there ? 1 : 0)) return false;
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
        const int m = id / COLS + u * STEP;
        if (m >= rows) break;
        float big = largest[m];
#pragma unroll
        for (int p = 1; p < CTAS; ++p) big = larger(big, largest[p * FEW + m]);
        const uint32_t byte = scale_byte_e4m3(big);
        o.codes[(size_t)m * wide + c] = byte == 255u ? 0 : (uint8_t)two_e4m3(v[u] * inverse_scale(byte), 0.f);
        if (c % GROUP == 0) o.scales[scale_at(m, c / BLOCK, wide / BLOCK) + c % BLOCK / GROUP] = (uint8_t)byte;
    }
    return true;
}

template <int SPLIT>
__global__ void __launch_bounds__(128)
few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ ws,
                const uint8_t* __restrict__ xs, const Out o, int T, int N, int kp, int NP, int stages, int tmem_cols) {
    constexpr int SHARE = TILE / SPLIT;                              // rows of the tile that this CTA adds up and stores
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * MAX_STAGES + 3];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed, asked;                                     // asked: stages that copies were asked for
    __shared__ float largest[SPLIT > 2 ? SPLIT / 2 * FEW : 1];        // of a group of 8-bit rows, by the CTAs that share it
    const int warp = threadIdx.x >> 5;
    const int rank = SPLIT > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int n0 = blockIdx.x / SPLIT * TILE;
    const int blocks = kp / BLOCK;

    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t stage0 = (raw + 1023) & ~1023u;                   // swizzle atoms want 1024-byte alignment
    const int stage_bytes = A_BYTES + NP * 128;
    const uint32_t scales0 = stage0 + stages * stage_bytes;
    // [SPLIT][T][SHARE] sums: behind the stages where others write them, over the idle stages where this CTA does
    const uint32_t sums0 = SPLIT > 1 ? scales0 + stages * SCALE_BYTES : stage0;
    float* sums = reinterpret_cast<float*>(smem_raw + (sums0 - raw));
    const uint32_t bar_full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t bar_empty = bar_full + 8 * MAX_STAGES, bar_done = bar_full + 16 * MAX_STAGES, bar_sums = bar_done + 8;
    const uint32_t bar_largest = bar_sums + 8;

    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        mbar_init(bar_done, 1);
        mbar_init(bar_sums, 1);
        mbar_init(bar_largest, 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        if (SPLIT > 1) mbar_expect_tx(bar_sums, T * TILE * 4);
        if (SPLIT > 2) mbar_expect_tx(bar_largest, SPLIT / 2 * T * 4);
    }
    if (warp == 0) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), tmem_cols);
    fence_before_sync();
    __syncthreads();
    if (SPLIT > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    fence_after_sync();
    const uint32_t tmem = tmem_slot;

    // this CTA's share of K: value blocks rank, rank + SPLIT, ...
    const int nk = (blocks - rank + SPLIT - 1) / SPLIT;
    // (a tile past W's rows, which only makes the padding of 8-bit rows, finds zeros there; their scales mean nothing, and its columns count as 0)
    const uint8_t* w_scales = ws + (size_t)min(n0 / BLOCK, (N - 1) / BLOCK) * blocks * BLOCK_BYTES;

    grid_dependents_launch();
    if (warp == 0 && elect_one()) {
        // ---- the copies.  The weights are constants of the model: the first tiles of W are on their way before this kernel
        // waits for the one that makes x.
        // W passes once: marked so, 1 x 73,728 x 4,608 takes 30.4 us instead of 32.1, 16 rows 34.6 instead of 37.3, 1 x 4,096 x 2,304 3.07 instead of 3.20.
        const int bytes = A_PACKED + NP * 128 + 2 * BLOCK_BYTES;
        const uint64_t once = read_once();
        const auto load_w = [&](int kb, int s) {
            mbar_expect_tx(bar_full + 8 * s, bytes);
            load_2d_by(stage0 + s * stage_bytes, &map_w, kb * BLOCK, n0, bar_full + 8 * s, once);
            bulk_load(scales0 + s * SCALE_BYTES, w_scales + (size_t)kb * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const auto load_x = [&](int kb, int s) {
            tma_load_2d(stage0 + s * stage_bytes + A_BYTES, &map_x, kb * BLOCK, 0, bar_full + 8 * s);
            bulk_load(scales0 + s * SCALE_BYTES + BLOCK_BYTES, xs + (size_t)kb * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const int pre = nk < stages ? nk : stages;
        for (int i = 0; i < pre; ++i) load_w(rank + i * SPLIT, i);
        grid_dependency_wait();
        for (int i = 0; i < pre; ++i) load_x(rank + i * SPLIT, i);
        int filled = pre, s = 0;
        uint32_t phase = 0;
        uint32_t free = 0;
        for (; filled < nk; ++filled) {
            if (!free && !mbar_wait(bar_empty + 8 * s, phase)) { atomicExch(&failed, 1); break; }
            const int now = s;
            if (++s == stages) { s = 0; phase ^= 1; }
            free = mbar_peek(bar_empty + 8 * s, phase);
            load_w(rank + filled * SPLIT, now);
            load_x(rank + filled * SPLIT, now);
        }
        asked = filled;
    } else if (warp == 1 && elect_one()) {
        // ---- the thread that issues the products
        grid_dependency_wait();
        int next = 0;
        uint32_t phase = 0, full = 0;
        for (int i = 0; i < nk; ++i) {
            const int s = next;
            if (!full && !mbar_wait(bar_full + 8 * s, phase)) { atomicExch(&failed, 1); break; }
            if (++next == stages) { next = 0; phase ^= 1; }
            full = mbar_peek(bar_full + 8 * next, phase);
            fence_after_sync();
            const uint32_t a = stage0 + s * stage_bytes, b = a + A_BYTES, sc = scales0 + s * SCALE_BYTES;
            const uint32_t ta = tmem + NP + s * SCALE_COLS, tb = ta + 4;
            scales_to_tmem(ta, sc);
            scales_to_tmem(tb, sc + BLOCK_BYTES);
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
        for (int j = asked > stages ? asked - stages : 0; j < asked; ++j) mbar_wait(bar_full + 8 * (j % stages), (j / stages) & 1);
    if (SPLIT > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");      // everybody's barriers are there

    // ---- sums of row (32 * warp + lane) of the tile of W, to the CTA that adds them up
    const uint32_t mine = sums0 + (uint32_t)(rank * T * SHARE + threadIdx.x % SHARE) * 4;
    uint32_t there = mine, there_bar = bar_sums;
    if (SPLIT > 1) {
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there) : "r"(mine), "r"((uint32_t)threadIdx.x / SHARE));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there_bar) : "r"(bar_sums), "r"((uint32_t)threadIdx.x / SHARE));
    }
    for (int c = 0; c < T; c += 16) {
        uint32_t r[16];
        tmem_load16(r, tmem + ((uint32_t)(warp * 32) << 16) + c);
        tmem_wait_load();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (c + j >= T) break;
            if (SPLIT > 1)
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];\n" ::"r"(there + (uint32_t)(c + j) * SHARE * 4),
                             "r"(r[j]), "r"(there_bar)
                             : "memory");
            else
                sums[(c + j) * TILE + threadIdx.x] = __uint_as_float(r[j]);
        }
    }
    fence_before_sync();
    if (SPLIT > 1) {
        // (others may be at their own waits' limits: this CTA's memory has to outlast what they send)
        bool all = false;
        for (int i = 0; i < 8 && !all; ++i) all = mbar_wait_cluster(bar_sums, 0);
        ok = ok && all;
    }
    ok = __syncthreads_and(ok ? 1 : 0);
    if (warp == 0) tmem_free(tmem, tmem_cols);
    if (!ok && threadIdx.x == 0) atomicAdd(&g_timeouts, 1);
    if constexpr (SPLIT > 2) {
        if (o.codes != nullptr) {                                     // (a CTA that gave up stays for what the others tell it)
            if (!store_group_shares<SPLIT>(sums, largest, bar_largest, rank, T, n0 + rank * SHARE, N, o) && threadIdx.x == 0) atomicAdd(&g_timeouts, 1);
            return;
        }
    }
    if (!ok) return;
    store_rows<SPLIT>(sums, T, n0 + rank * SHARE, N, o);
}

// how rows of out lie: 2 whole sectors, 1 whole 16 bytes, 0 neither
static int pieces(const Out& o, int cols) {
    const size_t row = (size_t)cols * (o.dtype == JANIS_BF16 ? 2 : 4), at = (uintptr_t)o.values;
    return ((row | at) & 31) == 0 ? 2 : ((row | at) & 15) == 0 ? 1 : 0;
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
constexpr int MANY_THREADS = 384;              // copies; products; two idle warps; two times four warps that drain
constexpr int X_BYTES = 128 * 128;
constexpr int MANY_STAGES = 6, MANY_STAGE = X_BYTES + A_BYTES, MANY_SCALES = 2 * BLOCK_BYTES;
constexpr int MANY_SMEM = MANY_STAGES * (MANY_STAGE + MANY_SCALES) + 1024;
constexpr int M_RUN = 16;                      // tiles of x that are taken with one tile of W after another

__device__ __forceinline__ void tile_at(int i, int m_tiles, int n_tiles, int& m, int& n) {
    const int run = i / (M_RUN * n_tiles), within = i - run * (M_RUN * n_tiles), height = min(M_RUN, m_tiles - run * M_RUN);
    n = within / height;
    m = run * M_RUN + within - n * height;
}

// 32 bytes of one lane: a whole sector of memory (16 bytes a lane, rows apart, write every sector twice)
__device__ __forceinline__ void store_sector(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}

// SQUARE values of each of SQUARE lanes turned: afterwards lane l has value l of each of them.  Lanes K apart exchange what the other needs, then
// K / 2 apart, ...
template <int K, int SQUARE>
__device__ __forceinline__ void turn_lanes(uint32_t* q) {
    const bool up = (threadIdx.x & K) != 0;
#pragma unroll
    for (int b = 0; b < SQUARE; b += 2 * K)
#pragma unroll
        for (int i = b; i < b + K; ++i) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? q[i] : q[i + K], K);
            q[i] = up ? got : q[i];
            q[i + K] = up ? q[i + K] : got;
        }
    if constexpr (K > 1) turn_lanes<K / 2, SQUARE>(q);
}

// Columns c .. c + COUNT - 1 of row t of out [T, cols], of which this thread has the values; a whole warp calls it, and COUNT (at most 32) lanes
// that lie together have rows that lie together.
// vec 2: rows are whole sectors, 1: whole 16 bytes, 0: neither.  Then the values are turned among the lanes first,
// so that a row's columns leave together.
template <int COUNT>
__device__ __forceinline__ void store_run(uint32_t* v, const Out& o, int t, int c, int T, int cols, int vec) {
    const size_t at = (size_t)t * cols + c;
    const int left = cols - c;
    if (vec != 0) {
        if (t >= T) return;
        if (o.dtype == JANIS_BF16) {
            bf16* p = reinterpret_cast<bf16*>(o.values) + at;
#pragma unroll
            for (int j = 0; j < COUNT; j += 8)
                if (j < left) {
                    if (COUNT % 16 == 0 && vec == 2) {
                        if (j % 16 != 0) continue;
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int k = COUNT % 16 == 0 ? j + 2 * e : 0;
                            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                            w[e] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        store_sector(p + j, w);
                    } else {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[j + e]);
                        store_eight(p + j, f);
                    }
                }
        } else {
            float* p = reinterpret_cast<float*>(o.values) + at;
#pragma unroll
            for (int j = 0; j < COUNT; j += 4)
                if (j < left) {
                    if (vec == 2) {
                        if (j % 8 == 0) store_sector(p + j, v + j);
                    } else {
                        *reinterpret_cast<uint4*>(p + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                }
        }
        return;
    }
    constexpr int SQUARE = COUNT < 32 ? COUNT : 32;
    const int mine = threadIdx.x % SQUARE, rows = T - (t - mine);
#pragma unroll
    for (int j = 0; j < COUNT; j += SQUARE) {
        turn_lanes<SQUARE / 2, SQUARE>(v + j);                        // now of rows t - mine, t - mine + 1, ..., column c + j + mine
        if (j + mine >= left) continue;
        const size_t first = (size_t)(t - mine) * cols + c + j + mine;
        if (o.dtype == JANIS_BF16) {
            bf16* p = reinterpret_cast<bf16*>(o.values) + first;
#pragma unroll
            for (int i = 0; i < SQUARE; ++i, p += cols)
                if (i < rows) *p = from_float<bf16>(__uint_as_float(v[j + i]));
        } else {
            float* p = reinterpret_cast<float*>(o.values) + first;
#pragma unroll
            for (int i = 0; i < SQUARE; ++i, p += cols)
                if (i < rows) *p = __uint_as_float(v[j + i]);
        }
    }
}

// 8-bit rows are padded with zeros of scale 1: columns from `left` on count as 0, whatever is there.  Behind W's rows the copies find zeros, but the
// scales that fill their block of 128 mean nothing, and a zero under a scale of NaN is a NaN.  (Whole warps agree on `left`; only the last tiles enter.)
template <int COUNT>
__device__ __forceinline__ void no_columns_from(uint32_t* v, int left) {
    if (left >= COUNT) return;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) v[j] = j < left ? v[j] : 0u;
}

// Holds what is made of `v` behind the arrival that gives tensor memory back: values of an asm volatile stay behind those before it.  Without it the
// compiler may move the activation in front, and the next tile's products wait for it: 2,048 rows x 18,432 x 2,304 took 82 us then, 75 with it behind.
template <int COUNT>
__device__ __forceinline__ void keep_behind(uint32_t (&v)[COUNT]) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) asm volatile("" : "+r"(v[j]));
}

// The end of a row's run of COLS columns of sums from column n0 on (rows of W), by the thread that holds them; a whole warp calls it.
template <int COLS, int EPI>
__device__ __forceinline__ void finish_run(uint32_t (&v)[COLS], const Out& o, int t, int n0, int T, int N, int vec) {
    if constexpr (EPI == EPI_NONE) {
        store_run<COLS>(v, o, t, n0, T, N, vec);
    } else {
        if (t >= T && (vec != 0 || o.codes != nullptr)) return;
        keep_behind(v);
        const int cols = N / 2, wide = o.codes != nullptr ? padded(cols) : cols, c = n0 / 2;
#pragma unroll
        for (int u = 0; u < COLS / 16; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[u * 8 + j] = __float_as_uint(gated(__uint_as_float(v[u * 16 + j]), __uint_as_float(v[u * 16 + 8 + j]), EPI, o));
        if (o.codes == nullptr) {
            store_run<COLS / 2>(v, o, t, c, T, cols, vec);
            return;
        }
        no_columns_from<COLS / 2>(v, cols - c);
#pragma unroll
        for (int g = 0; g < COLS / 64; ++g) {
            float big = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) big = larger(big, __uint_as_float(v[g * 32 + j]));
            const uint32_t byte = scale_byte_e4m3(big);
            const float inv = inverse_scale(byte);
            uint32_t q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t* p = v + g * 32 + j * 4;
                q[j] = byte == 255u ? 0u
                                    : two_e4m3(__uint_as_float(p[0]) * inv, __uint_as_float(p[1]) * inv) |
                                          two_e4m3(__uint_as_float(p[2]) * inv, __uint_as_float(p[3]) * inv) << 16;
            }
            const int cg = c + g * 32;
            if (cg < wide) {
                store_sector(o.codes + (size_t)t * wide + cg, q);
                o.scales[scale_at(t, cg / BLOCK, wide / BLOCK) + cg % BLOCK / GROUP] = (uint8_t)byte;
            }
        }
    }
}

template <int EPI>
__global__ void __launch_bounds__(MANY_THREADS, 1)
many_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ ws,
                 const uint8_t* __restrict__ xs, const Out o, int T, int N, int kp, int m_tiles, int n_tiles, int vec) {
    constexpr int COLS = 64;                                          // columns of a draining warp
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * MANY_STAGES + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed, asked;                                     // asked: stages that copies were asked for
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = kp / BLOCK, tiles = m_tiles * n_tiles;
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t stage0 = (raw + 1023) & ~1023u, scales0 = stage0 + MANY_STAGES * MANY_STAGE;
    const uint32_t bar_full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t bar_empty = bar_full + 8 * MANY_STAGES, bar_sums = bar_full + 16 * MANY_STAGES, bar_drained = bar_sums + 16;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * MANY_STAGES + 2; ++i) mbar_init(bar_full + 8 * i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(bar_drained + 8 * i, 8);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    grid_dependents_launch();

    if (warp == 0 && elect_one()) {
        const int w_last = (N - 1) / BLOCK;
        const auto load_w = [&](int s, int kb, int n) {               // (past W's rows are zeros, whose scales mean nothing: such columns count as 0)
            mbar_expect_tx(bar_full + 8 * s, X_BYTES + A_PACKED + 2 * BLOCK_BYTES);
            tma_load_2d(stage0 + s * MANY_STAGE + X_BYTES, &map_w, kb * BLOCK, n * 128, bar_full + 8 * s);
            bulk_load(scales0 + s * MANY_SCALES + BLOCK_BYTES, ws + ((size_t)min(n, w_last) * blocks + kb) * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const auto load_x = [&](int s, int kb, int m) {
            tma_load_2d(stage0 + s * MANY_STAGE, &map_x, kb * BLOCK, m * 128, bar_full + 8 * s);
            bulk_load(scales0 + s * MANY_SCALES, xs + ((size_t)m * blocks + kb) * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        // the weights are constants of the model: the first ones are on their way before x is there
        const int pre = min(MANY_STAGES, blocks);
        int m, n;
        tile_at(blockIdx.x, m_tiles, n_tiles, m, n);
        for (int i = 0; i < pre; ++i) load_w(i, i, n);
        grid_dependency_wait();
        for (int i = 0; i < pre; ++i) load_x(i, i, m);
        int filled = pre;
        int s = pre == MANY_STAGES ? 0 : pre;
        uint32_t phase = pre == MANY_STAGES ? 0 : 1, free = 0;             // (a stage that was never filled counts as free: parity 1 passes)
        bool ok = true;
        for (int i = blockIdx.x; i < tiles && ok; i += gridDim.x) {
            tile_at(i, m_tiles, n_tiles, m, n);
            for (int kb = i == blockIdx.x ? pre : 0; kb < blocks; ++kb, ++filled) {
                if (!free && !mbar_wait(bar_empty + 8 * s, phase)) { atomicExch(&failed, 1); ok = false; break; }
                const int now = s;
                if (++s == MANY_STAGES) { s = 0; phase ^= 1; }
                free = mbar_peek(bar_empty + 8 * s, phase);
                load_w(now, kb, n);
                load_x(now, kb, m);
            }
        }
        asked = filled;
    } else if (warp == 1 && elect_one()) {
        grid_dependency_wait();
        int next = 0, turn = 0;
        uint32_t phase = 0, full = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < tiles && ok; i += gridDim.x, ++turn) {
            const int b = turn & 1;
            const uint32_t d = tmem + b * 128;
            if (turn >= 2 && !mbar_wait(bar_drained + 8 * b, (turn / 2 - 1) & 1)) { atomicExch(&failed, 1); break; }
            fence_after_sync();
            for (int kb = 0; kb < blocks; ++kb) {
                const int s = next;
                if (!full && !mbar_wait(bar_full + 8 * s, phase)) { atomicExch(&failed, 1); ok = false; break; }
                if (++next == MANY_STAGES) { next = 0; phase ^= 1; }
                full = mbar_peek(bar_full + 8 * next, phase);
                fence_after_sync();
                const uint32_t x = stage0 + s * MANY_STAGE, w = x + X_BYTES, sc = scales0 + s * MANY_SCALES;
                const uint32_t tx = tmem + 256 + s * 8, tw = tx + 4;
                scales_to_tmem(tx, sc);
                scales_to_tmem(tw, sc + BLOCK_BYTES);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    umma_block(d, smem_desc(x + g * 32), smem_desc(w + g * 32), block_desc<ROWS>(128, 128, g), tx, tw, (kb > 0 || g > 0) ? 1u : 0u);
                umma_commit(bar_empty + 8 * s);
            }
            umma_commit(bar_sums + 8 * b);
            if (!ok) mbar_wait(bar_sums + 8 * b, (turn / 2) & 1);      // (no product is under way when the tensor memory goes)
        }
    } else if (warp >= 4) {
        grid_dependency_wait();
        const int half = (warp - 4) / 4, row = warp % 4 * 32 + lane;  // (a warp reaches the quarter of tensor memory that its number says)
        int turn = 0;
        for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++turn) {
            const int b = turn & 1;
            int m, n;
            tile_at(i, m_tiles, n_tiles, m, n);
            const bool there = mbar_wait_parked(bar_sums + 8 * b, (turn / 2) & 1, &failed);
            if (!__all_sync(0xffffffffu, there && *(volatile int*)&failed == 0)) { atomicExch(&failed, 1); break; }
            fence_after_sync();
            uint32_t v[COLS];
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_load32(v + c, tmem + ((uint32_t)(warp % 4 * 32) << 16) + b * 128 + half * COLS + c);
            tmem_wait_load();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_drained + 8 * b);
            finish_run<COLS, EPI>(v, o, m * 128 + row, n * 128 + half * COLS, T, N, vec);
        }
    } else {
        grid_dependency_wait();
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    if (failed != 0 && threadIdx.x == 0) {                            // no copy is under way when the CTA leaves
        atomicAdd(&g_timeouts, 1);
        for (int j = asked > MANY_STAGES ? asked - MANY_STAGES : 0; j < asked; ++j) mbar_wait(bar_full + 8 * (j % MANY_STAGES), (j / MANY_STAGES) & 1);
    }
    if (warp == 0) tmem_free(tmem, 512);
}

// ---------------------------------------------------------------------------
// many rows, two CTAs as one
// ---------------------------------------------------------------------------
constexpr int PAIR_STAGES = 6, PAIR_STAGE = X_BYTES + A_BYTES, PAIR_SCALES = 3 * BLOCK_BYTES, PAIR_COLS = 12;
constexpr int PAIR_SMEM = PAIR_STAGES * (PAIR_STAGE + PAIR_SCALES) + 1024;

// 256 rows of x by 256 of W: each SM holds half of both, so that it fetches and reads two thirds of what a tile of 128 x 256 wants for the same
// products, and its sums are 128 rows of 256 columns.  At prompts' sizes the products are bound by the power limit (1.1 to 1.5 GHz), so that what
// a tile does not fetch counts: 2,048 rows x 4,608 x 36,864 254 us, against 274 with tiles of 128 x 256 of one SM and 333 of 128 x 128.
// (Without a gate the 128 columns of a thread and what it stores them by spill 84 bytes.)
// Tensor memory holds one tile's sums, and the products wait some 2 us while they are taken out.  Tiles of 256 x 192, of which it holds two, close
// that gap and are no faster: 2,048 x 18,432 x 2,304 gated 74.5 us against 73.4, 2,048 x 4,608 x 36,864 281 against 255.
template <int EPI>
__global__ void __launch_bounds__(MANY_THREADS, 1)
pair_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_ws,
                 const __grid_constant__ CUtensorMap map_xs, const Out o, int T, int N, int kp, int m_tiles, int n_tiles, int vec) {
    constexpr int COLS = 128;                                         // columns of a draining warp
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * PAIR_STAGES + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cg::this_cluster().block_rank();
    const int blocks = kp / BLOCK, tiles = m_tiles * n_tiles, first = blockIdx.x / 2, step = gridDim.x / 2;
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t stage0 = (raw + 1023) & ~1023u, scales0 = stage0 + PAIR_STAGES * PAIR_STAGE;
    const uint32_t bar_full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t bar_empty = bar_full + 8 * PAIR_STAGES, bar_sums = bar_full + 16 * PAIR_STAGES, bar_drained = bar_sums + 8;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * PAIR_STAGES + 1; ++i) mbar_init(bar_full + 8 * i, 1);
        mbar_init(bar_drained, 16);                                   // the draining warps of both
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) pair_tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), 512);
    fence_before_sync();
    __syncthreads();
    cg::this_cluster().sync();                                        // the barriers of both are there
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    grid_dependents_launch();

    if (warp == 0 && elect_one()) {
        // ---- the copies of this CTA's half, counted in by the first CTA's barriers
        const uint32_t full = in_cta(bar_full, 0);
        const auto load_w = [&](int s, int kb, int n) {
            if (rank == 0) mbar_expect_tx(bar_full + 8 * s, 2 * (X_BYTES + A_PACKED + 3 * BLOCK_BYTES));
            pair_load_2d(stage0 + s * PAIR_STAGE + X_BYTES, &map_w, kb * BLOCK, n * 256 + (int)rank * 128, full + 8 * s);
            pair_load_3d(scales0 + s * PAIR_SCALES + BLOCK_BYTES, &map_ws, 0, kb * 2, n * 2, full + 8 * s);
        };
        const auto load_x = [&](int s, int kb, int m) {
            pair_load_2d(stage0 + s * PAIR_STAGE, &map_x, kb * BLOCK, m * 256 + (int)rank * 128, full + 8 * s);
            pair_load_3d(scales0 + s * PAIR_SCALES, &map_xs, 0, kb * 2, m * 2 + (int)rank, full + 8 * s);
        };
        const int pre = min(PAIR_STAGES, blocks);
        int m, n;
        tile_at(first, m_tiles, n_tiles, m, n);
        for (int i = 0; i < pre; ++i) load_w(i, i, n);
        grid_dependency_wait();
        for (int i = 0; i < pre; ++i) load_x(i, i, m);
        int s = pre == PAIR_STAGES ? 0 : pre;
        uint32_t phase = pre == PAIR_STAGES ? 0 : 1, free = 0;        // (a stage that was never filled counts as free: parity 1 passes)
        bool ok = true;
        for (int i = first; i < tiles && ok; i += step) {
            tile_at(i, m_tiles, n_tiles, m, n);
            for (int kb = i == first ? pre : 0; kb < blocks; ++kb) {
                if (!free && !mbar_wait(bar_empty + 8 * s, phase)) { atomicExch(&failed, 1); ok = false; break; }
                const int now = s;
                if (++s == PAIR_STAGES) { s = 0; phase ^= 1; }
                free = mbar_peek(bar_empty + 8 * s, phase);
                load_w(now, kb, n);
                load_x(now, kb, m);
            }
        }
    } else if (warp == 1 && rank == 0 && elect_one()) {
        grid_dependency_wait();
        int next = 0, turn = 0;
        uint32_t phase = 0, full = 0;
        bool ok = true;
        for (int i = first; i < tiles && ok; i += step, ++turn) {
            if (turn > 0 && !mbar_wait_cluster(bar_drained, (turn - 1) & 1)) { atomicExch(&failed, 1); break; }
            fence_after_sync();
            for (int kb = 0; kb < blocks; ++kb) {
                const int s = next;
                if (!full && !mbar_wait(bar_full + 8 * s, phase)) { atomicExch(&failed, 1); ok = false; break; }
                if (++next == PAIR_STAGES) { next = 0; phase ^= 1; }
                full = mbar_peek(bar_full + 8 * next, phase);
                fence_after_sync();
                const uint32_t x = stage0 + s * PAIR_STAGE, w = x + X_BYTES, sc = scales0 + s * PAIR_SCALES;
                const uint32_t tx = tmem + 256 + s * PAIR_COLS, tw = tx + 4;
                pair_scales_to_tmem(tx, sc);
                pair_scales_to_tmem(tw, sc + BLOCK_BYTES);
                pair_scales_to_tmem(tw + 4, sc + 2 * BLOCK_BYTES);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    pair_umma_block(tmem, smem_desc(x + g * 32), smem_desc(w + g * 32), block_desc<mx::ROWS>(256, 256, g), tx, tw, (kb > 0 || g > 0) ? 1u : 0u);
                pair_commit(bar_empty + 8 * s);
            }
            pair_commit(bar_sums);
            if (!ok) mbar_wait(bar_sums, turn & 1);                   // (no product is under way when the tensor memory goes)
        }
    } else if (warp >= 4) {
        grid_dependency_wait();
        const int half = (warp - 4) / 4, row = warp % 4 * 32 + lane;
        const uint32_t drained = in_cta(bar_drained, 0);
        int turn = 0;
        for (int i = first; i < tiles; i += step, ++turn) {
            int m, n;
            tile_at(i, m_tiles, n_tiles, m, n);
            const bool there = mbar_wait_parked(bar_sums, turn & 1, &failed);
            if (!__all_sync(0xffffffffu, there && *(volatile int*)&failed == 0)) { atomicExch(&failed, 1); break; }
            fence_after_sync();
            uint32_t v[COLS];
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_load32(v + c, tmem + ((uint32_t)(warp % 4 * 32) << 16) + half * COLS + c);
            tmem_wait_load();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_there(drained);
            finish_run<COLS, EPI>(v, o, m * 256 + (int)rank * 128 + row, n * 256 + half * COLS, T, N, vec);
        }
    } else {
        grid_dependency_wait();
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    if (failed != 0) {                                                // what is still under way for either CTA ends in microseconds: it waits for milliseconds
        if (threadIdx.x == 0) atomicAdd(&g_timeouts, 1);
        for (int i = 0; i < 1000; ++i) __nanosleep(10000);
    }
    cg::this_cluster().sync();                                        // neither leaves while the other's products or copies need it
    if (warp == 0) pair_tmem_free(tmem, 512);
}

// ---------------------------------------------------------------------------
// many rows of which there are not enough tiles for the SMs: a cluster shares K
// ---------------------------------------------------------------------------
constexpr int SHARED_STAGES = 5, SHARED_STAGE = X_BYTES + A_BYTES, SHARED_SCALES = 2 * BLOCK_BYTES;
constexpr int shared_smem(int split) { return SHARED_STAGES * (SHARED_STAGE + SHARED_SCALES) + 128 * 128 * 4 / split * (split - 1) + 1024; }

// where the sum for (row, column) stands among those that another CTA sent, or this one's own (place 0, over the idle stages): rows lie together,
// since the 32 lanes that send have a row each
template <int SPLIT>
__device__ __forceinline__ int sums_at(int place, int row, int c) {
    return (place * 128 + c) * (128 / SPLIT) + row;
}

template <int SPLIT, int EPI>
__global__ void __launch_bounds__(MANY_THREADS, 1)
shared_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ ws,
                   const uint8_t* __restrict__ xs, const Out o, int T, int N, int kp, int m_tiles, int vec) {
    constexpr int ROWS = 128 / SPLIT, RUN = 64 / SPLIT;               // rows that a CTA adds up; columns of a row that a thread does
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * SHARED_STAGES + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed, asked;
    __shared__ float largest[EPI == EPI_NONE ? 1 : 256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cg::this_cluster().block_rank(), tile = blockIdx.x / SPLIT, m = tile % m_tiles, n = tile / m_tiles;
    const int blocks = kp / BLOCK, nk = (blocks - rank + SPLIT - 1) / SPLIT;
    const int rows = min(T - m * 128, 128), mine = min(max(rows - rank * ROWS, 0), ROWS);
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t stage0 = (raw + 1023) & ~1023u, scales0 = stage0 + SHARED_STAGES * SHARED_STAGE, sums0 = scales0 + SHARED_STAGES * SHARED_SCALES;
    const uint32_t bar_full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t bar_empty = bar_full + 8 * SHARED_STAGES, bar_done = bar_full + 16 * SHARED_STAGES, bar_sums = bar_done + 8;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * SHARED_STAGES + 2; ++i) mbar_init(bar_full + 8 * i, 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        mbar_expect_tx(bar_sums, (SPLIT - 1) * mine * 512);
    }
    if (warp == 0) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), 256);
    fence_before_sync();
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    grid_dependents_launch();

    if (warp == 0 && elect_one()) {
        const uint8_t* w_scales = ws + (size_t)min(n, (N - 1) / BLOCK) * blocks * BLOCK_BYTES;
        const uint8_t* x_scales = xs + (size_t)m * blocks * BLOCK_BYTES;
        const auto load_w = [&](int kb, int s) {
            mbar_expect_tx(bar_full + 8 * s, X_BYTES + A_PACKED + 2 * BLOCK_BYTES);
            tma_load_2d(stage0 + s * SHARED_STAGE + X_BYTES, &map_w, kb * BLOCK, n * 128, bar_full + 8 * s);
            bulk_load(scales0 + s * SHARED_SCALES + BLOCK_BYTES, w_scales + (size_t)kb * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const auto load_x = [&](int kb, int s) {
            tma_load_2d(stage0 + s * SHARED_STAGE, &map_x, kb * BLOCK, m * 128, bar_full + 8 * s);
            bulk_load(scales0 + s * SHARED_SCALES, x_scales + (size_t)kb * BLOCK_BYTES, BLOCK_BYTES, bar_full + 8 * s);
        };
        const int pre = min(SHARED_STAGES, nk);
        for (int i = 0; i < pre; ++i) load_w(rank + i * SPLIT, i);
        grid_dependency_wait();
        for (int i = 0; i < pre; ++i) load_x(rank + i * SPLIT, i);
        int filled = pre;
        uint32_t free = 0;
        for (; filled < nk; ++filled) {
            const int s = filled % SHARED_STAGES, then = filled + 1;
            if (!free && !mbar_wait(bar_empty + 8 * s, (filled / SHARED_STAGES - 1) & 1)) { atomicExch(&failed, 1); break; }
            free = mbar_peek(bar_empty + 8 * (then % SHARED_STAGES), (then / SHARED_STAGES - 1) & 1);
            load_w(rank + filled * SPLIT, s);
            load_x(rank + filled * SPLIT, s);
        }
        asked = filled;
    } else if (warp == 1 && elect_one()) {
        grid_dependency_wait();
        uint32_t full = 0;
        for (int i = 0; i < nk; ++i) {
            const int s = i % SHARED_STAGES;
            if (!full && !mbar_wait(bar_full + 8 * s, (i / SHARED_STAGES) & 1)) { atomicExch(&failed, 1); break; }
            full = mbar_peek(bar_full + 8 * ((i + 1) % SHARED_STAGES), ((i + 1) / SHARED_STAGES) & 1);
            fence_after_sync();
            const uint32_t x = stage0 + s * SHARED_STAGE, w = x + X_BYTES, sc = scales0 + s * SHARED_SCALES, tx = tmem + 128 + s * 8, tw = tx + 4;
            scales_to_tmem(tx, sc);
            scales_to_tmem(tw, sc + BLOCK_BYTES);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                umma_block(tmem, smem_desc(x + g * 32), smem_desc(w + g * 32), block_desc<mx::ROWS>(128, 128, g), tx, tw, (i > 0 || g > 0) ? 1u : 0u);
            umma_commit(bar_empty + 8 * s);
        }
        umma_commit(bar_done);
    } else {
        grid_dependency_wait();
    }
    __syncwarp();
    bool ok = mbar_wait_parked(bar_done, 0, &failed);
    ok = __syncthreads_and(ok ? 1 : 0) && failed == 0;
    fence_after_sync();
    if (!ok && threadIdx.x == 0)                                      // no copy is under way when the CTA leaves
        for (int j = asked > SHARED_STAGES ? asked - SHARED_STAGES : 0; j < asked; ++j)
            mbar_wait(bar_full + 8 * (j % SHARED_STAGES), (j / SHARED_STAGES) & 1);
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");      // everybody's barriers are there

    float* own = reinterpret_cast<float*>(smem_raw + (stage0 - raw));
    if (warp >= 4) {
        const int half = (warp - 4) / 4, row = warp % 4 * 32 + lane, owner = row / ROWS;
        uint32_t there, there_bar;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there) : "r"(sums0), "r"((uint32_t)owner));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there_bar) : "r"(bar_sums), "r"((uint32_t)owner));
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
            uint32_t v[32];
            tmem_load32(v, tmem + ((uint32_t)(warp % 4 * 32) << 16) + half * 64 + c);
            tmem_wait_load();
            if (owner == rank) {
#pragma unroll
                for (int j = 0; j < 32; ++j) own[sums_at<SPLIT>(0, row % ROWS, half * 64 + c + j)] = __uint_as_float(v[j]);
            } else if (row < rows) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];\n" ::"r"(
                                     there + 4 * (uint32_t)sums_at<SPLIT>(rank - (rank > owner), row % ROWS, half * 64 + c + j)),
                                 "r"(v[j]), "r"(there_bar)
                                 : "memory");
            }
        }
    }
    fence_before_sync();
    {
        // (others may be at their own waits' limits: this CTA's memory has to outlast what they send)
        bool all = false;
        for (int i = 0; i < 8 && !all; ++i) all = mbar_wait_cluster(bar_sums, 0);
        ok = ok && all;
    }
    ok = __syncthreads_and(ok ? 1 : 0);
    if (warp == 0) tmem_free(tmem, 256);
    if (!ok) {
        if (threadIdx.x == 0) atomicAdd(&g_timeouts, 1);
        return;
    }
    if (warp < 4) return;
    // ---- a run of one row's columns, added up in the order of the ranks; a warp has 32 rows of the same run (or 16 of two)
    const int id = threadIdx.x - 128, row = id % ROWS, run = id / ROWS, c0 = run * RUN, t = m * 128 + rank * ROWS + row;
    const bool live = row < mine;
    const float* sums = reinterpret_cast<const float*>(smem_raw + (sums0 - raw));
    uint32_t v[RUN];
#pragma unroll
    for (int c = 0; c < RUN; ++c) {
        float f = 0.f;
#pragma unroll
        for (int r = 0; r < SPLIT; ++r) f += r == rank ? own[sums_at<SPLIT>(0, row, c0 + c)] : sums[sums_at<SPLIT>(r - (r > rank), row, c0 + c)];
        v[c] = __float_as_uint(f);
    }
    if (EPI == EPI_NONE) {
        store_run<RUN>(v, o, t, n * 128 + c0, T, N, vec);
        return;
    }
    if constexpr (EPI != EPI_NONE && RUN >= 16) {
        const int cols = N / 2, wide = o.codes != nullptr ? padded(cols) : cols, c = (n * 128 + c0) / 2;
#pragma unroll
        for (int u = 0; u < RUN / 16; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[u * 8 + j] = __float_as_uint(gated(__uint_as_float(v[u * 16 + j]), __uint_as_float(v[u * 16 + 8 + j]), EPI, o));
        if (o.codes == nullptr) {
            store_run<RUN / 2>(v, o, t, c, T, cols, vec);
            return;
        }
        constexpr int HELD = RUN / 2, RUNS = 32 / HELD;               // columns of a thread: 16 or 8 of a group of 32, the others in other warps
        no_columns_from<HELD>(v, cols - c);
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < HELD; ++j) big = larger(big, __uint_as_float(v[j]));
        largest[id] = big;
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
#pragma unroll
        for (int j = 0; j < RUNS; ++j) big = larger(big, largest[(run / RUNS * RUNS + j) * ROWS + row]);
        const uint32_t byte = scale_byte_e4m3(big);
        const float inv = inverse_scale(byte);
        if (!live || c >= wide) return;
#pragma unroll
        for (int j = 0; j < HELD; j += 4) {
            const uint32_t q = byte == 255u ? 0u
                                            : two_e4m3(__uint_as_float(v[j]) * inv, __uint_as_float(v[j + 1]) * inv) |
                                                  two_e4m3(__uint_as_float(v[j + 2]) * inv, __uint_as_float(v[j + 3]) * inv) << 16;
            *reinterpret_cast<uint32_t*>(o.codes + (size_t)t * wide + c + j) = q;
        }
        if (c % GROUP == 0) o.scales[scale_at(t, c / BLOCK, wide / BLOCK) + c % BLOCK / GROUP] = (uint8_t)byte;
    }
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
    if (T > FEW) return fail("mx_product: at most %d rows in this kernel, found %d", FEW, T);
    const int NP = (T + 15) / 16 * 16;
    // (8-bit rows are padded to whole blocks of 128 columns: 256 rows of gates and ups)
    const int tiles = o.codes != nullptr ? padded(N / 2) / (TILE / 2) : (N + TILE - 1) / TILE, blocks = kp / BLOCK;
    if (split == 0) {
        // K is shared while all CTAs are resident, two an SM, and keep four blocks each.  A cluster lies within a GPC, of whose 16 to 18
        // SMs four clusters of 8 take all: 32 in all, or 48 of three CTAs an SM, which pay where K is long only.  One row, us with 1, 2, 4,
        // 8 CTAs: 2,304 x 2,048 5.3, 3.6, 2.9, 3.3; 4,096 x 2,304 5.8, 3.8, 3.4, 4.2; 2,304 x 9,216 18, 10, 6.4, 4.8; 18,432 x 2,304 7.2, 6.1;
        // 4,608 x 4,096 -, -, 4.4, 4.8 (36 tiles); 4,608 x 36,864 66, 34, 22, 20 (36 tiles).
        split = 1;
        while (split < 8 && tiles * split * 2 <= 2 * sm_count() && blocks >= split * 2 * 4 && (split < 4 || tiles <= 32)) split *= 2;
        if (split == 4 && NP <= 32 && tiles > 32 && tiles <= 48 && blocks >= 128) split = 8;
    }
    if (split > 8 || split > blocks || (split & (split - 1)) != 0) return fail("mx_product: a split of %d is not possible here", split);
    const int most = FEW_ROOM;
    if (stages == 0) {
        // a ring as deep as the SM's memory allows for the CTAs that share it
        const int room = split == 8 && NP <= 32 && tiles > 32 ? 74 * 1024 : split > 1 || tiles > sm_count() ? 113 * 1024 : most;
        stages = (room - 1024 - (split > 1 ? NP * TILE * 4 : 0)) / (A_BYTES + NP * 128 + SCALE_BYTES);
        const int share = (blocks + split - 1) / split;
        if (stages > share) stages = share;
        if (stages > MAX_STAGES) stages = MAX_STAGES;
        while (split == 1 && stages * (A_BYTES + NP * 128) < NP * TILE * 4) ++stages;      // (the sums leave through them)
    }
    if (stages < 1 || stages > MAX_STAGES || few_smem(stages, NP, split) > most || (split == 1 && stages * (A_BYTES + NP * 128) < NP * TILE * 4))
        return fail("mx_product: %d stages of %d rows do not fit", stages, NP);
    int cols = 32;
    while (cols < NP + stages * SCALE_COLS) cols *= 2;
    CUtensorMap mw, mx;
    if (!make_map(&mw, WEIGHTS, wc, N, kp, TILE) || !make_map(&mx, ROWS, xc, T, kp, NP))
        return fail("mx_product: cuTensorMapEncodeTiled is not available or refused the operands");
    const auto kernel = split == 1 ? few_rows_kernel<1> : split == 2 ? few_rows_kernel<2> : split == 4 ? few_rows_kernel<4> : few_rows_kernel<8>;
    static std::once_flag once;
    static cudaError_t e = cudaSuccess;
    std::call_once(once, [] {
        for (const auto k : {few_rows_kernel<1>, few_rows_kernel<2>, few_rows_kernel<4>, few_rows_kernel<8>})
            if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_ROOM);
    });
    if (e != cudaSuccess) return fail("mx_product: shared memory refused: %s", cudaGetErrorString(e));
    return launch_kernel("mx_product", kernel, dim3(tiles * split), dim3(128), few_smem(stages, NP, split), stream, split, mw, mx, ws, xs, o,
                         T, N, kp, NP, stages, cols);
}

template <int EPI>
static int many_rows_as(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                        cudaStream_t stream) {
    const int m_tiles = (T + 127) / 128, n_tiles = o.codes != nullptr ? padded(N / 2) / 64 : (N + 127) / 128;
    if ((long long)m_tiles * n_tiles > 1 << 30) return fail("mx_product: too many tiles");
    const int vec = pieces(o, EPI == EPI_NONE ? N : N / 2);
    CUtensorMap mw, mx;
    if (!make_map(&mw, WEIGHTS, wc, N, kp, 128) || !make_map(&mx, ROWS, xc, T, kp, 128))
        return fail("mx_product: cuTensorMapEncodeTiled is not available or refused the operands");
    static std::once_flag once;
    static cudaError_t e = cudaSuccess;
    std::call_once(once, [] { e = cudaFuncSetAttribute(many_rows_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, MANY_SMEM); });
    if (e != cudaSuccess) return fail("mx_product: shared memory refused: %s", cudaGetErrorString(e));
    const int tiles = m_tiles * n_tiles;
    return launch_kernel("mx_product", many_rows_kernel<EPI>, dim3(tiles < sm_count() ? tiles : sm_count()), dim3(MANY_THREADS), MANY_SMEM,
                         stream, 1, mw, mx, ws, xs, o, T, N, kp, m_tiles, n_tiles, vec);
}

template <int EPI>
static int pair_rows_as(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                        cudaStream_t stream) {
    const int m_tiles = (T + 255) / 256, n_tiles = o.codes != nullptr ? padded(N / 2) / 128 : (N + 255) / 256;
    if ((long long)m_tiles * n_tiles > 1 << 30) return fail("mx_product: too many tiles");
    const int vec = pieces(o, EPI == EPI_NONE ? N : N / 2);
    CUtensorMap mw, mx, mws, mxs;
    if (!make_map(&mw, WEIGHTS, wc, N, kp, 128) || !make_map(&mx, ROWS, xc, T, kp, 128) ||
        !make_scales_map(&mws, ws, (N + 127) / 128, kp / BLOCK, 2) || !make_scales_map(&mxs, xs, (T + 127) / 128, kp / BLOCK, 1))
        return fail("mx_product: cuTensorMapEncodeTiled is not available or refused the operands");
    static std::once_flag once;
    static cudaError_t e = cudaSuccess;
    std::call_once(once, [] { e = cudaFuncSetAttribute(pair_rows_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM); });
    if (e != cudaSuccess) return fail("mx_product: shared memory refused: %s", cudaGetErrorString(e));
    const int tiles = m_tiles * n_tiles, pairs = sm_count() / 2;
    return launch_kernel("mx_product", pair_rows_kernel<EPI>, dim3(2 * (tiles < pairs ? tiles : pairs)), dim3(MANY_THREADS), PAIR_SMEM, stream, 2, mw, mx,
                         mws, mxs, o, T, N, kp, m_tiles, n_tiles, vec);
}

static int pair_rows(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp, cudaStream_t stream) {
    if (o.epi == EPI_NONE) return pair_rows_as<EPI_NONE>(xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_GELU) return pair_rows_as<EPI_GATED_GELU>(xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_SILU) return pair_rows_as<EPI_GATED_SILU>(xc, xs, wc, ws, o, T, N, kp, stream);
    return pair_rows_as<EPI_GATED_CLAMP>(xc, xs, wc, ws, o, T, N, kp, stream);
}

template <int SPLIT, int EPI>
static int shared_rows_as(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                          cudaStream_t stream) {
    const int m_tiles = (T + 127) / 128, n_tiles = o.codes != nullptr ? padded(N / 2) / 64 : (N + 127) / 128;
    const int vec = pieces(o, EPI == EPI_NONE ? N : N / 2);
    CUtensorMap mw, mx;
    if (!make_map(&mw, WEIGHTS, wc, N, kp, 128) || !make_map(&mx, ROWS, xc, T, kp, 128))
        return fail("mx_product: cuTensorMapEncodeTiled is not available or refused the operands");
    static std::once_flag once;
    static cudaError_t e = cudaSuccess;
    std::call_once(once, [] { e = cudaFuncSetAttribute(shared_rows_kernel<SPLIT, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_smem(SPLIT)); });
    if (e != cudaSuccess) return fail("mx_product: shared memory refused: %s", cudaGetErrorString(e));
    return launch_kernel("mx_product", shared_rows_kernel<SPLIT, EPI>, dim3(m_tiles * n_tiles * SPLIT), dim3(MANY_THREADS), shared_smem(SPLIT), stream, SPLIT,
                         mw, mx, ws, xs, o, T, N, kp, m_tiles, vec);
}

template <int EPI>
static int shared_rows_by(int split, const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                          cudaStream_t stream) {
    if (split > kp / BLOCK) return fail("mx_product: a split of %d is not possible here", split);
    if (split == 2) return shared_rows_as<2, EPI>(xc, xs, wc, ws, o, T, N, kp, stream);
    if (split == 4) return shared_rows_as<4, EPI>(xc, xs, wc, ws, o, T, N, kp, stream);
    if constexpr (EPI == EPI_NONE)
        if (split == 8) return shared_rows_as<8, EPI>(xc, xs, wc, ws, o, T, N, kp, stream);
    return fail("mx_product: a split of %d is not possible here", split);
}

static int shared_rows(int split, const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                       cudaStream_t stream) {
    if (o.epi == EPI_NONE) return shared_rows_by<EPI_NONE>(split, xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_GELU) return shared_rows_by<EPI_GATED_GELU>(split, xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_SILU) return shared_rows_by<EPI_GATED_SILU>(split, xc, xs, wc, ws, o, T, N, kp, stream);
    return shared_rows_by<EPI_GATED_CLAMP>(split, xc, xs, wc, ws, o, T, N, kp, stream);
}

// How many clusters of `split` CTAs of the kernel that shares K the GPU holds at once (a cluster lies within a GPC).
template <int SPLIT>
static int clusters_held() {
    static int n = -1;
    static std::once_flag once;
    std::call_once(once, [] {
        cudaFuncSetAttribute(shared_rows_kernel<SPLIT, EPI_NONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_smem(SPLIT));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(SPLIT * 16);
        cfg.blockDim = dim3(MANY_THREADS);
        cfg.dynamicSmemBytes = shared_smem(SPLIT);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = SPLIT;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, shared_rows_kernel<SPLIT, EPI_NONE>, &cfg) != cudaSuccess) {
            n = 0;
            cudaGetLastError();
        }
    });
    return n;
}

// The kernel of a product: 1 few rows, 2 and 3 many by pairs of CTAs and by one, 5, 6, 7 many whose K is shared by 2, 4, 8 CTAs.
// Up to 64 rows the first (32 with a gated epilogue, which is the longer the more rows a thread has: 64 rows x 28,672 x 3,584 27.5 us against 17.4),
// but where K is short (at 777, 1,000 weights and 32 rows 3.6 us against 3.1) or W alone fills the SMs (64 rows x 18,432 x 2,304: 9.0 against 7.8).
// Above, the least of what they take in us, as measured: a wave of tiles costs 0.22 a block of K and 1.2 by one CTA, 0.30 and 2.3 by pairs (of twice
// the rows and columns), and 1.5 and 2.5 once; sharing costs 0.28 a block and 4.2, as long as all clusters are resident.  So measured, by one CTA
// and by pairs: 128 rows x 18,432 x 2,304 9.0, 12.9 us; 256 rows 14.0, 13.2; 2,048 rows 92.8, 77.0.  Rows of out that start anywhere add 1.9, 4.5 and
// 0.5 once (128 rows x 777 x 1,000: 4.3 -> 6.2 by one CTA, 4.6 -> 4.9 by four that share).
static int choose(int T, int N, int blocks, const Out& o) {
    const int sms = sm_count(), m_tiles = (T + 127) / 128;
    const long long tiles128 = (long long)m_tiles * ((N + 127) / 128), pairs = (long long)((T + 255) / 256) * ((N + 255) / 256);
    const bool anywhere = o.codes == nullptr && pieces(o, o.epi == EPI_NONE ? N : N / 2) == 0;
    if (T <= 16 || (T <= (o.epi == EPI_NONE ? 64 : 32) && (blocks > 8 || anywhere) && !(T > 48 && tiles128 * 8 >= sms * 7))) return 1;
    const double cost_one = (tiles128 + sms - 1) / sms * (0.22 * blocks + 1.2) + (anywhere ? 3.4 : 1.5);
    const double cost_pair = (pairs + sms / 2 - 1) / (sms / 2) * (0.30 * blocks + 2.3) + (anywhere ? 7.0 : 2.5);
    int best = cost_one <= cost_pair ? 3 : 2;
    double least = cost_one <= cost_pair ? cost_one : cost_pair;
    const int held[3] = {tiles128 <= sms / 2 ? clusters_held<2>() : 0, tiles128 <= sms / 4 ? clusters_held<4>() : 0,
                         tiles128 <= sms / 8 && o.epi == EPI_NONE ? clusters_held<8>() : 0};
    for (int i = 0; i < 3; ++i) {
        const int split = 2 << i;
        const double cost = 0.28 * ((blocks + split - 1) / split) + (anywhere ? 4.7 : 4.2);
        if (tiles128 <= held[i] && blocks >= 2 * split && cost < least) {
            best = 5 + i;
            least = cost;
        }
    }
    return best;
}

static int many_rows(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& o, int T, int N, int kp,
                     cudaStream_t stream) {
    if (o.epi == EPI_NONE) return many_rows_as<EPI_NONE>(xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_GELU) return many_rows_as<EPI_GATED_GELU>(xc, xs, wc, ws, o, T, N, kp, stream);
    if (o.epi == EPI_GATED_SILU) return many_rows_as<EPI_GATED_SILU>(xc, xs, wc, ws, o, T, N, kp, stream);
    return many_rows_as<EPI_GATED_CLAMP>(xc, xs, wc, ws, o, T, N, kp, stream);
}

}  // namespace mx
}  // namespace janis

using namespace janis;

static int g_kernel = 0;

// Fixes the kernel of products: 0 chosen, 1 that of few rows, 2 and 3 those of many by pairs of CTAs and by one, 4 that of many whose K is shared by the
// CTAs of janis_mx_set_few, 5, 6 and 7 the same by 2, 4 and 8.  For tests and tuning.
JANIS_EXPORT void janis_mx_set_kernel(int kernel) { g_kernel = kernel; }

static int g_split = 0, g_stages = 0;

// Fixes the CTAs that share K (1, 2, 4, 8) and the depth of the ring of stages (0: chosen).  For tests and tuning.
JANIS_EXPORT void janis_mx_set_few(int split, int stages) {
    g_split = split;
    g_stages = stages;
}

// x: codes [T, padded K], W: codes [N, padded K / 2]; out [T, N] (N / 2 with a gated epilogue) of out_dtype, or 8-bit rows
// The arguments come as one block of 8-byte fields.
struct ProductArgs {
    const uint8_t *xc, *xs, *wc, *ws;
    void* out;
    long long out_dtype;
    uint8_t *out_codes, *out_scales;
    long long T, N, K, epi;
    double limit, alpha, up_add;
    cudaStream_t stream;
};
JANIS_EXPORT int janis_mx_product(const void* block) {
    ProductArgs a;
    memcpy(&a, block, sizeof(a));
    const uint8_t *xc = a.xc, *xs = a.xs, *wc = a.wc, *ws = a.ws;
    void* out = a.out;
    uint8_t *out_codes = a.out_codes, *out_scales = a.out_scales;
    if (a.T > 1 << 30 || a.N > 1 << 30 || a.K > 1 << 30) return fail("mx_product: sizes pass 2^30");
    const int out_dtype = (int)a.out_dtype, T = (int)a.T, N = (int)a.N, K = (int)a.K, epi = (int)a.epi;
    const float limit = (float)a.limit, alpha = (float)a.alpha, up_add = (float)a.up_add;
    cudaStream_t stream = a.stream;
    if (T <= 0 || N <= 0) return 0;
    if (K <= 0) return fail("mx_product: a row has no values");
    if (epi != mx::EPI_NONE && epi != mx::EPI_GATED_GELU && epi != mx::EPI_GATED_SILU && epi != mx::EPI_GATED_CLAMP)
        return fail("mx_product: unknown epilogue %d", epi);
    if (epi != mx::EPI_NONE && N % 16) return fail("mx_product: gates and ups alternate in groups of 8, found %d rows of weights", N);
    if (out_codes == nullptr && out_dtype != JANIS_BF16 && out_dtype != JANIS_F32) return fail("mx_product: unknown dtype %d", out_dtype);
    const mx::Out o = {out, out_codes, out_scales, out_dtype, epi, limit, alpha, up_add};
    const int kp = mx::padded(K);
    const int kernel = g_kernel != 0 ? g_kernel : mx::choose(T, N, kp / mx::BLOCK, o);
    if (kernel == 1) return mx::few_rows(xc, xs, wc, ws, o, T, N, kp, g_split, g_stages, stream);
    if (kernel == 2) return mx::pair_rows(xc, xs, wc, ws, o, T, N, kp, stream);
    if (kernel == 3) return mx::many_rows(xc, xs, wc, ws, o, T, N, kp, stream);
    return mx::shared_rows(kernel > 4 ? 1 << (kernel - 4) : g_split > 1 ? g_split : 2, xc, xs, wc, ws, o, T, N, kp, stream);
}

// The count of given-up waits copied into `host` (pinned memory, one int) in the order of `stream`.
JANIS_EXPORT int janis_mx_timeouts_async(int* host, cudaStream_t stream) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(host, mx::g_timeouts, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
    if (e != cudaSuccess) return fail("mx_timeouts_async: %s", cudaGetErrorString(e));
    return 0;
}
