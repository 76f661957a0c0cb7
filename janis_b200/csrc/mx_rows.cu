// Rows in and out of the 8-bit microscaling form (mx.cuh): the norms and the gated activation that leave it for the products
// behind them, plain rows, the weights' 4-bit form at load, and the values that either form stands for.
#include <type_traits>

#include "mx.cuh"

namespace janis {
namespace mx {

// The 32 values of a group, one a lane: its codes and its scale.
__device__ __forceinline__ void store_group(float v, uint8_t* codes, uint8_t* scales, int r, int g, int groups, int kp) {
    float big = fabsf(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = larger(big, __shfl_xor_sync(0xffffffffu, big, o));
    const uint32_t byte = scale_byte_e4m3(big);
    const int lane = threadIdx.x & 31;
    codes[(size_t)r * kp + g * GROUP + lane] = byte == 255u ? 0 : (uint8_t)two_e4m3(v * inverse_scale(byte), 0.f);
    if (lane == 0) scales[scale_at(r, g / 4, groups / 4) + g % 4] = (uint8_t)byte;
}

// ---------------------------------------------------------------------------
// h[r] += norm(res[r]; w_post) (res itself without w_post, nothing without res); y[r] = norm(h[src(r)]; w_next) in 8 bits.
// A block a row, a lane a value.
// ---------------------------------------------------------------------------
template <typename TR>
__global__ void __launch_bounds__(256)
norm_rows_kernel(float* __restrict__ h, const TR* __restrict__ res, int n_part, size_t part_stride, const float* __restrict__ w_post,
                 float eps_post, const float* __restrict__ w_next, float eps_next, const int* __restrict__ rows,
                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int H) {
    __shared__ float scratch[32];
    const int r = blockIdx.x;
    grid_dependents_launch();
    grid_dependency_wait();
    float* hr = h + (size_t)(rows ? rows[r] : r) * H;
    float ss = 0.f;
    if (res != nullptr) {
        const TR* rr = res + (size_t)r * H;
        float inv = 1.f;
        if (w_post != nullptr) {
            for (int i = threadIdx.x; i < H; i += blockDim.x) {
                float v = to_float(rr[i]);
                for (int p = 1; p < n_part; ++p) v += to_float(rr[p * part_stride + i]);
                ss = fmaf(v, v, ss);
            }
            ss = block_sum(ss, scratch);
            inv = 1.0f / sqrtf(ss / (float)H + eps_post);
        }
        ss = 0.f;
        for (int i = threadIdx.x; i < H; i += blockDim.x) {
            float v = to_float(rr[i]);
            for (int p = 1; p < n_part; ++p) v += to_float(rr[p * part_stride + i]);
            const float hv = hr[i] + (w_post != nullptr ? v * inv * w_post[i] : v);
            hr[i] = hv;                          // read back below by this same thread only
            ss = fmaf(hv, hv, ss);
        }
    } else {
        for (int i = threadIdx.x; i < H; i += blockDim.x) ss = fmaf(hr[i], hr[i], ss);
    }
    ss = block_sum(ss, scratch);
    const float inv = 1.0f / sqrtf(ss / (float)H + eps_next);
    const int kp = padded(H);
    for (int i = threadIdx.x; i < kp; i += blockDim.x)          // whole warps: kp is a multiple of 128
        store_group(i < H ? hr[i] * inv * w_next[i] : 0.f, codes, scales, r, i / GROUP, kp / GROUP, kp);
}

// Sum over a block in a fixed order, the warps' sums in 64 bits: a row's factor then has little more of rounding than its lanes' sums, which
// are many and err at random.  `scratch` holds at least 32.
__device__ __forceinline__ double block_sum_long(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = (blockDim.x + 31) >> 5;
    v = warp_sum(v);
    if (nwarp == 1) return v;
    __syncthreads();            // scratch may still be read from an earlier call
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    double t = 0.;
    for (int w = 0; w < nwarp; ++w) t += (double)scratch[w];
    return t;
}

// 1 / sqrt(mean) in 64 bits from the float `f`: one step of Newton's, whose error is the square of f's
__device__ __forceinline__ double refined(float f, double mean) { return fma(0.5 * f, fma(-mean * f, (double)f, 1.0), (double)f); }

constexpr int MANY_ROWS = 768;     // from here on what counts is the rows that an SM has on its way and how often a code turns, not how long a row takes

struct Nothing {};                 // for values that are what they are

// Eight values a thread, four threads a group, sixteen a block of 128: codes as 8 bytes, the block's four scales as 4.  Whole warps call it.
// With `exact` (value e in 64 bits) a value within 8 units in the last place of the middle between two codes, which a float's roundings may turn, is
// formed again and rounded once: one value in 60,000, for three instructions a value.
template <typename F>
__device__ __forceinline__ void store_eight_of_group(const float* v, uint8_t* codes, uint8_t* scales, int r, int j, int blocks, bool live,
                                                     F exact) {
    float big = fabsf(v[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) big = larger(big, v[e]);
    big = larger(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = larger(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const uint32_t byte = scale_byte_e4m3(big);
    const float inv = inverse_scale(byte);
    uint32_t four = byte << (8 * (threadIdx.x >> 2 & 3));
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    four |= __shfl_xor_sync(0xffffffffu, four, 8);
    float x[8];
    bool near = false;
    // (the last 20 bits of a float are what a code with 3 bits behind the point leaves; codes below the normal ones are not looked at)
    const auto near_middle = [](float a) { return ((__float_as_uint(a) + 0x80008u) & 0xfffffu) <= 0x10u; };
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = v[e] * inv;
        near = near || near_middle(x[e]);
    }
    if constexpr (!std::is_same<F, Nothing>::value) {
        if (near && byte != 255u && live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!near_middle(x[e])) continue;                     // (nor are the zeros behind a row's end)
                const double y = exact(e) * (double)inv;
                float f = __double2float_rz(y);                       // rounded to odd, so that rounding it again is rounding y once
                if ((double)f != y) f = __uint_as_float(__float_as_uint(f) | 1u);
                x[e] = f;
            }
        }
    }
    uint2 q;
    q.x = two_e4m3(x[0], x[1]) | two_e4m3(x[2], x[3]) << 16;
    q.y = two_e4m3(x[4], x[5]) | two_e4m3(x[6], x[7]) << 16;
    if (byte == 255u) q = make_uint2(0u, 0u);
    if (!live) return;
    *reinterpret_cast<uint2*>(codes + ((size_t)r * blocks * BLOCK + (size_t)j * 8)) = q;
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t*>(scales + scale_at(r, j / 16, blocks)) = four;
}

// The same with the row in registers where rows start anywhere or are no whole pieces of 8: thread i takes the values i, i + blockDim, ... (VPT of
// them), 4 or 2 bytes at a time, and the row is turned to pieces of 8 in shared memory.  8,192 rows of 1,001: 36.0 us with 8 values a
// thread; of 2,303 98 (loads and stores of single values).  Rows above 4,096 leave room for one block of 8 values a thread on an SM (64
// registers, 513 threads or more): with 16 there are two, 2,048 rows of 4,607 62.9 us against 82.1, 256 10.0 against 12.5; a single row, which
// has the SM to itself, 6.6 against 5.3; 16 spill 72 bytes, 40 with a float residual.  All of these are 2.6 to 4 times what the bytes take (13.8 us for
// 8,192 of 1,001, 31.8 of 2,303; 15.9 for 2,048 of 4,607), with neither memory nor issue slots at their limit.  Rows brought in 16-byte pieces
// through shared memory: 41.6 us (of 1,001), 105 (of 2,303), 62.8 (of 4,607).
template <typename TR, int VPT>
__global__ void __launch_bounds__(640)
norm_rows_odd_kernel(float* __restrict__ h, const TR* __restrict__ res, const float* __restrict__ w_post, float eps_post,
                     const float* __restrict__ w_next, float eps_next, const int* __restrict__ rows, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales, int H, double share) {
    extern __shared__ __align__(16) float y[];                        // the row, on its way from a value a lane to pieces of 8
    __shared__ float scratch[32];
    const int r = blockIdx.x, kp = padded(H);
    grid_dependents_launch();
    grid_dependency_wait();
    float* hr = h + (size_t)(rows ? rows[r] : r) * H;
    float v[VPT], hv[VPT], ss = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = threadIdx.x + k * blockDim.x;
        hv[k] = i < H ? hr[i] : 0.f;
        v[k] = res != nullptr && i < H ? to_float(res[(size_t)r * H + i]) : 0.f;
    }
    double mean_post = 1.;
    float post = 1.f;
    if (res != nullptr) {
        if (w_post != nullptr) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) ss = fmaf(v[k], v[k], ss);
            mean_post = fma(block_sum_long(ss, scratch), share, (double)eps_post);
            post = 1.0f / sqrtf((float)mean_post);
            ss = 0.f;
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int i = threadIdx.x + k * blockDim.x;
            if (i >= H) continue;
            hv[k] += w_post != nullptr ? v[k] * post * w_post[i] : v[k];
        }
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) ss = fmaf(hv[k], hv[k], ss);
    const double mean = fma(block_sum_long(ss, scratch), share, (double)eps_next);
    const float inv = 1.0f / sqrtf((float)mean);
    // (the sum as it was before it was rounded: what it is made of is still there)
    const auto exact = [&](int i) {
        double t = hr[i];
        if (res != nullptr) {
            const double add = to_float(res[(size_t)r * H + i]);
            t += w_post != nullptr ? add * refined(post, mean_post) * (double)w_post[i] : add;
        }
        return t * (double)w_next[i] * refined(inv, mean);
    };
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < kp) y[i] = i < H ? hv[k] * inv * w_next[i] : 0.f;
    }
    __syncthreads();
    for (int j = threadIdx.x; j - (int)(threadIdx.x & 31) < kp / 8; j += blockDim.x) {      // whole warps
        float e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (j < kp / 8) load_eight(y + j * 8, e);
        store_eight_of_group(e, codes, scales, r, j, kp / BLOCK, j < kp / 8, [&](int at) { return exact(j * 8 + at); });
    }
    if (res == nullptr) return;
    __syncthreads();                                                  // (what is exact reads the stream as it was)
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < H) hr[i] = hv[k];
    }
}

// eight values of the residual as they are stored
template <typename T> struct Eight;
template <> struct Eight<bf16> {
    uint4 raw;
    __device__ __forceinline__ void load(const bf16* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float get(int e) const {               // (e is a constant where this is used)
        const uint32_t w = e / 2 == 0 ? raw.x : e / 2 == 1 ? raw.y : e / 2 == 2 ? raw.z : raw.w;
        return __uint_as_float(e % 2 ? w & 0xffff0000u : w << 16);
    }
};
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) { load_eight(p, v); }
    __device__ __forceinline__ float get(int e) const { return v[e]; }
};

// The same with the row in registers: thread i takes the pieces of 8 values i, i + blockDim, ... (H a multiple of 8, at most VPT of them), so that
// each input is read once, 16 bytes at a time, and a row's scales leave four at a time.  Bound by memory at many rows, where what counts is how
// many rows an SM has on its way: the residual stays as it is stored, the norms' weights are read where they are used, and a thread takes two
// pieces.  8,192 rows of 2,304 over the same inputs, in us: one piece a thread 43.2, two 37.9, five 40.3, nine (a warp a row) 59.8; 31.9 at the copy's
// bandwidth.  With the warps' sums in 64 bits and values near a middle formed again 40.7, over inputs that L2 does not hold 43 to 44, for half as many codes
// that differ from those of 64 bits (69 of 75 million; plain float arithmetic 144).  Held weights and eight floats of the residual a thread: 60.0;
// rows that the copy engine brings into a ring: 66.7.  At few rows, bound by latency, one piece: one row 2.5 us, with two 2.8.
// At most 48 registers, since what is rare takes more otherwise; two pieces spill 28 bytes, 44 with a float residual.
template <typename TR, int VPT>
__global__ void __launch_bounds__(640, VPT == 3 ? 1 : 2)
norm_rows_vec_kernel(float* __restrict__ h, const TR* __restrict__ res, const float* __restrict__ w_post, float eps_post,
                      const float* __restrict__ w_next, float eps_next, const int* __restrict__ rows, uint8_t* __restrict__ codes,
                      uint8_t* __restrict__ scales, int H, double share) {
    __shared__ float scratch[32];
    // A few rows have few values that lie near a middle and want to be quick: one row of 2,304 2.58 us against 2.74 with sums in 64 bits, 64 of 4,608
    // 4.5 against 5.0.  Many rows take those at any width: 8,192 of 1,024 22.6 us against 22.0, of 640 17.7 against 17.1.
    const bool quick = VPT == 1 && gridDim.x < MANY_ROWS;
    const auto row_sum = [&](float v) { return quick ? (double)block_sum(v, scratch) : block_sum_long(v, scratch); };
    const int r = blockIdx.x, pieces = H / 8, all = padded(H) / 8;
    grid_dependents_launch();
    grid_dependency_wait();
    float* hr = h + (size_t)(rows ? rows[r] : r) * H;
    Eight<TR> v[VPT];
    float hv[VPT][8];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int j = threadIdx.x + k * blockDim.x;
        if (j < pieces) {
            if (res != nullptr) v[k].load(res + (size_t)r * H + j * 8);
            load_eight(hr + j * 8, hv[k]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[k][e] = 0.f;
        }
    }
    float ss = 0.f;
    double mean_post = 1.;
    float post = 1.f;
    if (res != nullptr) {
        if (w_post != nullptr) {
#pragma unroll
            for (int k = 0; k < VPT; ++k)
                if ((int)threadIdx.x + k * (int)blockDim.x < pieces)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss = fmaf(v[k].get(e), v[k].get(e), ss);
            mean_post = fma(row_sum(ss), share, (double)eps_post);
            post = 1.0f / sqrtf((float)mean_post);
            ss = 0.f;
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int j = threadIdx.x + k * blockDim.x;
            if (j >= pieces) continue;
            if (w_post != nullptr) {
                float w[8];
                load_eight(w_post + j * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) hv[k][e] += v[k].get(e) * post * w[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) hv[k][e] += v[k].get(e);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(hv[k][e], hv[k][e], ss);
    const double mean = fma(row_sum(ss), share, (double)eps_next);
    const float inv = 1.0f / sqrtf((float)mean);
    // (the sum as it was before it was rounded: what it is made of is still there)
    const auto exact = [&](int i) {
        double t = hr[i];
        if (res != nullptr) {
            const double add = to_float(res[(size_t)r * H + i]);
            t += w_post != nullptr ? add * refined(post, mean_post) * (double)w_post[i] : add;
        }
        return t * (double)w_next[i] * refined(inv, mean);
    };
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int j = threadIdx.x + k * blockDim.x;
        if (j - (int)(threadIdx.x & 31) >= all) break;                // (a whole warp)
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 0.f;
        if (j < pieces) load_eight(w_next + j * 8, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = hv[k][e] * inv * w[e];
        store_eight_of_group(w, codes, scales, r, j, all / 16, j < all, [&](int at) { return exact(j * 8 + at); });
        if (res != nullptr && j < pieces) store_eight(hr + j * 8, hv[k]);
    }
}

// ---------------------------------------------------------------------------
// rows as they are, and act(gate) * up over columns that alternate 8 gates, 8 ups (act 0: gelu's tanh form, 1: silu,
// 2: the clamped gate); a warp a group
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
plain_rows_kernel(const T* __restrict__ x, int act, float limit, float alpha, float up_add, uint8_t* __restrict__ codes,
                  uint8_t* __restrict__ scales, size_t n_groups, int K, int kp) {
    grid_dependents_launch();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, groups = kp / GROUP;
    for (size_t q = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); q < n_groups; q += (size_t)gridDim.x * 8) {
        const int r = (int)(q / groups), g = (int)(q % groups), i = g * GROUP + lane;
        float v = 0.f;
        if (i < K) {
            if (act < 0) {
                v = to_float(x[(size_t)r * K + i]);
            } else {
                const size_t at = (size_t)r * 2 * K + (size_t)(i / 8) * 16 + i % 8;
                const float gate = to_float(x[at]), up = to_float(x[at + 8]);
                v = act == 2 ? clamped_gate(gate, up, limit, alpha, up_add) : (act == 0 ? gelu_tanh(gate) : gate / (1.0f + expf(-gate))) * up;
            }
        }
        store_group(v, codes, scales, r, g, groups, kp);
    }
}

// the same, eight values a thread (K a multiple of 8, 16-byte pieces)
template <typename T>
__global__ void __launch_bounds__(256)
plain_rows_vec_kernel(const T* __restrict__ x, int act, float limit, float alpha, float up_add, uint8_t* __restrict__ codes,
                      uint8_t* __restrict__ scales, size_t n_pieces, int K, int kp) {
    grid_dependents_launch();
    grid_dependency_wait();
    const int per_row = kp / 8;
    for (size_t q = (size_t)blockIdx.x * 256 + threadIdx.x; q - (threadIdx.x & 31) < n_pieces; q += (size_t)gridDim.x * 256) {
        const bool live = q < n_pieces;
        const int r = live ? (int)(q / per_row) : 0, j = live ? (int)(q - (size_t)r * per_row) : 0;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (live && j * 8 < K) {
            if (act < 0) {
                load_eight(x + (size_t)r * K + j * 8, v);
            } else {
                float g[8], u[8];
                load_eight(x + (size_t)r * 2 * K + j * 16, g);
                load_eight(x + (size_t)r * 2 * K + j * 16 + 8, u);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = act == 2 ? clamped_gate(g[e], u[e], limit, alpha, up_add) : (act == 0 ? gelu_tanh(g[e]) : g[e] / (1.0f + expf(-g[e]))) * u[e];
            }
        }
        store_eight_of_group(v, codes, scales, r, j, kp / BLOCK, live, Nothing());
    }
}

// ---------------------------------------------------------------------------
// weights to 4 bits, at load: a warp a group
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, size_t n_groups, int K, int kp) {
    const int lane = threadIdx.x & 31, groups = kp / GROUP;
    for (size_t q = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); q < n_groups; q += (size_t)gridDim.x * 8) {
        const int r = (int)(q / groups), g = (int)(q % groups), i = g * GROUP + lane;
        const float v = i < K ? to_float(w[(size_t)r * K + i]) : 0.f;
        float big = fabsf(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = larger(big, __shfl_xor_sync(0xffffffffu, big, o));
        const uint32_t byte = scale_byte_e2m1(big);
        const float mine = byte == 255u ? 0.f : v * inverse_scale(byte), next = __shfl_down_sync(0xffffffffu, mine, 1);
        if (lane % 2 == 0) codes[((size_t)r * kp + i) / 2] = (uint8_t)two_e2m1(mine, next);
        if (lane == 0) scales[scale_at(r, g / 4, groups / 4) + g % 4] = (uint8_t)byte;
    }
}

// ---------------------------------------------------------------------------
// the values that a matrix stands for
// ---------------------------------------------------------------------------
template <typename TO>
__global__ void __launch_bounds__(256)
values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, TO* __restrict__ out, size_t n, int K, int kp, int bits) {
    grid_dependents_launch();
    grid_dependency_wait();
    for (size_t q = (size_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (size_t)gridDim.x * 256) {
        const int r = (int)(q / K), i = (int)(q % K);
        const size_t at = (size_t)r * kp + i;
        const float v = bits == 8 ? value_e4m3(codes[at]) : value_e2m1(codes[at / 2] >> (at % 2 * 4) & 15u);
        out[q] = from_float<TO>(v * scale_value(scales[scale_at(r, i / BLOCK, kp / BLOCK) + i % BLOCK / GROUP]));
    }
}

template <typename TR>
static int norm_rows(float* h, const TR* res, int n_part, size_t part_stride, const float* w_post, float eps_post, const float* w_next,
                     float eps_next, const int* rows, uint8_t* codes, uint8_t* scales, int R, int H, cudaStream_t stream) {
    const bool vec = H % 8 == 0 && (((uintptr_t)h | (uintptr_t)res | (uintptr_t)w_post | (uintptr_t)w_next) & 15) == 0 && part_stride % 8 == 0;
    const int pieces = padded(H) / 8;
    if (!vec && n_part <= 1 && pieces <= 640) {
        const int n = pieces > 512 && R > 148 ? 16 : pieces > 320 || (R >= MANY_ROWS && pieces > 80) ? 8 : 4;
        const auto kernel = n == 4 ? norm_rows_odd_kernel<TR, 4> : n == 8 ? norm_rows_odd_kernel<TR, 8> : norm_rows_odd_kernel<TR, 16>;
        return launch_kernel("mx_norm_rows", kernel, dim3(R), dim3((pieces * 8 / n + 31) / 32 * 32), pieces * 32, stream, 1, h, res, w_post, eps_post, w_next,
                             eps_next, rows, codes, scales, H, 1.0 / H);
    }
    if (!vec || n_part > 1 || pieces > 1920)
        return launch_kernel("mx_norm_rows", norm_rows_kernel<TR>, dim3(R), dim3(256), 0, stream, 1, h, res, n_part, part_stride, w_post, eps_post,
                             w_next, eps_next, rows, codes, scales, H);
    const int vpt = pieces > 1280 ? 3 : pieces > 640 || (R >= MANY_ROWS && pieces > 160) ? 2 : 1;
    const auto kernel = vpt == 1 ? norm_rows_vec_kernel<TR, 1> : vpt == 2 ? norm_rows_vec_kernel<TR, 2> : norm_rows_vec_kernel<TR, 3>;
    return launch_kernel("mx_norm_rows", kernel, dim3(R), dim3(((pieces + vpt - 1) / vpt + 31) / 32 * 32), 0, stream, 1, h, res, w_post, eps_post,
                         w_next, eps_next, rows, codes, scales, H, 1.0 / H);      // (share: a mean is a sum times 1 / H)
}

static int blocks_for(size_t warps) {
    const size_t b = (warps + 7) / 8;
    return (int)(b < 148 * 32 ? b : 148 * 32);
}

template <typename T>
static int plain_rows(const T* x, int act, float limit, float alpha, float up_add, uint8_t* codes, uint8_t* scales, int R, int K,
                      cudaStream_t stream) {
    const int kp = padded(K);
    const size_t n_groups = (size_t)R * (kp / GROUP);
    if (K % 8 == 0 && ((uintptr_t)x & 15) == 0)
        return launch_kernel("mx_rows", plain_rows_vec_kernel<T>, dim3(blocks_for(n_groups / 8 + 1)), dim3(256), 0, stream, 1, x, act, limit, alpha,
                             up_add, codes, scales, n_groups * 4, K, kp);
    return launch_kernel("mx_rows", plain_rows_kernel<T>, dim3(blocks_for(n_groups)), dim3(256), 0, stream, 1, x, act, limit, alpha, up_add, codes,
                         scales, n_groups, K, kp);
}

}  // namespace mx
}  // namespace janis

using namespace janis;

JANIS_EXPORT const char* janis_last_error() { return error_buffer(); }
JANIS_EXPORT void janis_mx_set_overlap(int on) { overlap_launches() = on; }

// h [R or more, H] float; res [n_part, R, H] or null; rows [R] or null (with res: null); codes [R, padded H]
// The arguments come as one block of 8-byte fields.
struct NormArgs {
    float* h;
    const void* res;
    long long res_dtype, n_part, part_stride;
    const float* w_post;
    double eps_post;
    const float* w_next;
    double eps_next;
    const int* rows;
    uint8_t *codes, *scales;
    long long R, H;
    cudaStream_t stream;
};
JANIS_EXPORT int janis_mx_norm_rows(const void* block) {
    NormArgs a;
    memcpy(&a, block, sizeof(a));
    float* h = a.h;
    const void* res = a.res;
    const float *w_post = a.w_post, *w_next = a.w_next;
    const float eps_post = (float)a.eps_post, eps_next = (float)a.eps_next;
    const int* rows = a.rows;
    uint8_t *codes = a.codes, *scales = a.scales;
    if (a.R > 1 << 30 || a.H > 1 << 30) return fail("mx_norm_rows: sizes pass 2^30");
    const int res_dtype = (int)a.res_dtype, n_part = (int)a.n_part, R = (int)a.R, H = (int)a.H;
    const long long part_stride = a.part_stride;
    cudaStream_t stream = a.stream;
    if (R <= 0) return 0;
    if (H <= 0) return fail("mx_norm_rows: a row has no values");
    if (res != nullptr && rows != nullptr) return fail("mx_norm_rows: rows are gathered without a residual only");
    if (res_dtype == JANIS_BF16)
        return mx::norm_rows(h, (const bf16*)res, n_part, (size_t)part_stride, w_post, eps_post, w_next, eps_next, rows, codes, scales, R, H, stream);
    if (res_dtype != JANIS_F32) return fail("mx_norm_rows: unknown dtype %d", res_dtype);
    return mx::norm_rows(h, (const float*)res, n_part, (size_t)part_stride, w_post, eps_post, w_next, eps_next, rows, codes, scales, R, H, stream);
}

// act < 0: x [R, K] as it is; otherwise x [R, 2 K] of gates and ups
JANIS_EXPORT int janis_mx_rows(const void* x, int dtype, int act, float limit, float alpha, float up_add, uint8_t* codes, uint8_t* scales,
                               int R, int K, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (K <= 0) return fail("mx_rows: a row has no values");
    if (act > 2) return fail("mx_rows: unknown activation %d", act);
    if (act >= 0 && K % 8) return fail("mx_rows: gates and ups alternate in groups of 8, found %d columns", K);
    if (dtype == JANIS_BF16) return mx::plain_rows((const bf16*)x, act, limit, alpha, up_add, codes, scales, R, K, stream);
    if (dtype != JANIS_F32) return fail("mx_rows: unknown dtype %d", dtype);
    return mx::plain_rows((const float*)x, act, limit, alpha, up_add, codes, scales, R, K, stream);
}

JANIS_EXPORT int janis_mx_weight(const void* w, int dtype, uint8_t* codes, uint8_t* scales, int N, int K, cudaStream_t stream) {
    if (N <= 0) return 0;
    if (K <= 0) return fail("mx_weight: a row has no values");
    const int kp = mx::padded(K);
    const size_t n_groups = (size_t)N * (kp / mx::GROUP);
    const dim3 grid(mx::blocks_for(n_groups));
    if (dtype == JANIS_BF16)
        return launch_kernel_after("mx_weight", mx::weight_kernel<bf16>, grid, dim3(256), 0, stream, 1, (const bf16*)w, codes, scales, n_groups, K, kp);
    if (dtype != JANIS_F32) return fail("mx_weight: unknown dtype %d", dtype);
    return launch_kernel_after("mx_weight", mx::weight_kernel<float>, grid, dim3(256), 0, stream, 1, (const float*)w, codes, scales, n_groups, K, kp);
}

// bits 8 or 4: the values of a matrix [R, K] in either form
JANIS_EXPORT int janis_mx_values(const uint8_t* codes, const uint8_t* scales, int bits, void* out, int dtype, int R, int K, cudaStream_t stream) {
    if (R <= 0 || K <= 0) return 0;
    if (bits != 8 && bits != 4) return fail("mx_values: 8 or 4 bits, found %d", bits);
    const size_t n = (size_t)R * K;
    const int kp = mx::padded(K);
    const dim3 grid(mx::blocks_for((n + 31) / 32));
    if (dtype == JANIS_BF16)
        return launch_kernel("mx_values", mx::values_kernel<bf16>, grid, dim3(256), 0, stream, 1, codes, scales, (bf16*)out, n, K, kp, bits);
    if (dtype != JANIS_F32) return fail("mx_values: unknown dtype %d", dtype);
    return launch_kernel("mx_values", mx::values_kernel<float>, grid, dim3(256), 0, stream, 1, codes, scales, (float*)out, n, K, kp, bits);
}
