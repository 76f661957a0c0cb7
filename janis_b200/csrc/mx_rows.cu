// Rows in and out of the 8-bit microscaling form (mx.cuh): the norms and the gated activation that leave it for the products
// behind them, plain rows, the weights' 4-bit form at load, and the values that either form stands for.
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

static int blocks_for(size_t warps) {
    const size_t b = (warps + 7) / 8;
    return (int)(b < 148 * 32 ? b : 148 * 32);
}

}  // namespace mx
}  // namespace janis

using namespace janis;

JANIS_EXPORT const char* janis_last_error() { return error_buffer(); }
JANIS_EXPORT void janis_mx_set_overlap(int on) { overlap_launches() = on; }

// h [R or more, H] float; res [n_part, R, H] or null; rows [R] or null (with res: null); codes [R, padded H]
JANIS_EXPORT int janis_mx_norm_rows(float* h, const void* res, int res_dtype, int n_part, long long part_stride, const float* w_post,
                                    float eps_post, const float* w_next, float eps_next, const int* rows, uint8_t* codes,
                                    uint8_t* scales, int R, int H, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (H <= 0) return fail("mx_norm_rows: a row has no values");
    if (res != nullptr && rows != nullptr) return fail("mx_norm_rows: rows are gathered without a residual only");
    if (res_dtype == JANIS_BF16)
        return launch_kernel("mx_norm_rows", mx::norm_rows_kernel<bf16>, dim3(R), dim3(256), 0, stream, 1, h, (const bf16*)res, n_part,
                             (size_t)part_stride, w_post, eps_post, w_next, eps_next, rows, codes, scales, H);
    if (res_dtype != JANIS_F32) return fail("mx_norm_rows: unknown dtype %d", res_dtype);
    return launch_kernel("mx_norm_rows", mx::norm_rows_kernel<float>, dim3(R), dim3(256), 0, stream, 1, h, (const float*)res, n_part,
                         (size_t)part_stride, w_post, eps_post, w_next, eps_next, rows, codes, scales, H);
}

// act < 0: x [R, K] as it is; otherwise x [R, 2 K] of gates and ups
JANIS_EXPORT int janis_mx_rows(const void* x, int dtype, int act, float limit, float alpha, float up_add, uint8_t* codes, uint8_t* scales,
                               int R, int K, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (K <= 0) return fail("mx_rows: a row has no values");
    if (act > 2) return fail("mx_rows: unknown activation %d", act);
    if (act >= 0 && K % 8) return fail("mx_rows: gates and ups alternate in groups of 8, found %d columns", K);
    const int kp = mx::padded(K);
    const size_t n_groups = (size_t)R * (kp / mx::GROUP);
    const dim3 grid(mx::blocks_for(n_groups));
    if (dtype == JANIS_BF16)
        return launch_kernel("mx_rows", mx::plain_rows_kernel<bf16>, grid, dim3(256), 0, stream, 1, (const bf16*)x, act, limit, alpha,
                             up_add, codes, scales, n_groups, K, kp);
    if (dtype != JANIS_F32) return fail("mx_rows: unknown dtype %d", dtype);
    return launch_kernel("mx_rows", mx::plain_rows_kernel<float>, grid, dim3(256), 0, stream, 1, (const float*)x, act, limit, alpha, up_add,
                         codes, scales, n_groups, K, kp);
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
