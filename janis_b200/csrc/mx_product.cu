// Products of 8-bit rows with 4-bit weights (both in the microscaling form of mx.cuh), with float sums:
//   out[t, n] = epilogue(sum_k x[t, k] W[n, k]);  the gated epilogues take gate and up rows of W that alternate in groups of 8 and
//   give act(gate) * up, as values or as 8-bit rows for the product behind.
#include "mx.cuh"

namespace janis {
namespace mx {

enum { EPI_NONE = 0, EPI_GATED_GELU = 1, EPI_GATED_SILU = 3, EPI_GATED_CLAMP = 4 };

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

// one row of x with one row of W, by a warp: a lane takes every 32nd group
__device__ __forceinline__ float dot(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, int t, int n, int kp) {
    float sum = 0.f;
    const int groups = kp / GROUP;
    for (int g = threadIdx.x & 31; g < groups; g += 32) {
        float s = 0.f;
        for (int i = 0; i < GROUP; ++i) {
            const size_t k = (size_t)g * GROUP + i;
            s = fmaf(value_e4m3(xc[(size_t)t * kp + k]), value_e2m1(wc[((size_t)n * kp + k) / 2] >> (k % 2 * 4) & 15u), s);
        }
        sum = fmaf(s, scale_value(xs[scale_at(t, g / 4, groups / 4) + g % 4]) * scale_value(ws[scale_at(n, g / 4, groups / 4) + g % 4]), sum);
    }
    return warp_sum(sum);
}

// a block: 32 columns of out in one row, a warp four of them
__global__ void __launch_bounds__(256)
product_kernel(const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ wc,
               const uint8_t* __restrict__ ws, Out o, int T, int N, int kp) {
    __shared__ float vals[32];
    const int t = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependents_launch();
    grid_dependency_wait();
    const int cols = o.epi == EPI_NONE ? N : N / 2;
    for (int j = warp; j < 32; j += 8) {
        const int c = blockIdx.x * 32 + j;
        float v = 0.f;
        if (c < cols) {
            if (o.epi == EPI_NONE) {
                v = dot(xc, xs, wc, ws, t, c, kp);
            } else {
                const int n = c / 8 * 16 + c % 8;
                v = gated(dot(xc, xs, wc, ws, t, n, kp), dot(xc, xs, wc, ws, t, n + 8, kp), o);
            }
        }
        if (lane == 0) vals[j] = v;
    }
    __syncthreads();
    if (warp != 0) return;
    const int c = blockIdx.x * 32 + lane;
    const float v = vals[lane];
    if (o.codes != nullptr) {
        float big = fabsf(v);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) big = larger(big, __shfl_xor_sync(0xffffffffu, big, s));
        const uint32_t byte = scale_byte_e4m3(big);
        const int op = padded(cols);
        o.codes[(size_t)t * op + c] = byte == 255u ? 0 : (uint8_t)two_e4m3(v * inverse_scale(byte), 0.f);
        if (lane == 0) o.scales[scale_at(t, c / BLOCK, op / BLOCK) + c % BLOCK / GROUP] = (uint8_t)byte;
    } else if (c < cols) {
        if (o.dtype == JANIS_BF16) reinterpret_cast<bf16*>(o.values)[(size_t)t * cols + c] = from_float<bf16>(v);
        else reinterpret_cast<float*>(o.values)[(size_t)t * cols + c] = v;
    }
}

}  // namespace mx
}  // namespace janis

using namespace janis;

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
    const mx::Out o = {out, out_codes, out_scales, out_dtype, epi, limit, alpha, up_add};
    const int cols = epi == mx::EPI_NONE ? N : N / 2;
    const int wide = out_codes != nullptr ? mx::padded(cols) : cols;
    if (T > 65535) return fail("mx_product: at most 65535 rows, found %d", T);
    return launch_kernel("mx_product", mx::product_kernel, dim3((wide + 31) / 32, T), dim3(256), 0, stream, 1, xc, xs, wc, ws, o, T, N, mx::padded(K));
}
