// q8_matmul.cu — the product of two sets of 8-bit rows,
//   out[t][n] = (sum_k x[t][k] w[n][k]) * sx[t] * sw[n] + bias[n],
// the sum exact in 32-bit integers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "q8.h"

namespace jhq {

namespace {

__device__ int g_q8_error;          // a bounded wait gave up

struct Epilogue {                   // what turns a sum into an output
    const float *sx, *sw, *bias;    // bias may be null
    void* out;
    int64_t ldo;
    int64_t T;
    int N, type;
};

__device__ __forceinline__ void store_out(const Epilogue& e, int64_t t, int n, float v) {
    const int64_t at = t * e.ldo + n;
    if (e.type == JHQ_F32) static_cast<float*>(e.out)[at] = v;
    else if (e.type == JHQ_F16) static_cast<__half*>(e.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(e.out)[at] = __float2bfloat16_rn(v);
}

constexpr int TILE = 64, KC = 64;   // outputs a side, bytes of K a step

// Any alignment: bytes are loaded one by one. 256 threads, 4 x 4 sums each.
__global__ void __launch_bounds__(256)
simple_kernel(const int8_t* __restrict__ x, int64_t ldx, const int8_t* __restrict__ w, int64_t ldw, int K,
              Epilogue e) {
    __shared__ int xs[TILE][KC / 4 + 1], ws[TILE][KC / 4 + 1];
    const int64_t t0 = (int64_t)blockIdx.x * TILE;
    const int n0 = blockIdx.y * TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += KC) {
        for (int i = threadIdx.x; i < TILE * KC; i += 256) {
            const int r = i / KC, c = i % KC, k = k0 + c;
            reinterpret_cast<int8_t*>(xs[r])[c] =
                t0 + r < e.T && k < K ? x[(t0 + r) * ldx + k] : (int8_t)0;
            reinterpret_cast<int8_t*>(ws[r])[c] =
                n0 + r < e.N && k < K ? w[(int64_t)(n0 + r) * ldw + k] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < KC / 4; ++c) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = xs[ty + 16 * i][c]; b[i] = ws[tx + 16 * i][c]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t t = t0 + ty + 16 * i;
            const int n = n0 + tx + 16 * j;
            if (t < e.T && n < e.N) {
                const float v = (float)acc[i][j] * e.sx[t] * e.sw[n];
                store_out(e, t, n, e.bias ? v + e.bias[n] : v);
            }
        }
}

}  // namespace

void q8_matmul(const jhq_q8_rows* x, const jhq_q8_rows* w, const jhq_view* bias, const jhq_view* out,
               cudaStream_t s) {
    q8_check_rows(x, "q8_matmul: x");
    q8_check_rows(w, "q8_matmul: w");
    if (x->dim != w->dim) fail(JHQ_EINVAL, "q8_matmul: x and w must have rows of one length");
    if (x->dim > 131071) fail(JHQ_EINVAL, "q8_matmul: rows are longer than 131071");
    if (x->groups != 1 || w->groups != 1) fail(JHQ_EINVAL, "q8_matmul: x and w must have one group");
    if (x->rows == 0 || w->rows == 0) return;
    q8_check_view(out, "q8_matmul: out");
    if (out->rows != x->rows || out->cols != w->rows)
        fail(JHQ_EINVAL, "q8_matmul: out must be x's rows by w's rows");
    if (x->rows > INT32_MAX || w->rows > INT32_MAX) fail(JHQ_EINVAL, "q8_matmul: too many rows");
    if (bias) {
        q8_check_view(bias, "q8_matmul: bias");
        if (bias->type != JHQ_F32 || bias->rows != 1 || bias->cols != out->cols)
            fail(JHQ_EINVAL, "q8_matmul: bias must be 1 x w's rows of float32");
    }
    const Epilogue e{x->scale, w->scale, bias ? (const float*)bias->data : nullptr, out->data, out->ld,
                     x->rows, (int)w->rows, out->type};
    const dim3 grid((unsigned)ceil_div(x->rows, TILE), (unsigned)ceil_div(w->rows, TILE));
    simple_kernel<<<grid, 256, 0, s>>>(x->q, x->ld, w->q, w->ld, (int)x->dim, e);
    JHQ_LAUNCH_CHECK();
    count_launch();
}

bool q8_take_error() {
    int v = 0;
    JHQ_CUDA(cudaMemcpyFromSymbol(&v, g_q8_error, sizeof(int)));
    if (v) {
        const int z = 0;
        JHQ_CUDA(cudaMemcpyToSymbol(g_q8_error, &z, sizeof(int)));
    }
    return v != 0;
}

}  // namespace jhq
