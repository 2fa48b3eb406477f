// q8_rows.cu — rows to 8 bits and back: the RMS norm with the residual's
// addition and 8-bit output, and the cache's write and read.
//
// With h = x + r, g = h * w and a = max |g| over a row, the normed row
// y = g / rms (rms = sqrt(mean h^2 + eps), one positive number for the row)
// has max |y| = a / rms, so its 8-bit values rint(y * 127 / max |y|) are
// rint(g * (127 * (1 / a))): they do not wait for the sum of squares, and one pass
// over the row gathers both a and sum h^2. The scale is a / (127 rms).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <string>

#include "kernels.cuh"
#include "q8.h"

namespace jhq {

void q8_check_view(const jhq_view* v, const char* what) {
    const std::string w(what);
    if (!v) fail(JHQ_EINVAL, w + ": null");
    if (v->type != JHQ_F32 && v->type != JHQ_F16 && v->type != JHQ_BF16)
        fail(JHQ_EINVAL, w + ": unknown type");
    if (v->rows < 0 || v->cols < 1 || v->cols > INT32_MAX)
        fail(JHQ_EINVAL, w + ": rows must be >= 0 and cols in 1..2^31-1");
    if (v->rows > 1 && v->ld < v->cols) fail(JHQ_EINVAL, w + ": ld is smaller than a row");
    if (v->rows > 0 && !v->data) fail(JHQ_EINVAL, w + ": null data");
    if ((uintptr_t)v->data % (v->type == JHQ_F32 ? 4 : 2))
        fail(JHQ_EINVAL, w + ": data is not aligned to its type");
}

void q8_check_rows(const jhq_q8_rows* r, const char* what) {
    const std::string w(what);
    if (!r) fail(JHQ_EINVAL, w + ": null");
    if (r->rows < 0 || r->dim < 1 || r->dim > INT32_MAX)
        fail(JHQ_EINVAL, w + ": rows must be >= 0 and dim in 1..2^31-1");
    if (r->groups < 1 || r->dim % r->groups) fail(JHQ_EINVAL, w + ": groups must divide dim");
    if (r->rows > 1 && r->ld < r->dim) fail(JHQ_EINVAL, w + ": ld is smaller than a row");
    if (r->rows > 0 && (!r->q || !r->scale)) fail(JHQ_EINVAL, w + ": null buffer");
    if ((uintptr_t)r->scale % 4) fail(JHQ_EINVAL, w + ": scale is not aligned to its type");
}

namespace {

constexpr int THREADS = 256;
constexpr uint32_t INF_BITS = 0x7f800000u;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Block-wide sum and maximum, returned to every thread.
__device__ float2 block_sum_max(float sum, uint32_t top, float* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    top = __reduce_max_sync(~0u, top);
    __syncthreads();                                     // red is free again
    if (lane == 0) { red[2 * warp] = sum; red[2 * warp + 1] = __uint_as_float(top); }
    __syncthreads();
    sum = 0.0f;
    top = 0;
    for (int i = 0; i < THREADS / 32; ++i) {
        sum += red[2 * i];
        top = max(top, __float_as_uint(red[2 * i + 1]));
    }
    return make_float2(sum, __uint_as_float(top));
}

// q = rint(g * (127 * (1 / a))). A tiny a would make 1 / a infinite: both are
// scaled by 2^64 first (exact).
struct Quant {
    float pre, inv;
    __device__ explicit Quant(float a) {
        pre = a < 1e-30f ? 0x1p64f : 1.0f;
        inv = a > 0.0f && __float_as_uint(a) < INF_BITS ? 127.0f * (1.0f / (a * pre)) : 0.0f;
    }
    __device__ int8_t operator()(float g) const {
        return inv == 0.0f ? (int8_t)0 : (int8_t)__float2int_rn(g * pre * inv);
    }
};

template <class T, class R>
__global__ void __launch_bounds__(THREADS)
rms_norm_kernel(const T* __restrict__ x, int64_t ldx, const R* res, int64_t ldr,
                const void* __restrict__ weight, int w32, float eps, R* res_out, int64_t ldo,
                int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale, int d) {
    __shared__ float red[2 * THREADS / 32];
    const int64_t row = blockIdx.x;
    x += row * ldx;
    if (res) res += row * ldr;
    if (res_out) res_out += row * ldo;
    q += row * ldq;
    auto h_of = [&](int j) {
        const float v = to_float(x[j]);
        return res ? v + to_float(res[j]) : v;
    };
    auto w_of = [&](int j) {
        if (!weight) return 1.0f;
        return w32 ? static_cast<const float*>(weight)[j] : to_float(static_cast<const T*>(weight)[j]);
    };
    float sum = 0.0f;
    uint32_t top = 0;                                    // bits of |g| order like |g|, NaN on top
    for (int j = threadIdx.x; j < d; j += THREADS) {
        const float h = h_of(j);
        sum += h * h;
        top = max(top, __float_as_uint(fabsf(h * w_of(j))));
    }
    const float2 st = block_sum_max(sum, top, red);
    float a = st.y, sc = 1.0f, step = a / (127.0f * sqrtf(st.x / (float)d + eps));
    if (!(st.x >= 0x1p-90f && st.x <= 0x1p120f && a >= 0x1p-100f && a <= 0x1p120f)) {
        // near the ends of float32's range: again with h scaled by a power of two
        uint32_t hm = 0;
        for (int j = threadIdx.x; j < d; j += THREADS) hm = max(hm, __float_as_uint(fabsf(h_of(j))));
        const float htop = block_sum_max(0.0f, hm, red).y;
        if (htop > 0.0f && __float_as_uint(htop) < INF_BITS) {
            const int e = min(max(ilogbf(htop), -126), 126);
            sc = ldexpf(1.0f, -e);
            sum = 0.0f;
            top = 0;
            for (int j = threadIdx.x; j < d; j += THREADS) {
                const float h = h_of(j) * sc;
                sum += h * h;
                top = max(top, __float_as_uint(fabsf(h * w_of(j))));
            }
            const float2 s2 = block_sum_max(sum, top, red);
            a = s2.y;
            step = (float)((double)a / (127.0 * sqrt((double)s2.x / d + (double)eps * sc * sc)));
        }
    }
    const Quant quant(a);
    for (int j = threadIdx.x; j < d; j += THREADS) {
        const float h = h_of(j);
        if (res_out) store(res_out + j, h);
        q[j] = quant(h * sc * w_of(j));
    }
    if (threadIdx.x == 0) {
        const bool fine = __float_as_uint(a) < INF_BITS;
        scale[row] = !fine ? __uint_as_float(0x7fffffffu) : a > 0.0f ? step : 0.0f;
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS)
write_kernel(const T* __restrict__ x, int64_t ldx, const int64_t* __restrict__ slots,
             int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale, int64_t nslots, int groups,
             int gdim) {
    __shared__ float red[2 * THREADS / 32];
    const int64_t row = blockIdx.x / groups;
    const int g = (int)(blockIdx.x % groups);
    const int64_t slot = slots ? slots[row] : row;
    if (slot < 0 || slot >= nslots) return;
    x += row * ldx + (int64_t)g * gdim;
    q += slot * ldq + (int64_t)g * gdim;
    uint32_t top = 0;
    for (int j = threadIdx.x; j < gdim; j += THREADS)
        top = max(top, __float_as_uint(fabsf(to_float(x[j]))));
    const float a = block_sum_max(0.0f, top, red).y;
    const Quant quant(a);
    for (int j = threadIdx.x; j < gdim; j += THREADS) q[j] = quant(to_float(x[j]));
    if (threadIdx.x == 0)
        scale[slot * groups + g] =
            __float_as_uint(a) < INF_BITS ? a / 127.0f : __uint_as_float(0x7fffffffu);
}

template <class T>
__global__ void __launch_bounds__(THREADS)
read_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale, int64_t nslots,
            const int64_t* __restrict__ slots, T* __restrict__ out, int64_t ldo, int groups, int gdim) {
    const int64_t row = blockIdx.x;
    const int64_t slot = slots ? slots[row] : row;
    const bool there = slot >= 0 && slot < nslots;
    out += row * ldo;
    for (int j = threadIdx.x; j < groups * gdim; j += THREADS)
        store(out + j, there ? scale[slot * groups + j / gdim] * (float)q[slot * ldq + j] : 0.0f);
}

template <class F>
void by_type(int type, F&& f) {
    if (type == JHQ_F32) f(float());
    else if (type == JHQ_F16) f(__half());
    else f(__nv_bfloat16());
}

}  // namespace

void q8_rms_norm(const jhq_view* x, const jhq_view* residual, const jhq_view* weight, float eps,
                 const jhq_view* residual_out, const jhq_q8_rows* out, cudaStream_t s) {
    q8_check_view(x, "q8_rms_norm: x");
    q8_check_rows(out, "q8_rms_norm: out");
    if (out->rows != x->rows || out->dim != x->cols)
        fail(JHQ_EINVAL, "q8_rms_norm: out must have x's rows and cols");
    if (out->groups != 1) fail(JHQ_EINVAL, "q8_rms_norm: out must have one group");
    if (!(eps >= 0.0f) || std::isinf(eps)) fail(JHQ_EINVAL, "q8_rms_norm: eps must be finite and >= 0");
    if (weight) {
        q8_check_view(weight, "q8_rms_norm: weight");
        if (weight->rows != 1 || weight->cols != x->cols)
            fail(JHQ_EINVAL, "q8_rms_norm: weight must be 1 x cols");
        if (weight->type != x->type && weight->type != JHQ_F32)
            fail(JHQ_EINVAL, "q8_rms_norm: weight must be of x's type or float32");
    }
    int rtype = x->type;
    for (const jhq_view* r : {residual, residual_out}) {
        if (!r) continue;
        const char* what = r == residual ? "q8_rms_norm: residual" : "q8_rms_norm: residual_out";
        q8_check_view(r, what);
        if (r->rows != x->rows || r->cols != x->cols)
            fail(JHQ_EINVAL, std::string(what) + " must have x's rows and cols");
        if (r->type != x->type && r->type != JHQ_F32)
            fail(JHQ_EINVAL, std::string(what) + " must be of x's type or float32");
        rtype = r->type;
    }
    if (residual && residual_out && residual->type != residual_out->type)
        fail(JHQ_EINVAL, "q8_rms_norm: residual and residual_out must have one type");
    if (x->rows == 0) return;
    if (x->rows > INT32_MAX) fail(JHQ_EINVAL, "q8_rms_norm: too many rows");
    by_type(x->type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto r) {
            using R = decltype(r);
            rms_norm_kernel<T, R><<<(unsigned)x->rows, THREADS, 0, s>>>(
                (const T*)x->data, x->ld, residual ? (const R*)residual->data : nullptr,
                residual ? residual->ld : 0, weight ? weight->data : nullptr,
                weight && weight->type == JHQ_F32, eps, residual_out ? (R*)residual_out->data : nullptr,
                residual_out ? residual_out->ld : 0, out->q, out->ld, out->scale, (int)x->cols);
        };
        if (rtype == x->type) go(t);
        else go(float());
    });
    JHQ_LAUNCH_CHECK();
    count_launch();
}

void q8_write(const jhq_view* x, const int64_t* slots, const jhq_q8_rows* cache, cudaStream_t s) {
    q8_check_view(x, "q8_write: x");
    q8_check_rows(cache, "q8_write: cache");
    if (cache->dim != x->cols) fail(JHQ_EINVAL, "q8_write: x's rows must be as long as the cache's");
    if (!slots && x->rows > cache->rows) fail(JHQ_EINVAL, "q8_write: more rows than the cache has");
    if ((uintptr_t)slots % 8) fail(JHQ_EINVAL, "q8_write: slots are not aligned to 8 bytes");
    if (x->rows == 0 || cache->rows == 0) return;
    if (x->rows * cache->groups > INT32_MAX) fail(JHQ_EINVAL, "q8_write: too many rows");
    by_type(x->type, [&](auto t) {
        using T = decltype(t);
        write_kernel<T><<<(unsigned)(x->rows * cache->groups), THREADS, 0, s>>>(
            (const T*)x->data, x->ld, slots, cache->q, cache->ld, cache->scale, cache->rows,
            cache->groups, (int)(cache->dim / cache->groups));
    });
    JHQ_LAUNCH_CHECK();
    count_launch();
}

void q8_read(const jhq_q8_rows* cache, const int64_t* slots, const jhq_view* out, cudaStream_t s) {
    q8_check_rows(cache, "q8_read: cache");
    q8_check_view(out, "q8_read: out");
    if (cache->dim != out->cols) fail(JHQ_EINVAL, "q8_read: out's rows must be as long as the cache's");
    if (!slots && out->rows > cache->rows) fail(JHQ_EINVAL, "q8_read: more rows than the cache has");
    if ((uintptr_t)slots % 8) fail(JHQ_EINVAL, "q8_read: slots are not aligned to 8 bytes");
    if (out->rows == 0) return;
    if (out->rows > INT32_MAX) fail(JHQ_EINVAL, "q8_read: too many rows");
    by_type(out->type, [&](auto t) {
        using T = decltype(t);
        read_kernel<T><<<(unsigned)out->rows, THREADS, 0, s>>>(
            cache->q, cache->ld, cache->scale, cache->rows, slots, (T*)out->data, out->ld,
            cache->groups, (int)(cache->dim / cache->groups));
    });
    JHQ_LAUNCH_CHECK();
    count_launch();
}

}  // namespace jhq
