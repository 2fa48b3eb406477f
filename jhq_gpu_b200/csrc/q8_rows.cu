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

#include <algorithm>
#include <cmath>
#include <string>

#include "kernels.cuh"
#include "q8.h"
#include "q8_launch.cuh"

namespace jhq {

static constexpr int64_t MAX_ROW = 1ll << 30;             // values: indexes within a row are 32-bit

void q8_check_view(const jhq_view* v, const char* what) {
    const std::string w(what);
    if (!v) fail(JHQ_EINVAL, w + ": null");
    if (v->type != JHQ_F32 && v->type != JHQ_F16 && v->type != JHQ_BF16)
        fail(JHQ_EINVAL, w + ": unknown type");
    if (v->rows < 0 || v->cols < 1 || v->cols > MAX_ROW)
        fail(JHQ_EINVAL, w + ": rows must be >= 0 and cols in 1..2^30");
    if (v->rows > 1 && v->ld < v->cols) fail(JHQ_EINVAL, w + ": ld is smaller than a row");
    if (v->rows > 0 && !v->data) fail(JHQ_EINVAL, w + ": null data");
    if ((uintptr_t)v->data % (v->type == JHQ_F32 ? 4 : 2))
        fail(JHQ_EINVAL, w + ": data is not aligned to its type");
}

void q8_check_rows(const jhq_q8_rows* r, const char* what) {
    const std::string w(what);
    if (!r) fail(JHQ_EINVAL, w + ": null");
    if (r->rows < 0 || r->dim < 1 || r->dim > MAX_ROW)
        fail(JHQ_EINVAL, w + ": rows must be >= 0 and dim in 1..2^30");
    if (r->groups < 1 || r->dim % r->groups) fail(JHQ_EINVAL, w + ": groups must divide dim");
    if (r->rows > 1 && r->ld < r->dim) fail(JHQ_EINVAL, w + ": ld is smaller than a row");
    if (r->rows > 0 && (!r->q || !r->scale)) fail(JHQ_EINVAL, w + ": null buffer");
    if ((uintptr_t)r->scale % 4) fail(JHQ_EINVAL, w + ": scale is not aligned to its type");
}

namespace {

constexpr uint32_t INF_BITS = 0x7f800000u;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_float(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void pack2(uint32_t* p, float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    *p = *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void pack2(uint32_t* p, float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    *p = *reinterpret_cast<const uint32_t*>(&h);
}

// Two 16-bit values of a word, as floats.
__device__ __forceinline__ void unpack2(uint32_t w, float* out, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    out[0] = f.x;
    out[1] = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t w, float* out, __nv_bfloat16) {
    out[0] = __uint_as_float(w << 16);
    out[1] = __uint_as_float(w & 0xffff0000u);
}

// How a thread touches its piece of V values at p, of which the first `left` are
// the row's: single values (V = 1), whole pieces of 16 bytes of x (all or nothing
// is the row's), the same with a ragged last one, value by value, or whole pieces
// that are all there.
enum Access { SINGLE, WHOLE, RAGGED, FULL };

__device__ __forceinline__ uint4 load16(const void* p) {     // not kept in L1, which is left to the weights
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
// Loads under a predicate, zeros without: a branch around each would part a
// thread's loads from one another. STREAM: read once, past L1.
template <bool STREAM>
__device__ __forceinline__ void load_if(bool ok, const uint4* p, uint4& v) {
    if (STREAM)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                     "@p ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
                     : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)ok));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                     "@p ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
                     : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)ok));
}

template <Access A, int V, bool STREAM, class T>
__device__ __forceinline__ void load(const T* p, int left, float* out) {
    constexpr int B = V * (int)sizeof(T);
    if constexpr (A == SINGLE) {
        out[0] = left > 0 ? to_float(*p) : 0.0f;
    } else {
        left -= A == RAGGED ? V - 1 : 0;                   // whole pieces alone; mend() follows
        uint32_t v[B / 4];
        static_assert(B % 16 == 0, "16-bit rows may have float32 weights and residuals, float32 rows only such");
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            const uint4* from = reinterpret_cast<const uint4*>(p) + i;
            uint4 u;
            if constexpr (A != FULL) load_if<STREAM>(left > 0, from, u);
            else u = STREAM ? load16(from) : *from;
            v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; i += 2) unpack2(v[i / 2], out + i, T());
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = __uint_as_float(v[i]);
        }
    }
}
// The values of a ragged piece, once a thread's whole pieces are on their way.
template <Access A, int V, class T>
__device__ __forceinline__ void mend(const T* p, int left, float* out) {
    if (A == RAGGED && left > 0 && left < V) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = i < left ? to_float(p[i]) : 0.0f;
    }
}
// odd: p is off its boundary, and the values are stored one by one.
template <Access A, int V, class T>
__device__ __forceinline__ void put(T* p, int left, const float* in, bool odd) {
    constexpr int B = V * (int)sizeof(T);
    if (A != SINGLE && (odd || (A == RAGGED && left < V))) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) from_float(p + i, in[i]);
        return;
    }
    if (left <= 0) return;
    alignas(16) T v[V];
    if constexpr (sizeof(T) == 2 && V > 1) {               // two at a time
#pragma unroll
        for (int i = 0; i < V; i += 2) pack2(reinterpret_cast<uint32_t*>(v) + i / 2, in[i], in[i + 1], T());
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) from_float(&v[i], in[i]);
    }
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
    } else {
        p[0] = v[0];
    }
}
template <Access A, int V>
__device__ __forceinline__ void put_bytes(int8_t* p, int left, const uint32_t* v, bool odd) {
    if (A != SINGLE && (odd || (A == RAGGED && left < V))) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) p[i] = (int8_t)v[i];
        return;
    }
    if (left <= 0) return;
    if constexpr (V == 1) {
        p[0] = (int8_t)v[0];
    } else {
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            w[i] = __byte_perm(__byte_perm(v[4 * i], v[4 * i + 1], 0x0040), __byte_perm(v[4 * i + 2], v[4 * i + 3], 0x0040), 0x5410);
        if constexpr (V == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
}

// rint(g * (127 * (1 / a))) in the low byte of the result: adding 1.5 * 2^23
// rounds to the nearest whole number, ties to even. A tiny a would make 1 / a
// infinite: both are scaled by 2^64 first (exact).
struct Quant {
    float pre, inv;
    bool fine;                                           // a is positive and finite; else all bytes are 0
    __device__ explicit Quant(float a) {
        pre = a < 1e-30f ? 0x1p64f : 1.0f;
        fine = a > 0.0f && __float_as_uint(a) < INF_BITS;
        inv = fine ? 127.0f * __frcp_rn(a * pre) : 0.0f;
    }
    __device__ uint32_t plain(float g) const { return __float_as_uint(g * inv + 12582912.0f); }   // fine, pre = 1
    __device__ uint32_t operator()(float g) const { return fine ? plain(g * pre) : 0u; }
};
__device__ __forceinline__ float max_nan(float a, float b) {   // of a and |b|; NaN if either is
    float r;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Sum and maximum over a team: up to 32 lanes of a warp, or the block (of TEAM
// threads, or of any number: TEAM = 0).
template <int TEAM>
__device__ __forceinline__ float2 team_sum_max(float sum, float top, float2* red) {
#pragma unroll
    for (int o = (TEAM && TEAM < 32 ? TEAM : 32) / 2; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        top = max_nan(top, __shfl_xor_sync(~0u, top, o));
    }
    if (TEAM == 0 || TEAM > 32) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) red[warp] = make_float2(sum, top);
        __syncthreads();
        const float2 v = lane < (int)blockDim.x / 32 ? red[lane] : make_float2(0.0f, 0.0f);
        sum = v.x;
        top = v.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sum += __shfl_xor_sync(~0u, sum, o);
            top = max_nan(top, __shfl_xor_sync(~0u, top, o));
        }
    }
    return make_float2(sum, top);
}
// The power of two (2^-128 .. 2^126) that brings a positive h into 1/2 .. 1 (a subnormal one as near as it goes): no
// product of it with a finite weight overflows then.
__device__ __forceinline__ float to_unit(float h) { return ldexpf(1.0f, -max(ilogbf(h) + 1, -126)); }
__device__ __forceinline__ bool is_finite(float a) { return (__float_as_uint(a) & 0x7fffffffu) < INF_BITS; }

struct Args {
    const void* x;
    int64_t ldx;
    const void *res, *weight;                            // null: none, ones
    void* res_out;                                       // null: not wanted; may be res
    int64_t ldr, ldo;
    int w32;                                             // weight is float32, else x's type
    float eps;
    int8_t* q;
    int64_t ldq;
    float* scale;
    const int64_t* slots;
    int64_t nslots;
    bool odd_out, odd_q;                                 // res_out's or q's rows begin off the accesses' boundaries
    unsigned teams;                                      // rows times groups
    int groups, d;                                       // d: values of a group
};

constexpr int SMS = 148;
// One pass over a row (a group, when the cache is written): a team of TPR threads
// holds EPT values each in registers, so x and the residual are read once and
// every output is written once. Bound by those bytes, as long as a thread has
// enough values that the instructions spent on a row and not on a value (addresses,
// the team's reductions, the reciprocal) stay few: 27 a value in all for a norm. Short
// groups share a warp, rows to 1024 values have a warp, longer ones a block, of as many
// threads as they need (TEAM = 0) or, for single values, of TEAM, so that their
// addresses differ by constants (20000 x 1001 in bfloat16, packed: 84 us without, 60 us
// with). Registers are held to 64, and to 80 where a thread holds 32 float32 values or
// residuals, for the whole pieces of most rows; the RAGGED norms of 32 values spill 130 to
// 220 bytes a thread under it in 16-bit types (20000 x 1003 in padded rows: 69 us).
// Measured: norm of 65536 x 4096 in bfloat16 with its residual 299 us (6.28 TB/s, 0.96 of
// a copy's rate), with a float32 residual 476 us (6.20 TB/s); 1 x 4096 2.5 us; 65536 x 1024
// 78 us (6.03 TB/s); cache write of 65536 x 16 x 128 in bfloat16 71 us (5.64 TB/s), of odd
// groups, value by value, 30000 x 7 x 333 95 us (2.21 TB/s).
constexpr int SHARED_BLOCK = 128, MOST_THREADS = 512;
template <class T, class R, int TEAM, int EPT, Access A, bool NORM>
__global__ void __maxnreg__(EPT == 32 && (sizeof(T) == 4 || sizeof(R) == 4) ? 80 : 64) rows_kernel(const __grid_constant__ Args a) {
    constexpr int V = A == SINGLE ? 1 : 16 / (int)sizeof(T), NV = EPT / V;
    let_next_start();
    before_memory();
    __shared__ float2 red[3][32];
    constexpr bool SHARED = TEAM && TEAM <= 32;            // blocks of several teams
    const int TPR = TEAM ? TEAM : (int)blockDim.x, me = SHARED ? threadIdx.x % TPR : threadIdx.x;
    const unsigned team = SHARED ? blockIdx.x * (SHARED_BLOCK / TPR) + threadIdx.x / TPR : blockIdx.x;
    const bool in = team < a.teams;                        // else the team only keeps the warp's shuffles company
    const int64_t row = !in ? 0 : a.groups == 1 ? team : team / (unsigned)a.groups;
    const int64_t off = !in ? 0 : (int64_t)(team - (unsigned)row * (unsigned)a.groups) * a.d;   // of the group
    const int64_t slot = !in ? -1 : a.slots ? a.slots[row] : row;
    const int d = in ? a.d : 0;
    auto at = [&](int i) { return (i * TPR + me) * V; };   // the thread's i-th piece

    float h[EPT];
    const T* x = static_cast<const T*>(a.x) + row * a.ldx + off;
#pragma unroll
    for (int i = 0; i < NV; ++i) load<A, V, true>(x + at(i), d - at(i), h + i * V);
#pragma unroll
    for (int i = 0; i < NV; ++i) mend<A, V>(x + at(i), d - at(i), h + i * V);
    if (NORM && a.res) {
        const R* res = static_cast<const R*>(a.res) + row * a.ldr;
        float r[EPT];
#pragma unroll
        for (int i = 0; i < NV; ++i) load<A, V, true>(res + at(i), d - at(i), r + i * V);
#pragma unroll
        for (int i = 0; i < NV; ++i) mend<A, V>(res + at(i), d - at(i), r + i * V);
#pragma unroll
        for (int i = 0; i < EPT; ++i) h[i] += r[i];
    }
    if (NORM && a.res_out) {
        R* o = static_cast<R*>(a.res_out) + row * a.ldo;
#pragma unroll
        for (int i = 0; i < NV; ++i) put<A, V>(o + at(i), d - at(i), h + i * V, a.odd_out);
    }
    auto weigh = [&](float* w, int i) {                    // the weights of piece i
        if (!NORM || !a.weight) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = 1.0f;
        } else if (a.w32) {
            load<A, V, false>(static_cast<const float*>(a.weight) + at(i), d - at(i), w);
            mend<A, V>(static_cast<const float*>(a.weight) + at(i), d - at(i), w);
        } else {
            load<A, V, false>(static_cast<const T*>(a.weight) + at(i), d - at(i), w);
            mend<A, V>(static_cast<const T*>(a.weight) + at(i), d - at(i), w);
        }
    };
    float sum = 0.0f, top = 0.0f;
    auto gather = [&](float by) {
        sum = top = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[V];
            weigh(w, i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = h[i * V + j] * by;
                if (NORM) sum = __fmaf_rn(v, v, sum);
                top = max_nan(top, v * w[j]);
            }
        }
    };
    gather(1.0f);
    const float2 st = team_sum_max<TEAM>(sum, top, red[0]);
    float top_g = st.y, by = 1.0f;
    double sum_sq = st.x;
    const bool odd = NORM && !(st.x >= 0x1p-90f && st.x <= 0x1p120f && top_g >= 0x1p-100f && top_g <= 0x1p120f);
    if (NORM && __any_sync(~0u, odd)) {                    // the teams of a warp go together
        // near the ends of float32's range: again with h scaled by a power of two
        float hm = 0.0f;
#pragma unroll
        for (int i = 0; i < EPT; ++i) hm = max_nan(hm, h[i]);
        const float htop = team_sum_max<TEAM>(0.0f, hm, red[1]).y;
        if (odd && htop > 0.0f && is_finite(htop)) by = to_unit(htop);
        gather(by);
        const float2 s2 = team_sum_max<TEAM>(sum, top, red[2]);
        top_g = s2.y;
        sum_sq = s2.x;
    }
    const Quant quant(top_g);
    const bool wanted = in && slot >= 0 && (NORM || slot < a.nslots);
    int8_t* q = a.q + (wanted ? slot * a.ldq + off : 0);
    const int keep = wanted ? d : 0;
    if (quant.fine && quant.pre == 1.0f && by == 1.0f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[V];
            weigh(w, i);
            uint32_t b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = quant.plain(NORM ? h[i * V + j] * w[j] : h[i * V + j]);
            put_bytes<A, V>(q + at(i), keep - at(i), b, a.odd_q);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[V];
            weigh(w, i);
            uint32_t b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = quant(NORM ? h[i * V + j] * by * w[j] : h[i * V + j]);
            put_bytes<A, V>(q + at(i), keep - at(i), b, a.odd_q);
        }
    }
    if (me == 0 && wanted) {
        float step = top_g / 127.0f;
        if (NORM) step = by == 1.0f ? top_g / (127.0f * sqrtf((float)sum_sq / (float)a.d + a.eps))
                                    : (float)((double)top_g / (127.0 * sqrt(sum_sq / a.d + (double)a.eps * by * by)));
        a.scale[slot * a.groups + (int)(off / a.d)] = !is_finite(top_g) ? __uint_as_float(0x7fffffffu) : top_g > 0.0f ? step : 0.0f;
    }
}

// Rows longer than a block's registers: the row is read twice (thrice near the
// ends of float32's range), value by value: bound by instructions. Measured: norm of 4096 x
// 32768 in bfloat16 336 us (2.8 TB/s).
constexpr int LONG_THREADS = 1024;
template <class T, class R, bool NORM>
__global__ void __launch_bounds__(LONG_THREADS) long_rows_kernel(const __grid_constant__ Args a) {
    let_next_start();
    before_memory();
    __shared__ float2 red[3][32];
    const int64_t row = a.groups == 1 ? blockIdx.x : blockIdx.x / (unsigned)a.groups;
    const int g = a.groups == 1 ? 0 : (int)(blockIdx.x % (unsigned)a.groups);
    const int64_t to = a.slots ? a.slots[row] : row;
    if (to < 0 || (!NORM && to >= a.nslots)) return;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx + (int64_t)g * a.d;
    const R* res = a.res ? static_cast<const R*>(a.res) + row * a.ldr : nullptr;
    R* res_out = a.res_out ? static_cast<R*>(a.res_out) + row * a.ldo : nullptr;
    int8_t* q = a.q + to * a.ldq + (int64_t)g * a.d;
    auto h_of = [&](int j) {
        const float v = to_float(x[j]);
        return NORM && res ? v + to_float(res[j]) : v;
    };
    auto w_of = [&](int j) {
        if (!NORM || !a.weight) return 1.0f;
        return a.w32 ? static_cast<const float*>(a.weight)[j] : to_float(static_cast<const T*>(a.weight)[j]);
    };
    auto gather = [&](float by, float2* r) {
        float sum = 0.0f, top = 0.0f;
#pragma unroll 4
        for (int j = threadIdx.x; j < a.d; j += LONG_THREADS) {
            const float h = h_of(j) * by;
            if (NORM) sum = __fmaf_rn(h, h, sum);
            top = max_nan(top, h * w_of(j));
        }
        return team_sum_max<0>(sum, top, r);
    };
    const float2 st = gather(1.0f, red[0]);
    float top_g = st.y, by = 1.0f, step = top_g / 127.0f;
    if (NORM) {
        step = top_g / (127.0f * sqrtf(st.x / (float)a.d + a.eps));
        if (!(st.x >= 0x1p-90f && st.x <= 0x1p120f && top_g >= 0x1p-100f && top_g <= 0x1p120f)) {
            float hm = 0.0f;
            for (int j = threadIdx.x; j < a.d; j += LONG_THREADS) hm = max_nan(hm, h_of(j));
            const float htop = team_sum_max<0>(0.0f, hm, red[1]).y;
            if (htop > 0.0f && is_finite(htop)) {
                by = to_unit(htop);
                const float2 s2 = gather(by, red[2]);
                top_g = s2.y;
                step = (float)((double)top_g / (127.0 * sqrt((double)s2.x / a.d + (double)a.eps * by * by)));
            }
        }
    }
    const Quant quant(top_g);
#pragma unroll 4
    for (int j = threadIdx.x; j < a.d; j += LONG_THREADS) {
        const float h = h_of(j), w = w_of(j);
        if (NORM && res_out) from_float(res_out + j, h);
        q[j] = (int8_t)quant(h * by * w);
    }
    if (threadIdx.x == 0)
        a.scale[to * a.groups + g] = !is_finite(top_g) ? __uint_as_float(0x7fffffffu) : top_g > 0.0f ? step : 0.0f;
}

template <class T, class R, int TEAM, int EPT, Access A, bool NORM>
void launch_team(const Args& a, cudaStream_t s) {
    if constexpr (A == WHOLE)
        if (a.d == TEAM * EPT) return launch_team<T, R, TEAM, EPT, FULL, NORM>(a, s);
    constexpr unsigned per = TEAM <= 32 ? SHARED_BLOCK / TEAM : 1;
    launch_q8(rows_kernel<T, R, TEAM, EPT, A, NORM>, dim3((a.teams - 1) / per + 1), TEAM <= 32 ? SHARED_BLOCK : TEAM, 0, 0, s, a);
}
template <class T, class R, int EPT, Access A, bool NORM>
void launch_block(const Args& a, cudaStream_t s) {
    if constexpr (A == WHOLE)
        if (a.d % (32 * EPT) == 0) return launch_block<T, R, EPT, FULL, NORM>(a, s);
    launch_q8(rows_kernel<T, R, 0, EPT, A, NORM>, dim3(a.teams), (a.d - 1) / EPT / 32 * 32 + 32, 0, 0, s, a);
}
// Many rows: the smallest team whose registers hold a row at 32 values a thread (at 16 and 8 the instructions spent on
// a row bind: 65536 x 4096 in bfloat16 took 441 us with 16, 303 us with 32), at 16 single values, whose registers
// 32 do not fit. Few rows: 8 or 16 values a thread where all rows then run at once (1 x 4096: 2.5 us with 8, 3.8 us with
// 32; 2000 x 1024: 4.5 us with 16, 5.7 us with 32; but 4000 x 1024: 8.3 and 6.9 us).
template <class T, class R, Access A, bool NORM>
void launch_rows(const Args& a, cudaStream_t s) {
    const int d = a.d;
    // whether all rows, `each` values a thread, are on the SMs at once
    const auto fits = [&](int each) { return d > 256 && d <= each * MOST_THREADS && (int64_t)a.teams * ((d - 1) / each + 1) <= SMS * 1024; };
    if constexpr (!NORM) {                                 // short groups, of which a cache has many
        if (d <= 16) return launch_team<T, R, 2, 8, A, NORM>(a, s);
        if (d <= 32) return launch_team<T, R, 4, 8, A, NORM>(a, s);
        if (d <= 64) return launch_team<T, R, A == SINGLE ? 4 : 2, A == SINGLE ? 16 : 32, A, NORM>(a, s);
    }
    if (fits(8)) return launch_block<T, R, 8, A, NORM>(a, s);
    if (fits(16)) return launch_block<T, R, 16, A, NORM>(a, s);
    if constexpr (A == SINGLE) {
        if (d <= 128) return launch_team<T, R, 8, 16, A, NORM>(a, s);
        if (d <= 256) return launch_team<T, R, 16, 16, A, NORM>(a, s);
        if (d <= 512) return launch_team<T, R, 32, 16, A, NORM>(a, s);
        if (d <= 1024) return launch_team<T, R, 64, 16, A, NORM>(a, s);
        if (d <= 2048) return launch_team<T, R, 128, 16, A, NORM>(a, s);
        if (d <= 4096) return launch_team<T, R, 256, 16, A, NORM>(a, s);
        if (d <= 8192) return launch_team<T, R, 512, 16, A, NORM>(a, s);
    } else {
        if (d <= 128) return launch_team<T, R, 4, 32, A, NORM>(a, s);
        if (d <= 256) return launch_team<T, R, 8, 32, A, NORM>(a, s);
        if (d <= 512) return launch_team<T, R, 16, 32, A, NORM>(a, s);
        const bool wide = NORM && sizeof(T) == 4 && a.res;
        if (d <= 1024 && !wide) return launch_team<T, R, 32, 32, A, NORM>(a, s);
        // float32 rows and residuals, 128 bytes of each a thread, leave too few threads room
        // (16384 x 2560: 95 us with 32 values, 86 us with 16; 4099 x 1024: 14.1 and 11.3 us)
        if (wide && d <= 16 * MOST_THREADS) return launch_block<T, R, 16, A, NORM>(a, s);
        if (d <= 32 * MOST_THREADS) return launch_block<T, R, 32, A, NORM>(a, s);
    }
    launch_q8(long_rows_kernel<T, R, NORM>, dim3(a.teams), LONG_THREADS, 0, 0, s, a);
}

bool on_bytes(const void* p, int64_t ld, int size, int rows_of, int64_t rows) {
    return (uintptr_t)p % rows_of == 0 && (rows <= 1 || ld * size % rows_of == 0);
}

// Reads rows back: V values of a row a thread (32 bytes of output where rows
// allow it: 16 took 125 us for the case below), tpr threads a row, several rows a thread
// when there are many. Bound by the bytes: one in, sizeof(T) out a value. Measured: 65536 x
// 2048 bfloat16 values from rows in any order 69 us (5.80 TB/s).
template <class T, int V>
struct alignas(V * sizeof(T)) Piece {
    T v[V];
};
// V bytes of a row, and value i of them as a float: the byte + 128 as the low bits
// of 2^23, less 2^23 + 128 (exact); half the cost of a conversion.
template <int V>
struct Bytes {
    uint32_t w[(V + 3) / 4];
    __device__ __forceinline__ void load(const int8_t* p) {
        if constexpr (V == 16) {
            const uint4 v = load16(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (V == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ float value(int i) const {
        return __uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4B000000u, 0x7440 + i % 4)) - 8388736.0f;
    }
};

template <class T, int V, int U>
__global__ void __launch_bounds__(256, U == 1 ? 8 : V <= 4 ? 5 : 6)
read_kernel(const int8_t* q, int64_t ldq, const float* scale, int64_t nslots, const int64_t* slots, T* out, int64_t ldo,
            int64_t rows, int tpr, int groups, int gdim, int dim) {
    let_next_start();
    before_memory();
    const int per = 256 / tpr;
    const int64_t row0 = (int64_t)blockIdx.x * per * U + threadIdx.x / tpr;
    const int8_t* from[U];
    const float* fac[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * per, slot = row >= rows ? -1 : slots ? slots[row] : row;
        const bool there = slot >= 0 && slot < nslots;
        from[u] = there ? q + slot * ldq : nullptr;
        fac[u] = scale + (there ? slot * groups : 0);
    }
    for (int j = (blockIdx.y * tpr + threadIdx.x % tpr) * V; j < dim; j += (int)gridDim.y * tpr * V) {
        Bytes<V> b[U];
        float sc[U];
        const unsigned g = groups == 1 ? 0u : (unsigned)j / (unsigned)gdim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            sc[u] = 0.0f;
            b[u] = Bytes<V>{};
            if (from[u]) {
                b[u].load(from[u] + j);
                sc[u] = fac[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = row0 + u * per;
            if (row >= rows) break;
            T* o = out + row * ldo + j;
            alignas(32) T v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) from_float(&v[i], sc[u] * b[u].value(i));
            if constexpr (V * sizeof(T) == 32) {
                const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                             :: "l"(o), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                                "r"(w[7]) : "memory");
            } else {
                *reinterpret_cast<Piece<T, V>*>(o) = *reinterpret_cast<const Piece<T, V>*>(v);
            }
        }
    }
}

// The four bytes at p (any address) of a buffer [first, end), byte by byte, zeros outside.
__device__ __noinline__ uint32_t word_edge(const int8_t* p, const int8_t* first, const int8_t* end) {
    uint32_t v = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i)
        if (p + i >= first && p + i < end) v |= (uint32_t)(uint8_t)p[i] << (8 * i);
    return v;
}

// Rows at odd addresses or of odd groups: a thread takes the V values of an aligned
// 32 bytes of output (the first and last piece of a row: of what the row has of
// them) and gathers their bytes from aligned words. WALK: groups shorter than a piece.
// Measured: 30000 x 7 x 333 bfloat16 values 96 us (2.18 TB/s; 238 us value by value),
// bound by instructions.
template <class T, bool WALK>
__global__ void __launch_bounds__(256)
read_odd_kernel(const int8_t* q, int64_t ldq, const int8_t* end, const float* scale, int64_t nslots,
                const int64_t* slots, T* out, int64_t ldo, int64_t rows, int tpr, int groups, int gdim, int dim) {
    constexpr int V = 32 / (int)sizeof(T);
    let_next_start();
    before_memory();
    const int64_t row = (int64_t)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
    if (row >= rows) return;
    const int64_t slot = slots ? slots[row] : row;
    const bool there = slot >= 0 && slot < nslots;
    const int8_t* const from = q + (there ? slot * ldq : 0);
    const float* const fac = scale + (there ? slot * groups : 0);
    T* const o = out + row * ldo;
    const int skew = (int)((uintptr_t)o % 32 / sizeof(T));             // values of the first piece before the row
    for (int j0 = (blockIdx.y * tpr + threadIdx.x % tpr) * V - skew; j0 < dim; j0 += (int)gridDim.y * tpr * V) {
        uint32_t w[V / 4 + 1];
        const int8_t* const p = from + j0;
        const int off = (int)((uintptr_t)p & 3);
        const int8_t* const a = p - off;
        const bool inside = j0 >= 0 && a >= q && a + V + 4 <= end;      // whole words of the buffer
#pragma unroll
        for (int i = 0; i <= V / 4; ++i) w[i] = there && inside ? reinterpret_cast<const uint32_t*>(a)[i] : 0u;
        const int first = max(j0, 0), g = groups == 1 ? 0 : (int)((unsigned)first / (unsigned)gdim);
        const int turn = groups == 1 ? dim : (g + 1) * gdim;            // where the next group begins
        const float sc = there ? fac[g] : 0.0f, sc1 = there && turn < min(j0 + V, dim) ? fac[g + 1] : 0.0f;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * off);
        if (there && !inside) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) w[i] = word_edge(p + 4 * i, from, from + dim);
        }
        alignas(16) T v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = j0 + i;
            float f = j < turn ? sc : sc1;
            if (WALK && there && j >= turn && j < dim) f = fac[(unsigned)j / (unsigned)gdim];
            const float b = __uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4B000000u, 0x7440 + i % 4)) - 8388736.0f;
            from_float(&v[i], there ? f * b : 0.0f);
        }
        if (j0 >= 0 && j0 + V <= dim) {
            reinterpret_cast<uint4*>(o + j0)[0] = reinterpret_cast<const uint4*>(v)[0];
            reinterpret_cast<uint4*>(o + j0)[1] = reinterpret_cast<const uint4*>(v)[1];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (j0 + i >= 0 && j0 + i < dim) o[j0 + i] = v[i];
        }
    }
}

template <class T>
void read_odd(const jhq_q8_rows* c, const int64_t* slots, const jhq_view* out, cudaStream_t s) {
    constexpr int V = 32 / (int)sizeof(T);
    const int gdim = (int)(c->dim / c->groups), dim = (int)c->dim;
    const int64_t pieces = ceil_div(dim, V) + 1;
    const int tpr = std::min(256, next_pow2((int)std::min<int64_t>(256, pieces)));
    const int64_t blocks = ceil_div(out->rows, 256 / tpr);
    if (blocks > INT32_MAX) fail(JHQ_EINVAL, "q8_read: too many rows");
    const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(65535, ceil_div(pieces, tpr)));
    launch_q8(gdim < V && c->groups > 1 ? read_odd_kernel<T, true> : read_odd_kernel<T, false>, grid, 256, 0, 0, s, c->q, c->ld, c->rows ? c->q + (c->rows - 1) * c->ld + dim : c->q, c->scale, c->rows, slots, (T*)out->data, out->ld,
        out->rows, tpr, c->groups, gdim, dim);
}

template <class T, int V>
bool try_read(const jhq_q8_rows* c, const int64_t* slots, const jhq_view* out, cudaStream_t s) {
    const int gdim = (int)(c->dim / c->groups), dim = (int)c->dim;
    if (gdim % V || !on_bytes(c->q, c->ld, 1, V, c->rows) ||
        !on_bytes(out->data, out->ld, sizeof(T), V * (int)sizeof(T), out->rows))
        return false;
    const int tpr = std::min(256, next_pow2((int)ceil_div(dim, V)));
    // several rows a thread once that leaves every SM eight blocks
    constexpr int MORE = V <= 4 ? 4 : 2;
    const int U = out->rows >= (int64_t)MORE * 8 * SMS * (256 / tpr) ? MORE : 1;
    const int64_t blocks = ceil_div(out->rows, 256 / tpr * U);
    if (blocks > INT32_MAX) fail(JHQ_EINVAL, "q8_read: too many rows");
    const dim3 grid((unsigned)blocks, (unsigned)(U > 1 ? 1 : std::min<int64_t>(65535, ceil_div(dim, tpr * V))));
    launch_q8(U > 1 ? read_kernel<T, V, MORE> : read_kernel<T, V, 1>, grid, 256, 0, 0, s, c->q, c->ld, c->scale, c->rows, slots, (T*)out->data, out->ld, out->rows, tpr, c->groups, gdim, dim);
    return true;
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
    Args a{};
    a.x = x->data;
    a.ldx = x->ld;
    if (residual) { a.res = residual->data; a.ldr = residual->ld; }
    if (residual_out) { a.res_out = residual_out->data; a.ldo = residual_out->ld; }
    if (weight) { a.weight = weight->data; a.w32 = weight->type == JHQ_F32; }
    a.eps = eps;
    a.q = out->q;
    a.ldq = out->ld;
    a.scale = out->scale;
    a.teams = (unsigned)x->rows;
    a.groups = 1;
    a.d = (int)x->cols;
    by_type(x->type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / (int)sizeof(T);
        auto go = [&](auto r) {
            using R = decltype(r);
            const bool vec = on_bytes(a.x, a.ldx, sizeof(T), 16, x->rows) && on_bytes(a.res, a.ldr, sizeof(R), 16, x->rows) &&
                             (uintptr_t)a.weight % 16 == 0;
            a.odd_q = !on_bytes(a.q, a.ldq, 1, V, x->rows);
            a.odd_out = !on_bytes(a.res_out, a.ldo, sizeof(R), 16, x->rows);
            if (!vec) launch_rows<T, R, SINGLE, true>(a, s);
            else if (a.d % V == 0) launch_rows<T, R, WHOLE, true>(a, s);
            else launch_rows<T, R, RAGGED, true>(a, s);
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
    if (x->rows > INT32_MAX / cache->groups) fail(JHQ_EINVAL, "q8_write: too many rows");
    Args a{};
    a.x = x->data;
    a.ldx = x->ld;
    a.q = cache->q;
    a.ldq = cache->ld;
    a.scale = cache->scale;
    a.slots = slots;
    a.nslots = cache->rows;
    a.teams = (unsigned)(x->rows * cache->groups);
    a.groups = cache->groups;
    a.d = (int)(cache->dim / cache->groups);
    by_type(x->type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / (int)sizeof(T);
        const bool vec = (a.groups == 1 || a.d % V == 0) && on_bytes(a.x, a.ldx, sizeof(T), 16, x->rows) &&
                         on_bytes(a.q, a.ldq, 1, V, cache->rows);
        if (!vec) launch_rows<T, T, SINGLE, false>(a, s);
        else if (a.d % V == 0) launch_rows<T, T, WHOLE, false>(a, s);
        else launch_rows<T, T, RAGGED, false>(a, s);
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
    by_type(out->type, [&](auto t) {
        using T = decltype(t);
        bool done = try_read<T, 32 / (int)sizeof(T)>(cache, slots, out, s);
        if constexpr (sizeof(T) == 2) done = done || try_read<T, 8>(cache, slots, out, s);
        if (!done && !try_read<T, 4>(cache, slots, out, s)) read_odd<T>(cache, slots, out, s);
    });
    JHQ_LAUNCH_CHECK();
    count_launch();
}

}  // namespace jhq
