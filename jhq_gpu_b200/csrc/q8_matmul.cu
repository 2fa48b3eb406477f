// q8_matmul.cu — the product of two sets of 8-bit rows,
//   out[t][n] = (sum_k x[t][k] w[n][k]) * sx[t] * sw[n] + bias[n],
// the sum exact in 32-bit integers on the tensor cores (tcgen05 kind::i8,
// operands in 128-byte K blocks staged in a ring of shared memory, sums in TMEM).
// Two kernels: panels (few tokens, where the weights' bytes count, or rows that
// TMA cannot fetch) and pairs (many tokens, where the multiply-adds count).
//
// Every wait on an mbarrier is bounded (about a second); one that gives up sets
// g_q8_error (jhq_q8_status) and the CTA's abort flag, which ends every role's
// loop. Before it leaves, a CTA lets the MMAs (bounded again) and the copies (for a
// fixed time) that it issued finish and frees its TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <mutex>

#include "kernels.cuh"
#include "q8.h"
#include "q8_launch.cuh"

namespace jhq {

namespace {

__device__ int g_q8_error;          // a bounded wait gave up

struct Epilogue {                   // what turns a sum into an output
    const float *sx, *sw, *bias;    // bias may be null
    void* out;
    int64_t ldo;
    int64_t T;
    int N, type;
    bool vec;                       // output rows begin on 16-byte boundaries
    long long limit;                // cycles that a wait may take
};

__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void store_out(const Epilogue& e, int64_t t, int n, float v) {
    const int64_t at = t * e.ldo + n;
    if (e.type == JHQ_F32) static_cast<float*>(e.out)[at] = v;
    else if (e.type == JHQ_F16) static_cast<__half*>(e.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(e.out)[at] = __float2bfloat16_rn(v);
}

constexpr long long WAIT_CYCLES = 1ll << 31;     // about a second

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(10000u) : "memory");   // may sleep so many ns
    return ok != 0;
}

// Bounded wait for the phase of parity `parity`; gives up when the CTA's abort
// flag is set or after `limit` cycles (at once if 0), which sets the flag and
// g_q8_error. The waits of a launch use its limit (WAIT_CYCLES unless a test shortens
// it); those for what was issued before an abort have abort = nullptr and WAIT_CYCLES.
__device__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort, long long limit = WAIT_CYCLES) {
    if (limit > 0 && mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (abort && *abort) return false;
        if (clock64() - t0 >= limit) {
            atomicExch(&g_q8_error, 1);
            if (abort) *abort = 1;
            return false;
        }
    } while (!mbar_try(bar, parity));
    return true;
}
// Before a CTA ends (all threads call it, their roles done): after an abort copies
// may still be in flight, whose barriers no longer tell; they land within microseconds
// and are given 2^24 cycles (8 ms).
__device__ __forceinline__ void settle(volatile int* abort) {
    __syncthreads();
    if (*abort) {
        if (threadIdx.x == 0) {
            const long long t0 = clock64();
            while (clock64() - t0 < (1ll << 24)) {}
        }
        __syncthreads();
    }
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared address `a` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t a, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}

// One lane of a converged warp; unlike a test of the lane's number, the compiler
// knows that a single thread goes on, and issues its MMAs and copies directly.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
// Stage and phase of a ring of N.
template <int N>
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == N) { s = 0; phase ^= 1u; }
    }
};

// K-major operand with 128-byte swizzle: rows of 128 bytes, 8-row groups 1024
// bytes apart, descriptor version 1, layout type 2.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <int CTAS>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add));
}
// The MMAs of one K block of `left` bytes, 32 each.
template <int CTAS>
__device__ __forceinline__ void mma_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int left, bool add) {
    if (left > 96) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_i8<CTAS>(d, a + 2 * k, b + 2 * k, idesc, k > 0 ? 1u : (uint32_t)add);
    } else {
        for (int k = 0; 32 * k < left; ++k) mma_i8<CTAS>(d, a + 2 * k, b + 2 * k, idesc, k > 0 ? 1u : (uint32_t)add);
    }
}
// s32 sums of s8 operands, both K-major.
constexpr uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld16(int* r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_ld32(int* r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}

// 16 outputs of channel n, tokens t .. t + 15, from the sums in r; lane l holds
// the scale of token t - at + l. Every lane of the warp calls it (n differs, t
// does not).
template <class O>
__device__ __forceinline__ void put16(const Epilogue& e, const int* r, int64_t t, float sx, int at, int n, float sw, float b) {
    const int left = (int)min((int64_t)16, e.T - t);
    O* o = static_cast<O*>(e.out) + t * e.ldo + n;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float v = (float)r[j] * __shfl_sync(~0u, sx, at + j) * sw;
        if (j < left && n < e.N) store(o + j * e.ldo, e.bias ? v + b : v);
    }
}
__device__ __forceinline__ void put16(const Epilogue& e, const int* r, int64_t t, float sx, int at, int n, float sw, float b) {
    if (t >= e.T) return;
    if (e.type == JHQ_BF16) put16<__nv_bfloat16>(e, r, t, sx, at, n, sw, b);
    else if (e.type == JHQ_F16) put16<__half>(e, r, t, sx, at, n, sw, b);
    else put16<float>(e, r, t, sx, at, n, sw, b);
}
// The scales of tokens t .. t + 32 COUNT - 1, 32 a register.
template <int COUNT>
__device__ __forceinline__ void get_scales(const Epilogue& e, int64_t t, float* sx) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const int64_t at = t + 32 * i + (threadIdx.x & 31);
        sx[i] = at < e.T ? e.sx[at] : 0.0f;
    }
}
// A warp's wait: lane 0 polls.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, long long limit) {
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort, limit);
    return __all_sync(~0u, ok);
}
// The wait of a panel's epilogue warps, through the whole of its products: the first
// one's lane 0 polls, the others sleep at a barrier. (With all eight polling, the barrier
// operations of the producers and the MMA thread took 0.16 us a K block.)
__device__ __forceinline__ bool epilogue_wait(uint32_t bar, uint32_t parity, bool polls, int threads) {
    bool ok = true;
    if (polls && (threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, nullptr);
    __syncwarp();
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((int)ok), "r"(threads) : "memory");
    return all != 0;
}

// ---- panels: few tokens, or rows at any address ------------------------------
//
// out^T = W x^T: a CTA takes 128 channels (the rows of the MMA) by TN tokens
// (its columns) over one slice of K; the S CTAs of a cluster take the S slices
// of one tile and add their sums through distributed shared memory, each
// finishing TN / S of the tokens. 32-bit integer sums are exact, so the split
// changes no output. Channels are the rows because few tokens would leave most of
// a 128-row MMA empty and 128 channels fill it with bytes that are read once anyway.
// Bound by the weights' bytes for long rows, by launch, ring and epilogue (3 to 5 us) for
// short ones. Measured: 1 x 8192 x 8192 13.7 us (4.9 TB/s, 0.75 of a copy's rate), 64 x 8192
// x 8192 16.3 us (4.2 TB/s), 16 x 16384 x 16384 43.5 us (6.2 TB/s), 1 x 1024 x 4096 3.9 us,
// 256 x 1024 x 4096 7.7 us; from rows at odd addresses, bound by the loads' latency, 1000 x 999
// x 1001 14.1 us, 4001 x 4001 x 4001 418 us (306 TOP/s, a tenth of the aligned rate; the kernel
// of 128 tokens spills 40 bytes a thread).
constexpr int BM = 128, BK = 128;
constexpr int LOADERS = 256;                               // threads of the epilogue, which load where TMA cannot
constexpr int LOAD_GROUPS = 2;                             // as many again, which load every other stage
constexpr int panel_threads(bool tma) { return 64 + LOADERS * (tma ? 1 : LOAD_GROUPS); }

template <int TN>
struct Panel {
    static constexpr int STAGE = (BM + TN) * BK;
    static constexpr int STAGES = TN == 16 ? 10 : TN == 32 ? 9 : TN == 64 ? 8 : 6;
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
    static constexpr uint32_t COLS = TN < 32 ? 32 : TN;
    static_assert(BM * TN * 4 <= STAGES * STAGE, "partial sums reuse the stages");
};

struct Rows8 {                       // operand rows for the loader threads
    const int8_t* p;
    int64_t ld, rows;
    const int8_t* end;               // behind the last row's last byte
};

// Past L1: each byte is loaded once (4001 x 4001 x 4001 packed: 418 us, through L1 428 us).
__device__ __forceinline__ uint4 load16_if(bool ok, const int8_t* p) {
    uint4 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)ok));
    return v;
}
// The 16 bytes at p, zeros outside [first, end): byte by byte.
__device__ __noinline__ uint4 load16_edge(const int8_t* p, const int8_t* first, const int8_t* end) {
    uint32_t w[4] = {};
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
        if (p + i >= first && p + i < end) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The loader warps copy bytes k .. k + 127 of BM rows of w (from w0) and TN rows of
// x (from x0) into swizzled 128-byte rows of shared memory, zeros beyond the rows'
// ends. Rows begin at any address: eight lanes take a row, each the aligned 16 bytes
// that its output begins in, and shift them together with the next lane's (the
// eighth reads one piece more). A piece may reach into a neighbouring row or the space
// between rows, whose bytes are cut off, but not out of the matrix: the few
// that straddle its first or last byte are read byte by byte. All pieces of a warp
// are in flight together.
template <int TN>
__device__ __forceinline__ void load_stage(const Rows8& w, const Rows8& x, int64_t w0, int64_t x0, int k, int K,
                                           uint32_t dst, int lw, int lane) {
    constexpr int STEP = LOADERS / 8, NW = BM / STEP, NX = (TN + STEP - 1) / STEP, N = NW + NX;
    const int c = lane & 7, r0 = lw * 4 + lane / 8;
    uint4 v[N], ex[N];
    int off[N];
#pragma unroll
    for (int b = 0; b < N; ++b) {
        const Rows8& m = b < NW ? w : x;
        const int r = r0 + STEP * (b < NW ? b : b - NW);
        const int64_t row = (b < NW ? w0 : x0) + r;
        const bool in = row < m.rows && (b < NW || r < TN);
        const int8_t* at = m.p + (in ? row : 0) * m.ld + k;
        off[b] = (int)((uintptr_t)at & 15);
        const int8_t* piece = at - off[b] + 16 * c;
        const int left = K - k + off[b] - 16 * c;          // of the row, from the piece's first byte
        const bool ok = in && left > 0, more = in && c == 7 && off[b] > 0 && left > 16;
        const bool whole = piece >= m.p && piece + 16 <= m.end, whole2 = piece + 32 <= m.end;
        v[b] = load16_if(ok && whole, piece);
        ex[b] = load16_if(more && whole2, piece + 16);
        if (ok && !whole) v[b] = load16_edge(piece, m.p, m.end);
        if (more && !whole2) ex[b] = load16_edge(piece + 16, m.p, m.end);
    }
#pragma unroll
    for (int b = 0; b < N; ++b) {
        const int r = r0 + STEP * (b < NW ? b : b - NW);
        uint32_t a[8] = {v[b].x, v[b].y, v[b].z, v[b].w};
        a[4] = __shfl_down_sync(~0u, v[b].x, 1);
        a[5] = __shfl_down_sync(~0u, v[b].y, 1);
        a[6] = __shfl_down_sync(~0u, v[b].z, 1);
        a[7] = __shfl_down_sync(~0u, v[b].w, 1);
        if (c == 7) { a[4] = ex[b].x; a[5] = ex[b].y; a[6] = ex[b].z; a[7] = ex[b].w; }
        const bool two = off[b] & 8, one = off[b] & 4;
#pragma unroll
        for (int i = 0; i < 6; ++i) a[i] = two ? a[i + 2] : a[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) a[i] = one ? a[i + 1] : a[i];
        const int sh = 8 * (off[b] & 3), left = K - k - 16 * c;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = __funnelshift_r(a[i], a[i + 1], sh);
            const int bytes = left - 4 * i;                // of the row, in this word
            if (bytes < 4) o[i] = bytes > 0 ? o[i] & ((1u << (8 * bytes)) - 1) : 0u;
        }
        if (b < NW || r < TN)
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};"
                         :: "r"(dst + (b < NW ? 0 : BM * BK) + r * 128 + ((c ^ (r & 7)) << 4)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                         : "memory");
    }
}

// Adds the S CTAs' sums of this thread's channel for the rank's TN / S tokens and
// finishes them, the two warps of a quarter every other batch; `part` is the shared
// address of the channel's first sum, sx holds the scales of the rank's tokens. The
// reads of up to eight tokens from all CTAs are in flight together.
template <int TN, int S>
__device__ __forceinline__ void join(const Epilogue& e, uint32_t part, int rank, int half, int64_t t0, const float* sx,
                                     int n, float sw, float b) {
    constexpr int PER = TN / S, R = PER < 16 ? (PER + 1) / 2 : 8;
    uint32_t from[S];
#pragma unroll
    for (int p = 0; p < S; ++p) from[p] = map_to(part, p);
#pragma unroll
    for (int k = 0; k < (PER + 2 * R - 1) / (2 * R); ++k) {
        const int i = (2 * k + half) * R, c = rank * PER + i;
        if (i >= PER || t0 + c >= e.T) break;
        int v[S][R];
#pragma unroll
        for (int p = 0; p < S; ++p)
#pragma unroll
            for (int j = 0; j < R; ++j)
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[p][j]) : "r"(from[p] + (c + j) * BM * 4));
#pragma unroll
        for (int j = 0; j < R; ++j) {
            int sum = 0;
#pragma unroll
            for (int p = 0; p < S; ++p) sum += v[p][j];
            const float f = (float)sum * __shfl_sync(~0u, sx[2 * k * R / 32], (i + j) % 32) * sw;
            if (t0 + c + j < e.T && n < e.N) store_out(e, t0 + c + j, n, e.bias ? f + b : f);
        }
    }
}

template <int TN, bool TMA>
__global__ void __launch_bounds__(panel_threads(TMA), 1)
panel_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Rows8 w,
             Rows8 x, int K, int S, int ttiles, Epilogue e) {
    using P = Panel<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[2 * P::STAGES + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort;
    const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * P::STAGES, done = empty0 + 8 * P::STAGES;
    const uint32_t base = smem_u32(smem);
    const int rank = (int)(blockIdx.x % (unsigned)S);
    const unsigned tile = blockIdx.x / (unsigned)S;
    const int64_t t0 = (int64_t)(tile % (unsigned)ttiles) * TN;
    const int m0 = (int)(tile / (unsigned)ttiles) * BM;
    const int nkb = (K + BK - 1) / BK;                     // K blocks; this CTA's: kb0 .. kb0 + nk - 1
    const int kb0 = (int)((int64_t)nkb * rank / S), nk = (int)((int64_t)nkb * (rank + 1) / S) - kb0;

    // Block kb0 + it of one operand into stage s (one thread; two share the copies).
    auto load = [&](int it, int s, bool of_w) {
        const uint32_t fb = full0 + 8 * s, dst = base + s * P::STAGE + (of_w ? 0 : BM * BK);
        mbar_expect(fb, of_w ? BM * BK : TN * BK);
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
            :: "r"(dst), "l"((uint64_t)(of_w ? &map_w : &map_x)), "r"((kb0 + it) * BK), "r"(of_w ? m0 : (int)t0), "r"(fb)
            : "memory");
    };
    auto produce = [&](int it, bool of_w) {                // blocks it, it + 1, ...; it = 0, or those of the ring are done
        const uint32_t odd = it == 0 ? 1u : 0u;            // the ring's second round waits for the first phase
        Ring<P::STAGES> r;                                 // begins at a multiple of STAGES, or ends there
        for (; it < nk; ++it, r.next()) {
            if (it >= P::STAGES && !mbar_wait(empty0 + 8 * r.s, r.phase ^ odd, &abort, e.limit)) break;
            load(it, r.s, of_w);
        }
    };

    if (tid == 0) {
        for (int i = 0; i < P::STAGES; ++i) {
            mbar_init(full0 + 8 * i, TMA ? 2 : LOADERS);
            mbar_init(empty0 + 8 * i, 1);
        }
        mbar_init(done, 1);
        abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        let_next_start();
        if (TMA) {                                         // the ring is filled before anything else is set up
            for (int it = 0; it < min(nk, P::STAGES); ++it)   // only into L2, where it can turn out to be any kernel's
                asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];"
                             :: "l"((uint64_t)&map_w), "r"((kb0 + it) * BK), "r"(m0) : "memory");
            before_memory();
            for (int it = 0; it < min(nk, P::STAGES); ++it) load(it, it, true);
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&tmem_slot)), "r"(P::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    before_memory();

    if (warp == 0) {
        if (TMA && elect_one()) produce(min(nk, P::STAGES), true);
    } else if (warp == 1) {
        if (elect_one()) {
            const uint64_t d0 = sw128_desc(base);
            int left = K - kb0 * BK;
            Ring<P::STAGES> r;
            for (int it = 0; it < nk; ++it, r.next(), left -= BK) {
                if (!mbar_wait(full0 + 8 * r.s, r.phase, &abort, e.limit)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t d = d0 + (uint64_t)(r.s * (P::STAGE >> 4));
                mma_block<1>(tmem, d, d + (BM * BK >> 4), idesc_i8(BM, TN), left, it > 0);
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                             :: "r"(empty0 + 8 * r.s) : "memory");
            }
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                         :: "r"(done) : "memory");
        }
    } else if (TMA) {
        if (warp == 2 && elect_one()) produce(0, false);
    } else {                                               // the other warps fill the stages
        const int group = (warp - 2) / (LOADERS / 32), lw = (warp - 2) % (LOADERS / 32);
        for (int it = group; it < nk; it += LOAD_GROUPS) {
            const int s = it % P::STAGES;
            if (it >= P::STAGES && !warp_wait(empty0 + 8 * s, (it / P::STAGES - 1) & 1, &abort, e.limit)) break;
            const uint32_t dst = base + s * P::STAGE;
            const int k = (kb0 + it) * BK;
            load_stage<TN>(w, x, m0, t0, k, K, dst, lw, lane);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(full0 + 8 * s) : "memory");
        }
    }

    // epilogue: warp w and w + 4 share a TMEM lane quarter and split the tokens
    constexpr int HALF = TN == 16 ? 16 : TN / 2;
    const int q4 = warp & 3, row = q4 * 32 + lane, n = m0 + row, half = warp >= 6 ? 1 : 0;
    const bool epi = warp >= 2 && warp < 10 && half * HALF < TN;
    const int c0 = half * HALF;
    const bool mine = warp >= 2 && warp < 10 && n < e.N;
    const float sw = mine ? e.sw[n] : 0.0f, b = mine && e.bias ? e.bias[n] : 0.0f;
    constexpr int NSX = (HALF + 31) / 32;
    float sx[NSX];                                         // of this CTA's tokens c0 .. (S = 1), or of those it finishes
    const int per = TN / S;
    if (warp >= 2 && warp < 10) get_scales<NSX>(e, t0 + (S == 1 ? c0 : rank * per), sx);
    bool ok = true;
    __syncwarp();
    if (epi) {
        ok = epilogue_wait(done, 0, warp == 2, TN == 16 ? 128 : 256);
        ok = __all_sync(~0u, ok && !abort);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    const uint32_t lanes = tmem + ((uint32_t)(q4 * 32) << 16) + c0;
    if (S == 1) {
        if (epi && ok) {
#pragma unroll
            for (int c = 0; c < HALF; c += 16) {
                int r[16];
                tmem_ld16(r, lanes + c);
                put16(e, r, t0 + c0 + c, sx[c / 32], c % 32, n, sw, b);
            }
        }
    } else {
        int* part = reinterpret_cast<int*>(smem);          // [TN][128]: every MMA has read its stage
        if (epi && ok) {
#pragma unroll
            for (int c = 0; c < HALF; c += 16) {
                int r[16];
                tmem_ld16(r, lanes + c);
#pragma unroll
                for (int j = 0; j < 16; ++j) part[(c0 + c + j) * BM + row] = r[j];
            }
        }
        cluster_sync();
        if (warp >= 2 && warp < 10 && ok) {
            if (S == 2) join<TN, 2>(e, base + row * 4, rank, half, t0, sx, n, sw, b);
            else if (S == 4) join<TN, 4>(e, base + row * 4, rank, half, t0, sx, n, sw, b);
            else join<TN, 8>(e, base + row * 4, rank, half, t0, sx, n, sw, b);
        }
        cluster_sync();                                    // no CTA leaves while its sums are read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    settle(&abort);
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(P::COLS));
}

// ---- pairs: many tokens --------------------------------------------------------
//
// Two CTAs on neighbouring SMs share each MMA (cta_group::2): 256 tokens (rows)
// by TN channels (columns), each CTA loading its 128 tokens and half of the
// channels, so that an SM takes in 32 KB for 128 x 256 x 128 products where it
// would alone take in 48 KB. Persistent: the pair's two accumulators alternate,
// and a tile's epilogue runs under the next tile's products. Tokens are the rows
// here so that a thread has neighbouring outputs of one token (5 instructions an
// output; 32 with channels as rows and 2-byte stores). Bound by the tensor cores, and
// over seconds by the power limit. Measured: 32768 x 8192 x 8192 1270 to 1390 us in a burst,
// by the GPU (3.46 to 3.16 POP/s; twice the bfloat16 rate of a library product is 3.32),
// 1530 to 1650 us sustained (2.87 to 2.67; twice its sustained rate is 2.77); 8192 x 4096 x
// 4096 88 us (3.14, tensor pipe 89% active); 65536 x 1024 x 4096 185 us; 65536 x 512 x 512,
// bound by outputs, 30 us.
constexpr int PAIR_EPI_WARPS = 8;
constexpr int PAIR_THREADS = 96 + 32 * PAIR_EPI_WARPS;
constexpr int RASTER = 8;                                  // tiles of tokens walked together
constexpr int ROW_BYTES = 64;                              // of a token's outputs staged at a time

template <int TN>
struct Pair {
    static constexpr int STAGE = (BM + TN / 2) * BK;
    static constexpr int STAGES = TN == 256 ? 6 : 8;
    static constexpr int FACTORS = 2 * (TN / 2) * 4;       // a warp's channel scales and biases
    static constexpr int STAGED = 32 * ROW_BYTES;          // a warp's outputs on their way out
    static constexpr int SMEM = STAGES * STAGE + PAIR_EPI_WARPS * (FACTORS + STAGED) + 1024;
};

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's 32 tokens (from t; lane = token, scale sx) by `cols` channels (from n),
// 64 bytes of outputs a token at a time: staged in shared memory (16-byte piece
// p of row r at p ^ (r / 2 % 4): no bank conflicts either way) and written out
// with four lanes a row where rows begin on 16-byte boundaries, else a row's
// values side by side.
template <class O>
__device__ __forceinline__ void put_rows(const Epilogue& e, uint32_t taddr, int64_t t, int n, int cols, float sx,
                                         const float* factors, uint8_t* staged, int lane) {
    constexpr int CH = ROW_BYTES / (int)sizeof(O);
    const int rows = (int)min((int64_t)32, e.T - t);
    O* const out = static_cast<O*>(e.out) + t * e.ldo + n;
#pragma unroll 1
    for (int c = 0; c < cols && n + c < e.N; c += CH) {
        int r[CH];
        if (CH == 32) tmem_ld32(r, taddr + c);
        else tmem_ld16(r, taddr + c);
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < CH; j += 4) {
            const float4 w = *reinterpret_cast<const float4*>(factors + c + j);
            const float4 b = *reinterpret_cast<const float4*>(factors + cols + c + j);
            const float v0 = (float)r[j] * sx * w.x + b.x, v1 = (float)r[j + 1] * sx * w.y + b.y,
                        v2 = (float)r[j + 2] * sx * w.z + b.z, v3 = (float)r[j + 3] * sx * w.w + b.w;
            if constexpr (sizeof(O) == 4) {
                v[j] = __float_as_uint(v0); v[j + 1] = __float_as_uint(v1);
                v[j + 2] = __float_as_uint(v2); v[j + 3] = __float_as_uint(v3);
            } else {
                v[j / 2] = pack2(v0, v1, O());
                v[j / 2 + 1] = pack2(v2, v3, O());
            }
        }
        __syncwarp();                                      // the last piece has been read
#pragma unroll
        for (int p = 0; p < 4; ++p)
            *reinterpret_cast<uint4*>(staged + lane * ROW_BYTES + 16 * (p ^ (lane / 2 % 4))) =
                make_uint4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
        __syncwarp();
        if (e.vec && n + c + CH <= e.N) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 8 * i + lane / 4, p = lane % 4;
                const uint4 o = *reinterpret_cast<const uint4*>(staged + row * ROW_BYTES + 16 * (p ^ (row / 2 % 4)));
                if (row < rows) *reinterpret_cast<uint4*>(out + row * e.ldo + c + p * (16 / (int)sizeof(O))) = o;
            }
        } else {
            for (int row = lane / CH; row < rows; row += 32 / CH) {
                const int col = lane % CH, at = col * (int)sizeof(O);
                if (n + c + col < e.N)
                    out[row * e.ldo + c + col] = *reinterpret_cast<const O*>(
                        staged + row * ROW_BYTES + 16 * (at / 16 ^ (row / 2 % 4)) + at % 16);
            }
        }
    }
}

template <int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, int K, int mt,
            int nt, Epilogue e) {
    using P = Pair<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[2 * P::STAGES + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort;
    const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * P::STAGES, tfull0 = empty0 + 8 * P::STAGES,
                   tempty0 = tfull0 + 16, drain = tempty0 + 16;
    const uint32_t base = smem_u32(smem);
    const int rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), npairs = (int)(gridDim.x >> 1);
    const int nk = (K + BK - 1) / BK;
    const int64_t tiles = (int64_t)mt * nt;

    if (tid == 0) {
        for (int i = 0; i < P::STAGES; ++i) {
            mbar_init(full0 + 8 * i, 2);                   // used in the first CTA only
            mbar_init(empty0 + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(tfull0 + 8 * i, 1);
            mbar_init(tempty0 + 8 * i, 2 * PAIR_EPI_WARPS);   // used in the first CTA only
        }
        mbar_init(drain, 1);
        abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&tmem_slot)), "r"((uint32_t)(2 * TN)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    before_memory();

    auto tile_at = [&](int64_t i, int64_t& t0, int& n0) {  // the first token and channel of tile i
        const int64_t group = i / ((int64_t)RASTER * nt), r = i - group * RASTER * nt;
        const int wide = min(RASTER, mt - (int)group * RASTER);
        t0 = (group * RASTER + r % wide) * 2 * BM;
        n0 = (int)(r / wide) * TN;
    };

    if (warp == 0 || warp == 2) {                          // the tokens' and the channels' copies
        if (elect_one()) {
            const bool of_x = warp == 0;
            const uint64_t map = (uint64_t)(of_x ? &map_x : &map_w);
            const uint32_t lead0 = map_to(full0, 0);       // the first CTA's barriers
            const uint32_t bytes = of_x ? BM * BK : TN / 2 * BK, dst0 = base + (of_x ? 0 : BM * BK);
            Ring<P::STAGES> r;
            uint32_t first = 1;                            // the ring's first round waits for nothing
            bool ok = true;
            for (int64_t i = pair; ok && i < tiles; i += npairs) {
                int n0;
                int64_t t0;
                tile_at(i, t0, n0);
                const int y = of_x ? (int)t0 + rank * BM : n0 + rank * (TN / 2);
                for (int kb = 0; kb < nk; ++kb) {
                    if (!first && !mbar_wait(empty0 + 8 * r.s, r.phase ^ 1u, &abort, e.limit)) { ok = false; break; }
                    if (rank == 0) mbar_expect(full0 + 8 * r.s, 2 * bytes);
                    asm volatile(
                        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
                        " [%0], [%1, {%2, %3}], [%4];"
                        :: "r"(dst0 + r.s * P::STAGE), "l"(map), "r"(kb * BK), "r"(y), "r"(lead0 + 8 * r.s) : "memory");
                    r.next();
                    if (r.s == 0) first = 0;
                }
            }
            if (of_x) let_next_start();                    // under the last tile: called at the start, it cost a norm that followed 40 us
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint64_t d0 = sw128_desc(base);
            Ring<P::STAGES> r;
            Ring<2> acc;
            bool ok = true;
            for (int64_t i = pair; ok && i < tiles; i += npairs, acc.next()) {
                if (i >= pair + 2 * (int64_t)npairs && !mbar_wait(tempty0 + 8 * acc.s, acc.phase ^ 1u, &abort, e.limit)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                int left = K;
                for (int kb = 0; kb < nk; ++kb, r.next(), left -= BK) {
                    if (!mbar_wait(full0 + 8 * r.s, r.phase, &abort, e.limit)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t d = d0 + (uint64_t)(r.s * (P::STAGE >> 4));
                    mma_block<2>(tmem + acc.s * TN, d, d + (BM * BK >> 4), idesc_i8(2 * BM, TN), left, kb > 0);
                    asm volatile(
                        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                        :: "r"(empty0 + 8 * r.s), "h"((uint16_t)3) : "memory");
                }
                if (!ok) break;
                asm volatile(
                    "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                    :: "r"(tfull0 + 8 * acc.s), "h"((uint16_t)3) : "memory");
            }
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(drain) : "memory");
            mbar_wait(drain, 0, nullptr);                  // every MMA issued has completed
        }
    } else {
        const int q4 = warp & 3, half = (warp - 3) >> 2;   // TMEM lane quarter, column half
        constexpr int COLS = TN / 2;
        uint8_t* mine = smem + P::STAGES * P::STAGE + (warp - 3) * (P::FACTORS + P::STAGED);
        float* factors = reinterpret_cast<float*>(mine);
        uint8_t* staged = mine + P::FACTORS;
        Ring<2> acc;
        float sx = 0.0f, sw[COLS / 32], b[COLS / 32];      // of the next tile: this lane's token, every 32nd channel
        int64_t t = 0;
        int n = 0;
        auto fetch = [&](int64_t i) {
            if (i >= tiles) return;
            int n0;
            tile_at(i, t, n0);
            t += rank * BM + q4 * 32;
            n = n0 + half * COLS;
            sx = t + lane < e.T ? e.sx[t + lane] : 0.0f;
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                const int at = n + 32 * c + lane;
                sw[c] = at < e.N ? e.sw[at] : 0.0f;
                b[c] = e.bias && at < e.N ? e.bias[at] : 0.0f;
            }
        };
        fetch(pair);
        for (int64_t i = pair; i < tiles; i += npairs, acc.next()) {
            const int64_t t1 = t;
            const int n1 = n;
            const float sx1 = sx;
            __syncwarp();
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                factors[32 * c + lane] = sw[c];
                factors[COLS + 32 * c + lane] = b[c];
            }
            __syncwarp();
            fetch(i + npairs);                             // arrives under this tile's products and outputs
            if (!warp_wait(tfull0 + 8 * acc.s, acc.phase, &abort, e.limit)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem + ((uint32_t)(q4 * 32) << 16) + acc.s * TN + half * COLS;
            if (t1 < e.T) {
                if (e.type == JHQ_BF16) put_rows<__nv_bfloat16>(e, taddr, t1, n1, COLS, sx1, factors, staged, lane);
                else if (e.type == JHQ_F16) put_rows<__half>(e, taddr, t1, n1, COLS, sx1, factors, staged, lane);
                else put_rows<float>(e, taddr, t1, n1, COLS, sx1, factors, staged, lane);
            }
            // relaxed: the arrival hands over TMEM alone, whose reads have completed;
            // a release would wait for the outputs' stores as well
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];"
                             :: "r"(map_to(tempty0 + 8 * acc.s, 0)) : "memory");
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    settle(&abort);
    cluster_sync();                                        // no MMA or arrival still heads for the other CTA
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t)(2 * TN)));
}

// ---- host ------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess &&
            qr == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    if (!fn) fail(JHQ_EDEVICE, "q8_matmul: cuTensorMapEncodeTiled unavailable");
    return fn;
}

// What a tensor map takes: rows that begin on 16-byte boundaries.
bool on_boundaries(const jhq_q8_rows* r) {
    return (uintptr_t)r->q % 16 == 0 && (r->rows == 1 || (r->ld % 16 == 0 && r->ld < (1ll << 40)));
}

// Boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside the array.
CUtensorMap make_map(const jhq_q8_rows* r, int box_rows) {
    CUtensorMap m;
    const cuuint64_t dims[2] = {(cuuint64_t)r->dim, (cuuint64_t)r->rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(r->rows == 1 ? (r->dim + 15) / 16 * 16 : r->ld)};
    const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult rc = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, r->q, dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) fail(JHQ_EDEVICE, "q8_matmul: tensor map encoding failed");
    return m;
}

constexpr int SMS = 148;

Rows8 rows8(const jhq_q8_rows* r) { return {r->q, r->ld, r->rows, r->q + (r->rows - 1) * r->ld + r->dim}; }

template <int TN, bool TMA>
void panel_attributes() {
    static std::atomic<uint64_t> done{0};
    once_per_device(done, [] {
        JHQ_CUDA(cudaFuncSetAttribute(panel_kernel<TN, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, Panel<TN>::SMEM));
    });
}

// CTAs of panels that run at once in clusters of S (one an SM; a cluster stays within a GPC, so fewer with large S).
int panel_capacity(int S) {
    static std::atomic<uint64_t> done{0};
    static std::atomic<int> held[4];                       // of the last device asked; all B200s alike but for spare SMs
    once_per_device(done, [] {
        panel_attributes<64, true>();
        for (int k = 0; k < 4; ++k) {
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 1u << k;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(SMS << k);
            cfg.blockDim = dim3(panel_threads(true));
            cfg.dynamicSmemBytes = Panel<64>::SMEM;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            int n = 0;
            JHQ_CUDA(cudaOccupancyMaxActiveClusters(&n, panel_kernel<64, true>, &cfg));
            held[k] = std::max(1, n << k);
        }
    });
    return held[S == 1 ? 0 : S == 2 ? 1 : S == 4 ? 2 : 3];
}

template <int TN, bool TMA>
void panels(const jhq_q8_rows* x, const jhq_q8_rows* w, int S, const Epilogue& e, cudaStream_t s) {
    panel_attributes<TN, TMA>();
    const int64_t ttiles = ceil_div(x->rows, TN), blocks = ttiles * ceil_div(w->rows, BM) * S;
    if (blocks > INT32_MAX) fail(JHQ_EINVAL, "q8_matmul: too many rows");
    CUtensorMap mw{}, mx{};
    if (TMA) { mw = make_map(w, BM); mx = make_map(x, TN); }
    launch_q8(panel_kernel<TN, TMA>, dim3((unsigned)blocks), panel_threads(TMA), Panel<TN>::SMEM, S, s, mw, mx, rows8(w),
              rows8(x), (int)x->dim, S, (int)ttiles, e);
}
template <bool TMA>
void panels(const jhq_q8_rows* x, const jhq_q8_rows* w, int TN, int S, const Epilogue& e, cudaStream_t s) {
    if (TN == 16) panels<16, TMA>(x, w, S, e, s);
    else if (TN == 32) panels<32, TMA>(x, w, S, e, s);
    else if (TN == 64) panels<64, TMA>(x, w, S, e, s);
    else panels<128, TMA>(x, w, S, e, s);
}

template <int TN>
void pairs(const jhq_q8_rows* x, const jhq_q8_rows* w, const Epilogue& e, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    once_per_device(done, [] {
        JHQ_CUDA(cudaFuncSetAttribute(pair_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Pair<TN>::SMEM));
    });
    const int64_t mt = ceil_div(x->rows, 2 * BM), nt = ceil_div(w->rows, TN);
    const unsigned grid = 2 * (unsigned)std::min<int64_t>(SMS / 2, mt * nt);
    launch_q8(pair_kernel<TN>, dim3(grid), PAIR_THREADS, Pair<TN>::SMEM, 0, s, make_map(x, BM), make_map(w, TN / 2),
              (int)x->dim, (int)mt, (int)nt, e);
}

// Which kernel, tile and split: the least of the costs below, fitted to microseconds of launches in a graph. They leave the
// operands' bytes out, and where those bind only order the choices (64 x 8192 x 8192 costs 9.8 and takes 16.3 us, 16 x 16384 x
// 16384 20.9 and 43.5). A K block of 128 bytes takes 0.14 us in a panel (barriers and issue) and in a pair with 128 channels, 0.272 us
// in one with 256 (the MMAs), more as all pairs draw on L2; the rest is launch, filling the ring, joining slices and the
// epilogue. Best panel / pair of 128 / pair of 256, in us: 256 x 1024 x 4096 7.5 / 8.9 / 14.3; 512 x 1024 x 1024
// 5.2 / 5.5 / 7.8; 256 x 4096 x 4096 10.1 / 9.3 / 14.7; 8192 x 4096 x 4096 236 / 99 / 86. Above 2048 tokens only pairs are
// looked at: the panels' costs are too low there (4096 x 512 x 4096: panels cost 10.8 and take 13.6 us, pairs 10.8 and 10.7).
// The limit loses where few channels meet long rows (4096 x 128 x 16384: panels would take 18.3 us, pairs take 26.6).
struct Plan {
    int tile, split;                                       // split 0: pairs
    double us;
};
// The best panel, if it beats `best`: tiles of 16, 32, 64 and 128 tokens at block[] us a K block and first[] us a tile.
void best_panel(const jhq_q8_rows* x, const jhq_q8_rows* w, const double* block, const double* first, Plan& best) {
    const int64_t nkb = ceil_div(x->dim, BK), mt = ceil_div(w->rows, BM);
    for (int k = 0; k < 4; ++k) {
        const int tn = 16 << k;
        for (int S = 1; S <= 8 && 2 * S <= std::max<int64_t>(nkb, 2); S *= 2) {
            const int64_t waves = ceil_div(ceil_div(x->rows, tn) * mt * S, panel_capacity(S));
            const double us = (double)waves * ((double)ceil_div(nkb, S) * block[k] + first[k] + (S > 1 ? 0.9 : 0.0));
            if (us < best.us) best = {tn, S, us};
        }
        if (tn >= x->rows) break;
    }
}
Plan plan(const jhq_q8_rows* x, const jhq_q8_rows* w) {
    const int64_t nkb = ceil_div(x->dim, BK);
    Plan best{256, 0, 0.0};
    for (int tn : {256, 128}) {
        const int64_t tiles = ceil_div(x->rows, 2 * BM) * ceil_div(w->rows, tn), waves = ceil_div(tiles, SMS / 2);
        const double busy = (double)std::min<int64_t>(tiles, SMS / 2) / (SMS / 2);
        const double block = tn == 256 ? 0.272 + 0.05 * busy : 0.14 + 0.07 * busy;
        const double first = tn == 256 ? 5.6 : 4.4, least = tn == 256 ? 4.0 : 2.3;
        const double us = first + nkb * block + (double)(waves - 1) * std::max(nkb * block, least);
        if (tn == 256 || us < best.us) best = {tn, 0, us};
    }
    if (x->rows > 2048) return best;
    const double block[4] = {0.14, 0.14, 0.14, 0.14}, first[4] = {3.0, 3.4, 4.4, 6.3};
    best_panel(x, w, block, first, best);
    return best;
}
// Rows that TMA cannot fetch: panels, whose loader threads bind, who bring 128 + tile rows for 128 x tile products.
// 1 x 4001 x 4001 in tiles of 16 took 32 / 18 / 11.5 us in 1 / 2 / 4 slices, 1000 x 999 x 1001 in tiles of 64 14.0 us, of
// 128 in two slices 15.4 us, 4001 x 4001 x 4001 in tiles of 64 555 us, of 128 418 us.
Plan plan_unaligned(const jhq_q8_rows* x, const jhq_q8_rows* w) {
    Plan best{128, 1, 1e30};
    const double block[4] = {0.85, 0.85, 1.0, 1.5}, first[4] = {4.8, 5.0, 5.4, 6.5};
    best_panel(x, w, block, first, best);
    return best;
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
    long long limit = WAIT_CYCLES;
    if (const char* v = std::getenv("JHQ_TEST_TC_WAIT_CYCLES")) limit = std::atoll(v);
    const Epilogue e{x->scale, w->scale, bias ? (const float*)bias->data : nullptr, out->data, out->ld,
                     x->rows, (int)w->rows, out->type,
                     (uintptr_t)out->data % 16 == 0 && out->ld % (out->type == JHQ_F32 ? 4 : 8) == 0, limit};
    const bool tma = on_boundaries(x) && on_boundaries(w);
    const Plan p = tma ? plan(x, w) : plan_unaligned(x, w);
    if (!tma) panels<false>(x, w, p.tile, p.split, e, s);
    else if (p.split) panels<true>(x, w, p.tile, p.split, e, s);
    else if (p.tile == 128) pairs<128>(x, w, e, s);
    else pairs<256>(x, w, e, s);
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
