// A paged key-value cache for batched serving: the append of new rows with the position
// rotation applied on the way, and attention of one new token per sequence.
//
// Cache layout: K and V are [pages][kv_heads][page_size][head_dim], so that the rows of one
// head in one page are one contiguous tile: a TMA box for the reader, whole sectors for the
// writer.  A Q8_0 cache keeps its int8 values in that layout and its f16 scales in planes of
// their own, [pages][kv_heads][page_size][head_dim / 32]: the 34-byte blocks of the
// contiguous cache would start at addresses that neither TMA nor 16-byte loads can take.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include "../../include/ncm.h"
#include "ncm_internal.h"
#include "common.cuh"
#include "synth.h"

namespace ncm {

static const char* pointer_error(const void* p, int dev) {
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();   // not a sticky error: leave none behind
        return "a pointer the driver does not know";
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) return "not a device pointer";
    if (a.type == cudaMemoryTypeDevice && a.device != dev) return "a pointer of another device than the current one";
    return nullptr;
}
const char* device_pointers_error(const void* const* p, int n) {
    // The driver's own call is asked first: it takes two thirds of the runtime's time, and a call
    // of the library has a dozen pointers.
    typedef CUresult (*GetFn)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
    static const GetFn get = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &fn, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return (GetFn)fn;
        return (GetFn) nullptr;
    }();
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return "no CUDA device";
    }
    for (int i = 0; i < n; ++i) {
        if (!p[i]) continue;
        int ordinal = -1;
        unsigned type = 0;
        CUpointer_attribute which[2] = {CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, CU_POINTER_ATTRIBUTE_MEMORY_TYPE};
        void* data[2] = {&ordinal, &type};
        if (get && get(2, which, data, (CUdeviceptr)p[i]) == CUDA_SUCCESS && ordinal == dev && type == CU_MEMORYTYPE_DEVICE) continue;
        if (const char* e = pointer_error(p[i], dev)) return e;
    }
    return nullptr;
}

namespace {

constexpr uint64_t kPagedWaitNs = 4000000000ull;   // bound on a wait for a TMA copy

// ------------------------------------------------------------------ append
struct AppendParams {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;   // elements between tokens
    void* q_out;                            // [tokens][heads][head_dim]
    int heads, kv_heads, hd, tokens, batch;
    const int *cu, *lengths, *table;
    int table_width, log2ps;
    int64_t pages, page_stride;             // page_stride in elements
    const float2* rope;                     // [rope_len][rope_half] (sin, cos), or null
    int rope_len, rope_half, halves;
    int kind, out_bf16;                     // cache type id; q_out is bf16 (else f16)
    void *kc, *vc;
    __half *ks, *vs;
    int* err;
};

// Sequence of a packed token, how many of cu[1 .. batch] are <= token, and its position: one
// warp.  Up to 32 sequences take one round of loads; more, 32 probes a step (two steps up to
// 1023) and a round.  Returns the sequence, or -1 for a row that belongs to none.
__device__ __forceinline__ int place_of_token(const int* cu, const int* lengths, int batch, int token, int& pos) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = batch;
    while (n > 32) {
        const int step = (n + 31) >> 5;
        const int at = lo + min((lane + 1) * step, n);   // cu index of the probe: its end
        const int k = __popc(__ballot_sync(NCM_FULL, __ldg(cu + at) <= token));
        if (k == 32) return -1;
        lo += k * step;
        // the answer is among these (the last probe's end is past the token)
        n = min(step, n - k * step);
    }
    const int at = lo + min(lane, n - 1);
    const int first = __ldg(cu + at), end = __ldg(cu + at + 1), length = __ldg(lengths + at);
    const int k = __popc(__ballot_sync(NCM_FULL, lane < n && end <= token));
    if (k >= n) return -1;
    pos = __shfl_sync(NCM_FULL, max(length, 0) - (end - token), k);
    // not so before the first sequence, nor for starts that are out of order
    return __shfl_sync(NCM_FULL, (int)(first <= token && token < end), k) ? lo + k : -1;
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float* x);
template <> __device__ __forceinline__ void load8<float>(const float* p, float* x) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float* x) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* x) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint32_t pack2(bool bf16, float a, float b) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(bool bf16, void* p, const float* x) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(bf16, x[0], x[1]), pack2(bf16, x[2], x[3]),
                                              pack2(bf16, x[4], x[5]), pack2(bf16, x[6], x[7]));
}
// One 8-value part of a Q8_0 block whose four parts lie in four neighbouring lanes.  The scale
// is the largest magnitude times 1 / 127: a multiply where the contiguous cache's store divides
// (kv_store_kernel), one f32 step apart at most before both are cut to f16's eleven bits.
// All lanes of the warp take part.
__device__ __forceinline__ void store_q8(bool active, int8_t* values, __half* scale, const float* x, int part) {
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[i]));
    mx = fmaxf(mx, __shfl_xor_sync(NCM_FULL, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(NCM_FULL, mx, 2));
    if (!active) return;
    const float sc = mx * (1.0f / 127.0f), inv = sc > 0.0f ? 1.0f / sc : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int v = (int)fminf(fmaxf(roundf(x[i] * inv), -127.0f), 127.0f);
        w[i >> 2] |= (uint32_t)(v & 0xff) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(values) = make_uint2(w[0], w[1]);
    if (part == 0) *reinterpret_cast<uint16_t*>(scale) = ncm_f32_to_f16_trunc(sc);
}

// One CTA per token; a thread takes 16 values of one head, 8 from each half of it, so that
// both rotation styles find their pairs in one thread and Q8_0 blocks lie in four lanes.
// The rows are read before the token's place is looked up: the two latencies overlap.
template <typename T>
__global__ void __launch_bounds__(512) paged_append_kernel(const __grid_constant__ AppendParams p) {
    const int token = blockIdx.x, hd = p.hd, per = hd >> 4;   // threads per head: 4 or 8
    const int all = (p.heads + 2 * p.kv_heads) * per;
    // the same for all of a thread's rows
    const int part = threadIdx.x & (per - 1), lo = 8 * part, hi = (hd >> 1) + lo;
    int off = 0, page = -1;
    float4 turn[4];                        // two (sin, cos) each, of the thread's eight pairs
    bool ready = false;
    // The first CTA looks over the starts; the first of them are on their way with the rows.
    const bool looks = p.cu && token == 0;
    int cu0 = 0, cu1 = 0;
    if (looks && threadIdx.x < p.batch) { cu0 = __ldg(p.cu + threadIdx.x); cu1 = __ldg(p.cu + threadIdx.x + 1); }
    for (int base = 0; base < all; base += blockDim.x) {
        const int task = base + threadIdx.x;
        const bool active = task < all;
        const int row = active ? task / per : 0;
        const bool is_q = row < p.heads, is_k = !is_q && row < p.heads + p.kv_heads;
        const int head = is_q ? row : is_k ? row - p.heads : row - p.heads - p.kv_heads;
        float x[16];
        if (active) {
            const T* src = static_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) +
                           (int64_t)token * (is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride) + head * hd;
            load8<T>(src + lo, x);
            load8<T>(src + hi, x + 8);
        }
        if (!ready) {
            ready = true;
            if (looks) {
                bool bad = cu0 < 0 || cu1 < cu0 || cu1 > p.tokens;
                for (int b = threadIdx.x + blockDim.x; b < p.batch; b += blockDim.x) {
                    cu0 = __ldg(p.cu + b); cu1 = __ldg(p.cu + b + 1);
                    bad |= cu0 < 0 || cu1 < cu0 || cu1 > p.tokens;
                }
                if (bad) set_dev_error(p.err, NCM_DEVERR_BAD_ARG);
                __syncwarp();
            }
            int seq = token, pos = 0;
            if (p.cu) {
                seq = place_of_token(p.cu, p.lengths, p.batch, token, pos);
                if (seq < 0) return;   // a row of padding: left alone
            } else {
                pos = __ldg(p.lengths + seq) - 1;
            }
            off = pos & ((1 << p.log2ps) - 1);
            const bool good = pos >= 0 && (pos >> p.log2ps) < p.table_width && (!p.rope || pos < p.rope_len);
            if (good) {
                page = __ldg(p.table + (int64_t)seq * p.table_width + (pos >> p.log2ps));
                if (p.rope) {
                    const float2* table = p.rope + (int64_t)pos * p.rope_half;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int pair = p.halves ? lo + 2 * i : ((i < 2 ? lo : hi - 8) >> 1) + 2 * i;
                        if (pair < p.rope_half) turn[i] = __ldg(reinterpret_cast<const float4*>(table + pair));
                    }
                }
            }
            if (!good || page < 0 || page >= p.pages) {   // nothing of this token is stored
                if (threadIdx.x == 0) set_dev_error(p.err, NCM_DEVERR_BAD_ARG);
                return;
            }
        }
        if (p.rope && active && (is_q || is_k)) {
            if (p.halves) {   // pairs (i, i + hd / 2)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float4 t = turn[i >> 1];
                    const float a = x[i], b = x[i + 8], c = x[i + 1], d = x[i + 9];
                    x[i] = a * t.y - b * t.x; x[i + 8] = a * t.x + b * t.y;
                    x[i + 1] = c * t.w - d * t.z; x[i + 9] = c * t.z + d * t.w;
                }
            } else {          // pairs (2i, 2i + 1), the first rope_half of them
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    // rope_half is even: two pairs at a time
                    if ((((i < 8 ? lo : hi - 8) + i) >> 1) >= p.rope_half) continue;
                    const float4 t = turn[i >> 2];
                    const float a = x[i], b = x[i + 1], c = x[i + 2], d = x[i + 3];
                    x[i] = a * t.y - b * t.x; x[i + 1] = a * t.x + b * t.y;
                    x[i + 2] = c * t.w - d * t.z; x[i + 3] = c * t.z + d * t.w;
                }
            }
        }
        const int64_t slot = ((int64_t)head << p.log2ps) + off;   // row within the page
        if (p.kind == NCM_TYPE_Q8_0) {
            const bool mine = active && !is_q;
            int8_t* row8 = static_cast<int8_t*>(is_k ? p.kc : p.vc) + (int64_t)page * p.page_stride + slot * hd;
            __half* scales = (is_k ? p.ks : p.vs) +
                             (((int64_t)page * p.kv_heads << p.log2ps) + slot) * (hd >> 5) + (part >> 2);
            store_q8(mine, row8 + lo, scales, x, part & 3);
            store_q8(mine, row8 + hi, scales + (hd >> 6), x + 8, part & 3);
        } else if (active && !is_q) {
            uint16_t* dst = static_cast<uint16_t*>(is_k ? p.kc : p.vc) + (int64_t)page * p.page_stride + slot * hd;
            store8(p.kind == NCM_TYPE_BF16, dst + lo, x);
            store8(p.kind == NCM_TYPE_BF16, dst + hi, x + 8);
        }
        if (active && is_q) {
            uint16_t* dst = static_cast<uint16_t*>(p.q_out) + ((int64_t)token * p.heads + head) * hd;
            store8(p.out_bf16, dst + lo, x);
            store8(p.out_bf16, dst + hi, x + 8);
        }
    }
}

// ------------------------------------------------------------------ attention of one token
constexpr int kUnit = 32;              // keys that a warp takes at a time
// Units per warp up to which a segment stays in one CTA: 1, 2 or 4, the first with which there are
// CTAs enough.  One sequence of 4000 keys (32 / 8 heads of 128) takes 11.5 us with 1 (and the join over
// CTAs that it means), 12.0 with 2, 13.4 with 3, 14.7 with 4; one of 16000 20.9 with 2 and 4, 22.4 without.
constexpr int kPieces = 3;
constexpr int kPagedBatch = 1024;      // sequences of one launch (their lengths lie in shared memory)
constexpr int kPagedSmem = 232448;     // 227 KB

struct alignas(64) PagedAttnParams {
    CUtensorMap km, vm;                // {hd, page_size, kv_heads, pages}, box {128 bytes (64 for int8 of 64), rows}
    CUtensorMap ksm, vsm;              // Q8_0 scales: {page_size * hd / 32, kv_heads, pages}
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int *lengths, *table;
    int table_width, batch, heads, kv_heads, group;
    int chunk, nchunk;                 // heads of a group that a segment takes, and segments per group
    int log2ps, box_rows, nstages;
    int64_t pages;
    float scale_log2;
    float* part;                       // workspace: [2 * grid][chunk][hd] sums, then [2 * grid][chunk][2] (max, sum)
    unsigned* counters;                // [grid], zero between calls
    int* err;
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Integer products of int8 rows A with int8 (or unsigned) columns B, 32 deep.  The sum starts
// from the bits of 1.5 * 2^23, so that the result is the float 1.5 * 2^23 + sum while |sum| < 2^22.
constexpr uint32_t kIntBase = 0x4b400000u;
constexpr float kIntBaseF = 12582912.0f;
template <bool UNSIGNED_B>
__device__ __forceinline__ void imma16832(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    uint32_t r0, r1, r2, r3;
    if (UNSIGNED_B)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kIntBase));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kIntBase));
    d[0] = __uint_as_float(r0); d[1] = __uint_as_float(r1); d[2] = __uint_as_float(r2); d[3] = __uint_as_float(r3);
}
// 256 hi + lo of two such results.
__device__ __forceinline__ float joined(float hi, float lo) { return fmaf(hi - kIntBaseF, 256.0f, lo - kIntBaseF); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16> __device__ __forceinline__ float2 widen2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A segment is one (sequence, key-value head, chunk of its query heads); its keys are cut in
// units of 32.  All units of all segments lie in one row that is shared out evenly, first
// over the CTAs, then over a CTA's warps; when there are so few that every CTA can take at
// most 4 units per warp of a single segment, the row is padded so that no CTA has
// two segments: a segment that fits one CTA is then joined in shared memory alone (a join
// over CTAs costs about 4 us).  Positions fit 32 bits: the host sees to it.  A place in the row:
struct Place {
    int b, hk, u, n;   // sequence, segment within it, unit within the segment, units of the segment
};

// Four values of out, from `at` on, rounded to its 16-bit type.
template <bool BF16>
__device__ __forceinline__ void store_out(void* out, int64_t at, float4 v) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(pack2(BF16, v.x, v.y), pack2(BF16, v.z, v.w));
}
// 1 / sum; a row whose scores are all -infinity has nothing to divide and stays zero.
__device__ __forceinline__ float inverse(float sum) { return sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f; }
// (also where its values are not finite, whose products with zero are not zero)
__device__ __forceinline__ float scaled(float v, float inv) { return inv == 0.0f ? 0.0f : v * inv; }
__device__ __forceinline__ float4 scaled(float4 v, float inv) {
    return make_float4(scaled(v.x, inv), scaled(v.y, inv), scaled(v.z, inv), scaled(v.w, inv));
}
// What a part (a maximum and a sum per head, and a row of hd sums) counts in a join whose largest
// maximum is `top`: nothing if none of its keys scored above -infinity.
__device__ __forceinline__ float part_weight(float m, float top) { return m == -INFINITY ? 0.0f : ex2(m - top); }

__host__ __device__ constexpr bool one_stage(bool q8, int hd, int nt) { return nt == 1 && (hd == 128 || !q8); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(NCM_FULL, v, 0); }
// One lane of a converged warp, in a form that the compiler knows for one.
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(yes));
    return yes != 0;
}

template <bool BF16, bool Q8, int HD, int NT, int W>
__global__ void __launch_bounds__(W * 32, 1) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    constexpr int GH = 8 * NT;                                   // head slots of a segment
    constexpr int KB = kUnit * HD * (Q8 ? 1 : 2);                // bytes of a unit's K (or V) values
    constexpr int SB = Q8 ? 512 : 0;                             // ... and of its scales
    constexpr int STAGE = 2 * (KB + SB);
    constexpr int KS = HD / 16, NB = HD / 32;
    constexpr bool ONE = one_stage(Q8, HD, NT);                      // K and V of a unit are then fetched apart
    // p and its sums times 2^7 where p is rounded to f16: 2^15 at most then, and what is below 2^-14 of
    // the largest, where f16's steps no longer shrink, is held 2^7 times finer.
    constexpr float kLift = BF16 || Q8 ? 0.0f : 7.0f;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c4 = lane & 3, r8 = lane >> 2;
    const int nst = p.nstages;

    uint8_t* smem = smem_raw;                                    // ring [warp][stage][STAGE]
    uint8_t* after = smem + (size_t)W * nst * STAGE;
    float* first = reinterpret_cast<float*>(after);              // [warp][GH][HD], then [warp][GH][2]
    float* first_ml = first + W * GH * HD;
    uint64_t* bars = reinterpret_cast<uint64_t*>(first_ml + W * GH * 2);   // [warp][stage][2]
    int* ent = reinterpret_cast<int*>(bars + W * nst * 2);       // [2 W][4]: sequence (-1: none), segment, begin, end
    int* sums = ent + 2 * W * 4;                                 // [4 W + 1]
    int* prefix = sums + 4 * W + 1;                                      // [batch + 1]
    int* lens = prefix + p.batch + 1;                            // [batch]

    // ---- lengths and their running sum of units, as they are and padded to pieces
    const int HK = p.kv_heads * p.nchunk;
    int piece = 0;   // units of a piece; 0: no padding
    {
        const int per = (p.batch + W * 32 - 1) / (W * 32);
        const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
        int sum[kPieces + 1], run[kPieces + 1];   // in units, and in pieces of W, 2 W, 4 W
        auto pieces_of = [&](int n, int size) { return ((n + kUnit - 1) / kUnit + size - 1) / size; };
#pragma unroll
        for (int i = 0; i <= kPieces; ++i) sum[i] = 0;
        const int cap = p.table_width << p.log2ps;
        for (int b = b0; b < b1; ++b) {
            int n = __ldg(p.lengths + b);
            if (n > cap) {
                n = cap;
                if (blockIdx.x == 0) set_dev_error(p.err, NCM_DEVERR_BAD_ARG);
            }
            n = max(n, 0);
            lens[b] = n;
#pragma unroll
            for (int i = 0; i <= kPieces; ++i) sum[i] += pieces_of(n, i ? W << (i - 1) : 1);
        }
#pragma unroll
        for (int i = 0; i <= kPieces; ++i) {
            run[i] = sum[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(NCM_FULL, run[i], o);
                if (lane >= o) run[i] += v;
            }
        }
        if (lane == 31) *reinterpret_cast<int4*>(sums + 4 * warp) = make_int4(run[0], run[1], run[2], run[3]);
        if (tid < 2 * W) ent[4 * tid] = -1;
        if (lane == 0)
            for (int i = 0; i < 2 * nst; ++i) mbar_init(bars + warp * nst * 2 + i, 1);
        fence_mbar_init();
        __syncthreads();
        int4 before = make_int4(0, 0, 0, 0), all = before;
        for (int w = 0; w < W; ++w) {
            const int4 v = *reinterpret_cast<const int4*>(sums + 4 * w);
            if (w < warp) { before.x += v.x; before.y += v.y; before.z += v.z; before.w += v.w; }
            all.y += v.y; all.z += v.z; all.w += v.w;
        }
        const int room = (int)gridDim.x / HK;
        int at = before.x + run[0] - sum[0];
        if (all.y <= room) { piece = W; at = before.y + run[1] - sum[1]; }
        else if (all.z <= room) { piece = 2 * W; at = before.z + run[2] - sum[2]; }
        else if (all.w <= room) { piece = 4 * W; at = before.w + run[3] - sum[3]; }
        if (tid == 0) prefix[0] = 0;
        for (int b = b0; b < b1; ++b) {
            at += piece ? pieces_of(lens[b], piece) : pieces_of(lens[b], 1);
            prefix[b + 1] = piece ? at * piece : at;
        }
        __syncthreads();
    }
    // rows of sequences without keys
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
        if (lens[b] == 0)
            for (int i = 4 * tid; i < p.heads * HD; i += 4 * W * 32)
                store_out<BF16>(p.out, b * p.out_stride + i, make_float4(0.f, 0.f, 0.f, 0.f));

    const int total = prefix[p.batch] * HK;
    const int share = piece ? piece : max(W, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int u0 = (int)min((int64_t)total, (int64_t)blockIdx.x * share);
    if (u0 >= total) return;
    Place c;
    auto find = [&](int at) {   // the place at this position of the row
        int lo = 0, hi = p.batch;   // last b with prefix[b] * HK <= at
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] * HK <= at) lo = mid; else hi = mid;
        }
        const int stride = prefix[lo + 1] - prefix[lo], rest = at - prefix[lo] * HK;
        c.b = lo;
        c.n = (lens[lo] + kUnit - 1) / kUnit;
        c.hk = rest / stride;
        c.u = rest - c.hk * stride;
    };
    find(u0);
    const int u1 = piece ? u0 + min(share, c.n - c.u) : (int)min((int64_t)total, (int64_t)u0 + share);
    const int per_warp = (u1 - u0 + W - 1) / W;
    const int w0 = min(u1, u0 + warp * per_warp), w1 = min(u1, w0 + per_warp);
    const int count = w1 - w0;
    if (count > 0) {
        if (piece) c.u += w0 - u0; else find(w0);
    }

    // ---- this warp's units
    uint8_t* ring = smem + (size_t)warp * nst * STAGE;
    uint64_t* bar = bars + warp * nst * 2;
    auto next = [&](Place& t) {
        if (++t.u < t.n) return;
        t.u = 0;
        if (++t.hk < HK) return;
        t.hk = 0;
        do { ++t.b; } while (t.b < p.batch && lens[t.b] == 0);
        t.n = t.b < p.batch ? (lens[t.b] + kUnit - 1) / kUnit : 1;
    };
    // boxes of a unit: one per page, or one of 32 rows
    const int box = p.box_rows, lbox = 31 - __clz(box), lnpg = 5 - lbox, npg = 1 << lnpg;
    auto page_at = [&](const Place& t, int i) -> int {   // the page of box i < npg
        const int key = t.u * kUnit + i * box;
        if (i >= npg || key >= lens[t.b]) return -1;
        const int id = __ldg(p.table + (int64_t)t.b * p.table_width + (key >> p.log2ps));
        if (id < 0 || id >= p.pages) set_dev_error(p.err, NCM_DEVERR_BAD_ARG);   // TMA reads zeros there
        return id;
    };
    auto head_of = [&](int hk) { return p.nchunk == 1 ? hk : hk / p.nchunk; };
    // Fetches a unit (with one stage its K or its V, since K's place is free before the softmax)
    // whose boxes' pages lie in lanes 0 to npg - 1.  One lane issues, from uniform values: copies
    // issued by the lanes that hold the pages took about 1000 cycles a unit.
    auto issue = [&](const Place& t, int page, int stage, bool key_rows, bool value_rows) {
        const int key = uniform(t.u * kUnit), h = uniform(head_of(t.hk));
        const int boxes = min(npg, uniform((lens[t.b] - key + box - 1) >> lbox));
        uint8_t* st = ring + stage * STAGE;
        uint64_t* kb = bar + 2 * stage;
        const uint32_t bytes = boxes * box * (HD * (Q8 ? 1 : 2) + (Q8 ? NB * 2 : 0));
        if (elected()) {
            if (key_rows) mbar_arrive_expect_tx(kb, bytes);
            if (value_rows) mbar_arrive_expect_tx(kb + 1, bytes);
        }
        constexpr int ROW = Q8 ? HD : 128;   // bytes of a swizzled row
#pragma unroll 1
        for (int i = 0; i < boxes; ++i) {
            const int id = __shfl_sync(NCM_FULL, page, i), row = (key + i * box) & ((1 << p.log2ps) - 1);
            if (elected()) {
                if (key_rows) {
#pragma unroll
                    for (int j = 0; j < KB / (kUnit * ROW); ++j)
                        tma_load_4d(st + j * kUnit * ROW + i * box * ROW, &p.km, kb, j * 64, row, h, id);
                    if (Q8) tma_load_3d(st + 2 * KB + i * 128, &p.ksm, kb, row * NB, h, id);
                }
                if (value_rows) {
#pragma unroll
                    for (int j = 0; j < KB / (kUnit * ROW); ++j)
                        tma_load_4d(st + KB + j * kUnit * ROW + i * box * ROW, &p.vm, kb + 1, j * 64, row, h, id);
                    if (Q8) tma_load_3d(st + 2 * KB + SB + i * 128, &p.vsm, kb + 1, row * NB, h, id);
                }
            }
            __syncwarp();
        }
    };
    // Queries: 16-bit values as they are; over Q8_0 as 16-bit integers per block of 32 (high bytes in
    // qf[2 k], low bytes in qf[2 k + 1]), whose scales qs belong to this lane's two heads of the products.
    uint32_t qf[KS][NT][2];
    float qs[NB][NT][2];
    float o[KS][NT][4], m[NT][2], l[NT][2];
    auto begin = [&]() {          // the segment's queries, and empty sums
        const int h = head_of(c.hk), ch = c.hk - h * p.nchunk;
        const int heads = min(p.chunk, p.group - ch * p.chunk);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int head = t * 8 + r8;
            const uint16_t* q = static_cast<const uint16_t*>(p.q) + c.b * p.q_stride +
                                (int64_t)(h * p.group + ch * p.chunk + head) * HD;
            if (!Q8) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    qf[s][t][0] = head < heads ? __ldg(reinterpret_cast<const uint32_t*>(q + s * 16 + 2 * c4)) : 0u;
                    qf[s][t][1] = head < heads ? __ldg(reinterpret_cast<const uint32_t*>(q + s * 16 + 8 + 2 * c4)) : 0u;
                }
            } else {
                uint2 raw[NB][2];   // d = 32 k + 16 i + 4 c4 + 0..3
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        raw[k][i] = head < heads ? __ldg(reinterpret_cast<const uint2*>(q + 32 * k + 16 * i + 4 * c4)) : make_uint2(0, 0);
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    float x[8], top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 f0 = widen2<BF16>(raw[k][i].x), f1 = widen2<BF16>(raw[k][i].y);
                        x[4 * i] = f0.x; x[4 * i + 1] = f0.y; x[4 * i + 2] = f1.x; x[4 * i + 3] = f1.y;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
                    top = max_nan(top, __shfl_xor_sync(NCM_FULL, top, 1));
                    top = max_nan(top, __shfl_xor_sync(NCM_FULL, top, 2));
                    // 127 * 256: high bytes fit
                    const float inv = top > 0.0f && top < INFINITY ? 32512.0f / top : 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t v[4];
#pragma unroll
                        // low 16 bits
                        for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(fmaf(x[4 * i + e], inv, kIntBaseF));
                        const uint32_t v01 = __byte_perm(v[0], v[1], 0x5410), v23 = __byte_perm(v[2], v[3], 0x5410);
                        qf[2 * k][t][i] = __byte_perm(v01, v23, 0x7531);
                        qf[2 * k + 1][t][i] = __byte_perm(v01, v23, 0x6420);
                    }
                    // a query that is not finite: NaN
                    const float sc = top < INFINITY ? top * (1.0f / 32512.0f) : NAN;
                    qs[k][t][0] = __shfl_sync(NCM_FULL, sc, 8 * c4);
                    qs[k][t][1] = __shfl_sync(NCM_FULL, sc, 8 * c4 + 4);
                }
            }
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[s][t][i] = 0.0f;
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
        }
    };
    // d of o[s][t][i]: the int8 path's rows of the product are pairs of neighbouring d
    auto d_of = [&](int s, int i) { return s * 16 + (Q8 ? 2 * r8 + (i >> 1) : r8 + 8 * (i >> 1)); };
    auto sum_lanes = [&]() {      // l over the lanes that share a head
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[t][j] += __shfl_xor_sync(NCM_FULL, l[t][j], x);
                // a score that overflowed makes the row NaN: beside it every p is zero
                if (m[t][j] == INFINITY) l[t][j] = NAN;
            }
    };
    auto keep = [&](float* rows, float* ml) {   // a part, in shared memory
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int head = t * 8 + 2 * c4 + (i & 1);
#pragma unroll
                for (int s = 0; s < KS; ++s) rows[head * HD + d_of(s, i)] = o[s][t][i];
                if (r8 == 0 && i < 2) { ml[2 * head] = m[t][i]; ml[2 * head + 1] = l[t][i]; }
            }
    };
    int began = 0;                // first unit (of this warp) of the current segment
    bool failed = false;
    if (count > 0) begin();
    Place f = c;                  // the next unit to be fetched, and its pages
    int fetched = 0, fpage = 0;
    {
        // The first units' pages by one load: lane i of the unit i / npg.  The loads of the
        // queries above are on their way meanwhile.
        const int most = min(count, nst), mine = lane >> lnpg;   // 8 units of 4 boxes at most
        int page = 0;
        if (mine < most) {
            Place t = c;
            for (int i = 0; i < mine; ++i) next(t);
            page = page_at(t, lane & (npg - 1));
        }
        __syncwarp();
        for (; fetched < most; ++fetched) {
            issue(f, __shfl_sync(NCM_FULL, page, ((fetched << lnpg) + lane) & 31), fetched, true, true);
            next(f);
        }
        if (fetched < count) fpage = page_at(f, lane);
    }
    for (int i = 0, stage = 0, phase = 0; i < count && !failed; ++i) {
        uint8_t* st = ring + stage * STAGE;
        const uint32_t ka = smem_u32(st), va = ka + KB;
        const __half* ksc = reinterpret_cast<const __half*>(st + 2 * KB);
        __half* vsc = reinterpret_cast<__half*>(st + 2 * KB + SB);
        const int valid = lens[c.b] - c.u * kUnit;   // keys of this unit (32 or more: all)
        // scale rows lie 128 bytes apart per box when a box has few rows
        auto scale_at = [&](int row) { return (row >> lbox) * 64 + (row & (box - 1)) * NB; };
        // the scales of this lane's four rows
        auto scales_of = [&](const __half* at, float (*to)[NB]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[NB / 2];
                const __half* row = at + scale_at(r8 + 8 * i);
                if (NB == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(row);
                else w[0] = *reinterpret_cast<const uint32_t*>(row);
#pragma unroll
                for (int k = 0; k < NB / 2; ++k) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                    to[i][2 * k] = f.x; to[i][2 * k + 1] = f.y;
                }
            }
        };
        // (the vote brings the lanes together again: ldmatrix and mma want them all)
        if (!__all_sync(NCM_FULL, mbar_wait(bar + 2 * stage, phase, kPagedWaitNs))) { failed = true; break; }
        // scores: rows = keys, columns = heads
        float s[2][NT][4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[a][t][j] = 0.0f;
        if (!Q8) {
            const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const int col = 2 * k + (lane >> 4);   // 16-byte column
                    uint32_t x[4];
                    ldsm4(x, ka + (col >> 3) * (kUnit * 128) + (a * 16 + row) * 128 + (((col & 7) ^ (row & 7)) << 4));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma16816<BF16>(s[a][t], x[0], x[1], x[2], x[3], qf[k][t][0], qf[k][t][1]);
                }
        } else {
            const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
            const int swz = HD == 128 ? (row & 7) : ((row >> 1) & 3);
            float sk[4][NB];
            scales_of(ksc, sk);
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    const int col = 2 * k + (lane >> 4);
                    uint32_t x[4];
                    ldsm4(x, ka + (a * 16 + row) * HD + ((col ^ swz) << 4));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float hi[4], lo[4];
                        imma16832<false>(hi, x[0], x[1], x[2], x[3], qf[2 * k][t][0], qf[2 * k][t][1]);
                        imma16832<true>(lo, x[0], x[1], x[2], x[3], qf[2 * k + 1][t][0], qf[2 * k + 1][t][1]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s[a][t][j] = fmaf(joined(hi[j], lo[j]), sk[2 * a + (j >> 1)][k] * qs[k][t][j & 1], s[a][t][j]);
                    }
                }
        }
        if (valid < kUnit) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (a * 16 + r8 + 8 * (j >> 1) >= valid) s[a][t][j] = -INFINITY;
        }
        // Running maximum, in units of log2.  It need not be exact: it is moved only when a
        // score has passed it by more than 2^8, so p stays below 2^8 and the sums are rarely rescaled.
        bool over = false;
        float top[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[t][j] = fmaxf(fmaxf(s[0][t][j], s[0][t][j + 2]), fmaxf(s[1][t][j], s[1][t][j + 2])) * p.scale_log2;
                over |= top[t][j] > m[t][j] + 8.0f;
            }
        if (__any_sync(NCM_FULL, over)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float v = top[t][j];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(NCM_FULL, v, x));
                    v = fmaxf(v, m[t][j]);
                    const float a = v == m[t][j] ? 1.0f : ex2(m[t][j] - v);
                    m[t][j] = v;
                    l[t][j] *= a;
#pragma unroll
                    for (int k = 0; k < KS; ++k) { o[k][t][j] *= a; o[k][t][j + 2] *= a; }
                }
        }
        // all lanes have their scores (the vote): K has been read
        if (ONE && fetched < count) issue(f, fpage, stage, true, false);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float mm = m[t][j & 1] == -INFINITY ? 0.0f : m[t][j & 1] - kLift;
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    s[a][t][j] = ex2(fmaf(s[a][t][j], p.scale_log2, -mm));
                    l[t][j & 1] += s[a][t][j];
                }
            }
        if (!__all_sync(NCM_FULL, mbar_wait(bar + 2 * stage + 1, phase, kPagedWaitNs))) { failed = true; break; }
        if (valid < kUnit) {   // rows behind the last key may hold anything: zero x NaN is NaN
            constexpr int ROW = Q8 ? HD : 128;
            for (int e = lane; e < (kUnit - valid) * (ROW / 16); e += 32) {
                const int row = valid + e / (ROW / 16);
#pragma unroll
                for (int j = 0; j < KB / (kUnit * ROW); ++j)
                    *reinterpret_cast<uint4*>(st + KB + j * kUnit * ROW + row * ROW + (e % (ROW / 16)) * 16) = make_uint4(0, 0, 0, 0);
            }
            if (Q8)
                for (int e = lane; e < (kUnit - valid) * NB; e += 32) vsc[scale_at(valid + e / NB) + e % NB] = __half(0.0f);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into this stage
            __syncwarp();
        }
        if (!Q8) {
            const int key = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                uint32_t b[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {   // p in the inputs' type: a rounding of half a step, as the output's
                    b[t][0] = transposed(pack2(BF16, s[a][t][0], s[a][t][1]));
                    b[t][1] = transposed(pack2(BF16, s[a][t][2], s[a][t][3]));
                }
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const int col = 2 * k + ((lane >> 3) & 1);
                    uint32_t x[4];
                    ldsm4t(x, va + (col >> 3) * (kUnit * 128) + (a * 16 + key) * 128 + (((col & 7) ^ (key & 7)) << 4));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma16816<BF16>(o[k][t], x[0], x[1], x[2], x[3], b[t][0], b[t][1]);
                }
            }
        } else {
            // The weights p times scale of this unit's 32 keys as 16-bit integers (two bytes, two
            // products) per head and block, relative to the largest such product: relative to the
            // largest p times the largest scale (69.5 us where this takes 70.9: 48 sequences of 300
            // to 6000, 32 / 8 heads of 128) a key of large p and small scale would take the others'
            // bits.  The largest is rounded up to bf16's eight bits, two heads to a register for the
            // shuffles: each weight is off by 1 / 130000 of it at most.  A NaN among the products
            // becomes the largest, and with it the unit's share of the output.
            const int swz = HD == 128 ? (lane & 7) : ((lane >> 1) & 3);
            float sv[4][NB];
            uint32_t top2[NB][NT];
            scales_of(vsc, sv);
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float v[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        v[j] = max_nan(max_nan(s[0][t][j] * sv[0][k], s[0][t][j + 2] * sv[1][k]),
                                       max_nan(s[1][t][j] * sv[2][k], s[1][t][j + 2] * sv[3][k])) * (1.0f + 0x1p-8f);
                    top2[k][t] = pack2(true, v[0], v[1]);
                }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1)
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                    for (int t = 0; t < NT; ++t) top2[k][t] = max_nan_bf16x2(top2[k][t], __shfl_xor_sync(NCM_FULL, top2[k][t], x));
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                uint32_t hi[NT][2], lo[NT][2];
                float step[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float r[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float v = max_nan(__uint_as_float(j ? top2[k][t] & 0xffff0000u : top2[k][t] << 16), 0x1p-84f);
                        r[j] = __fdividef(65534.0f, v);
                        step[t][j] = v * (1.0f / 65534.0f);
                    }
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        uint32_t w[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float f = sv[2 * a + j][k];
                            w[j] = transposed(__byte_perm(__float_as_uint(fmaf(s[a][t][2 * j] * f, r[0], 0x1p23f)),
                                                          __float_as_uint(fmaf(s[a][t][2 * j + 1] * f, r[1], 0x1p23f)), 0x5410));
                        }
                        hi[t][a] = __byte_perm(w[0], w[1], 0x7531);   // keys 16 a + 2 c4, + 1, + 8, + 9
                        lo[t][a] = __byte_perm(w[0], w[1], 0x6420);
                    }
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {   // 16 values of d; x[i]: keys 8 i + 2 c4, + 1, of d 2 r8 and 2 r8 + 1
                    uint32_t x[4];
                    ldsm4t(x, va + lane * HD + (((2 * k + g) ^ swz) << 4));
                    const uint32_t a0 = __byte_perm(x[0], x[1], 0x6420), a1 = __byte_perm(x[0], x[1], 0x7531);
                    const uint32_t a2 = __byte_perm(x[2], x[3], 0x6420), a3 = __byte_perm(x[2], x[3], 0x7531);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float h[4], w[4];
                        imma16832<true>(h, a0, a1, a2, a3, hi[t][0], hi[t][1]);
                        imma16832<true>(w, a0, a1, a2, a3, lo[t][0], lo[t][1]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            o[2 * k + g][t][j] = fmaf(joined(h[j], w[j]), step[t][j & 1], o[2 * k + g][t][j]);
                    }
                }
            }
        }
        __syncwarp();
        if (fetched < count) {
            issue(f, fpage, stage, !ONE, true);
            next(f);
            if (++fetched < count) fpage = page_at(f, lane);
        }
        if (++stage == nst) { stage = 0; phase ^= 1; }

        if (c.u + 1 == c.n || i + 1 == count) {   // the segment, or this warp's part of it, is complete
            const bool whole = c.u + 1 == c.n && i - began + 1 == c.n;
            sum_lanes();
            if (whole) {
                const int h = head_of(c.hk), ch = c.hk - h * p.nchunk;
                const int heads = min(p.chunk, p.group - ch * p.chunk);
                uint16_t* out = static_cast<uint16_t*>(p.out) + c.b * p.out_stride +
                                (int64_t)(h * p.group + ch * p.chunk) * HD;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int head = t * 8 + 2 * c4 + (j & 1);
                        const float inv = inverse(l[t][j & 1]);
                        if (head < heads)
#pragma unroll
                            for (int k = 0; k < KS; ++k)
                                out[head * HD + d_of(k, j)] = (uint16_t)pack2(BF16, scaled(o[k][t][j], inv), 0.0f);
                    }
            } else {
                const bool at_end = i + 1 == count;
                int* e = ent + 4 * (2 * warp + (at_end ? 1 : 0));
                if (lane == 0) {
                    const int base = prefix[c.b] * HK + c.hk * (prefix[c.b + 1] - prefix[c.b]);
                    e[0] = c.b; e[1] = c.hk; e[2] = base; e[3] = base + c.n;
                }
                if (!at_end) keep(first + warp * GH * HD, first_ml + warp * GH * 2);
            }
            if (i + 1 < count) { next(c); began = i + 1; begin(); }
        } else {
            next(c);
        }
    }
    if (failed) {      // (copies in flight are waited for, again with the limit)
        set_dev_error(p.err, NCM_DEVERR_MBAR_TIMEOUT);
        for (int i = 0; i < 2 * nst; ++i)
            for (int phase = 0; phase < 2 && lane == 0; ++phase) mbar_wait(bar + i, phase, kPagedWaitNs / 16);
        __syncwarp();
    }
    __syncthreads();   // every copy has landed: the ring holds the warps' last parts now
    float* last = reinterpret_cast<float*>(smem);
    float* last_ml = last + W * GH * HD;
    if (count > 0 && ent[4 * (2 * warp + 1)] >= 0) keep(last + warp * GH * HD, last_ml + warp * GH * 2);
    __syncthreads();

    // ---- the CTA's parts, joined where they are of one segment
    float* weights = last_ml + W * GH * 2;   // [parts + 1][GH] of the join over CTAs
    for (int e = 0; e < 2 * W;) {
        const int4 seg = *reinterpret_cast<const int4*>(ent + 4 * e);
        if (seg.x < 0) { ++e; continue; }
        const int b = seg.x, hk = seg.y, sb = seg.z, se = seg.w, h = head_of(hk), ch = hk - h * p.nchunk;
        uint32_t of = 0;   // the entries of this segment: those up to the next one's first
        int e1 = e;
        for (; e1 < 2 * W; ++e1) {
            const int4 o = *reinterpret_cast<const int4*>(ent + 4 * e1);
            if (o.x < 0) continue;
            if (o.x != b || o.y != hk) break;
            of |= 1u << e1;
        }
        const int heads = min(p.chunk, p.group - ch * p.chunk);
        const int64_t out_at = b * p.out_stride + (int64_t)(h * p.group + ch * p.chunk) * HD;
        const bool inside = sb >= u0 && se <= u1;
        const int slot = sb < u0 ? 0 : 1;
        float* rows = p.part + (int64_t)(2 * blockIdx.x + slot) * p.chunk * HD;
        float* mls = p.part + (int64_t)2 * gridDim.x * p.chunk * HD;
        static_assert(2 * W <= 32, "an entry per lane");
        for (int head = warp; head < heads; head += W) {   // lane y: entry y; then lane: four values of d
            const bool has = lane < 2 * W && (of >> lane & 1);
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (has) ml = *reinterpret_cast<const float2*>(((lane & 1) ? last_ml : first_ml) + ((lane >> 1) * GH + head) * 2);
            float top = ml.x;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(NCM_FULL, top, x));
            const float weight = part_weight(ml.x, top);
            float sum = weight * ml.y;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(NCM_FULL, sum, x);
            const int d = 4 * lane;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t left = of; left; left &= left - 1) {
                const int y = __ffs(left) - 1;
                const float w = __shfl_sync(NCM_FULL, weight, y);
                if (d >= HD) continue;
                const float4 v = *reinterpret_cast<const float4*>(((y & 1) ? last : first) + ((y >> 1) * GH + head) * HD + d);
                acc.x = fmaf(w, v.x, acc.x); acc.y = fmaf(w, v.y, acc.y);
                acc.z = fmaf(w, v.z, acc.z); acc.w = fmaf(w, v.w, acc.w);
            }
            if (d >= HD) continue;
            if (inside) {
                const float inv = inverse(sum);
                store_out<BF16>(p.out, out_at + head * HD + d, scaled(acc, inv));
            } else {
                *reinterpret_cast<float4*>(rows + head * HD + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(mls + ((int64_t)(2 * blockIdx.x + slot) * p.chunk + head) * 2) = make_float2(top, sum);
            }
        }
        if (!inside) {
            // The CTA that stores its part last joins them all, in the CTAs' order: the result
            // does not depend on which one that is.  Nobody waits.
            const int i0 = sb / share, i1 = (se - 1) / share;
            // (the barriers carry the other threads' stores and loads over one thread's release
            // and acquire)
            __syncthreads();
            if (tid == 0) {
                unsigned before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + i0) : "memory");
                sums[4 * W] = (int)before == i1 - i0;
                if (sums[4 * W]) p.counters[i0] = 0;
            }
            __syncthreads();
            if (sums[4 * W]) {
                const int np = i1 - i0 + 1;
                auto part_of = [&](int i) { return (int64_t)(2 * (i0 + i) + (i == 0 ? 1 : 0)); };
                if (np <= 8) {   // one round of loads
                    for (int x = tid; x < heads * (HD / 4); x += W * 32) {
                        const int head = x / (HD / 4), d = 4 * (x % (HD / 4));
                        float2 ml[8];
                        float4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int64_t at = part_of(min(i, np - 1)) * p.chunk + head;
                            ml[i] = __ldcg(reinterpret_cast<const float2*>(mls + at * 2));
                            v[i] = __ldcg(reinterpret_cast<const float4*>(p.part + at * HD + d));
                        }
                        float top = -INFINITY, sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[i].x);
                        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (i >= np) break;
                            const float w = part_weight(ml[i].x, top);
                            acc.x = fmaf(w, v[i].x, acc.x); acc.y = fmaf(w, v[i].y, acc.y);
                            acc.z = fmaf(w, v[i].z, acc.z); acc.w = fmaf(w, v[i].w, acc.w);
                            sum = fmaf(w, ml[i].y, sum);
                        }
                        const float inv = inverse(sum);
                        store_out<BF16>(p.out, out_at + head * HD + d, scaled(acc, inv));
                    }
                    e = e1;
                    continue;
                }
                // weights of the parts, one warp per head in turn, and the inverse of their joint sum
                for (int head = warp; head < heads; head += W) {
                    float top = -INFINITY, sum = 0.0f;
                    for (int i = lane; i < np; i += 32) top = fmaxf(top, __ldcg(mls + (part_of(i) * p.chunk + head) * 2));
#pragma unroll
                    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(NCM_FULL, top, x));
                    for (int i = lane; i < np; i += 32) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(mls + (part_of(i) * p.chunk + head) * 2));
                        const float w = part_weight(ml.x, top);
                        weights[i * GH + head] = w;
                        sum = fmaf(w, ml.y, sum);
                    }
#pragma unroll
                    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(NCM_FULL, sum, x);
                    if (lane == 0) weights[np * GH + head] = inverse(sum);
                }
                __syncthreads();
                for (int x = tid; x < heads * (HD / 4); x += W * 32) {
                    const int head = x / (HD / 4), d = 4 * (x % (HD / 4));
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (int i = 0; i < np; ++i) {
                        const float w = weights[i * GH + head];
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + (part_of(i) * p.chunk + head) * HD + d));
                        acc.x = fmaf(w, v.x, acc.x); acc.y = fmaf(w, v.y, acc.y);
                        acc.z = fmaf(w, v.z, acc.z); acc.w = fmaf(w, v.w, acc.w);
                    }
                    store_out<BF16>(p.out, out_at + head * HD + d, scaled(acc, weights[np * GH + head]));
                }
                __syncthreads();
            }
        }
        e = e1;
    }
}

// ------------------------------------------------------------------ host side
int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
}
bool aligned16(const void* p) { return (((uintptr_t)p) & 15) == 0; }
bool aligned4(const void* p) { return (((uintptr_t)p) & 3) == 0; }
bool is_16bit(int t) { return t == NCM_TYPE_F16 || t == NCM_TYPE_BF16; }

// What every call on a cache checks; null when it is sound.
const char* cache_error(const ncm_paged_kv* kv) {
    if (!kv) return "no cache";
    if (!is_16bit(kv->type) && kv->type != NCM_TYPE_Q8_0) return "cache type must be F16, BF16 or Q8_0";
    if (kv->head_dim != 64 && kv->head_dim != 128) return "head_dim must be 64 or 128";
    if (kv->page_size < 8 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
        return "page_size must be a power of two from 8 to 256";
    if (kv->kv_heads < 1 || kv->kv_heads > 1024) return "kv_heads must be 1 to 1024";
    if (kv->pages < 1 || kv->pages > 0x7fffffff) return "pages must be 1 to 2^31 - 1";
    const int64_t dense = (int64_t)kv->kv_heads * kv->page_size * kv->head_dim;
    if (kv->page_stride && (kv->page_stride < dense || kv->page_stride % 16 || kv->page_stride > ((int64_t)1 << 38)))
        return "page_stride must be a multiple of 16 elements and hold a page";
    if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v)) return "k and v must be 16-byte aligned";
    if (kv->type == NCM_TYPE_Q8_0 && (!kv->k_scales || !kv->v_scales || !aligned16(kv->k_scales) || !aligned16(kv->v_scales)))
        return "a Q8_0 cache needs 16-byte aligned scales";
    return nullptr;
}
int64_t page_stride_of(const ncm_paged_kv* kv) {
    return kv->page_stride ? kv->page_stride : (int64_t)kv->kv_heads * kv->page_size * kv->head_dim;
}

int chunk_of(int group, int* nchunk) {   // heads of a group per segment: 16 at most, evenly
    *nchunk = (group + 15) / 16;
    return (group + *nchunk - 1) / *nchunk;
}

int paged_maps(const ncm_paged_kv* kv, int box, PagedAttnParams& p) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return 1;
    const bool q8 = kv->type == NCM_TYPE_Q8_0;
    const cuuint64_t es = q8 ? 1 : 2, hd = kv->head_dim, ps = kv->page_size, kh = kv->kv_heads, np = kv->pages;
    const cuuint64_t dim[4] = {hd, ps, kh, np};
    const cuuint64_t stride[3] = {hd * es, ps * hd * es, (cuuint64_t)page_stride_of(kv) * es};
    const cuuint32_t boxes[4] = {q8 ? (cuuint32_t)hd : 64u, (cuuint32_t)box, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle swz = q8 && hd == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const CUtensorMapDataType t = q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    void* base[2] = {kv->k, kv->v};
    CUtensorMap* map[2] = {&p.km, &p.vm};
    for (int i = 0; i < 2; ++i)
        if (enc(map[i], t, 4, base[i], dim, stride, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return 1;
    if (!q8) return 0;
    const cuuint64_t nb = hd / 32, sdim[3] = {ps * nb, kh, np}, sstride[2] = {ps * nb * 2, kh * ps * nb * 2};
    const cuuint32_t sbox[3] = {(cuuint32_t)(box * nb), 1, 1};
    void* sbase[2] = {kv->k_scales, kv->v_scales};
    CUtensorMap* smap[2] = {&p.ksm, &p.vsm};
    for (int i = 0; i < 2; ++i)
        if (enc(smap[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, sbase[i], sdim, sstride, sbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) !=
            CUDA_SUCCESS)
            return 1;
    return 0;
}

template <bool BF16, bool Q8, int HD, int NT, int W>
int paged_attn_run(PagedAttnParams& p, int grid, cudaStream_t s) {
    const int stage = 2 * (kUnit * HD * (Q8 ? 1 : 2) + (Q8 ? 512 : 0));
    const int fixed = W * 8 * NT * (HD + 2) * 4 + 2 * W * 16 + (4 * W + 1) * 4 + (2 * p.batch + 1) * 4;
    int n = 1;   // stages: as many as fit, 8 at most
    while (!one_stage(Q8, HD, NT) && n < 8 && fixed + W * (n + 1) * (stage + 16) <= kPagedSmem) ++n;
    p.nstages = n;
    auto fn = paged_attn_kernel<BF16, Q8, HD, NT, W>;
    if (int r = set_smem_limit((const void*)fn, kPagedSmem)) return r;
    fn<<<grid, W * 32, fixed + W * n * (stage + 16), s>>>(p);
    return (int)cudaGetLastError();
}
template <bool BF16, bool Q8>
int paged_attn_pick(PagedAttnParams& p, int hd, int grid, cudaStream_t s) {
    const bool two = p.chunk > 8;
    // Warps of a CTA.  Over Q8_0 each warp waits on its own instructions (0.53 issued a cycle and
    // scheduler, no pipe above 28 %): as many as the registers allow without more stages falling out.
    // 16-bit values need only enough in flight.  Measured in us, 32 / 8 heads but where said:
    //   16-bit, heads of 128: 64 sequences of 1 to 8192  6 warps of two stages 166.6, 7 of one 168.9, 9 169.9;
    //     48 of 300 to 6000  97.3, 95.0, 98.6; 4 of those  19.8, 18.4, 18.9
    //   16-bit, heads of 64: 64 of 300 to 6000  8 warps 75.0, 10 75.1, 12 75.1; 64 of 300 to 8000  83.0,
    //     80.9, 81.7; 4 of 300 to 6000  13.2, 14.0, 14.6
    //   Q8_0, heads of 128: 48 of 300 to 6000  8 warps 77.5, 10 79.8, 12 71.1; 8 / 1 heads, 64 of them
    //     26.2, 26.3, 26.0
    //   Q8_0, heads of 64: 48 of 300 to 6000  10 warps 55.0, 12 50.4, 14 52.7
    //   9 to 16 heads a segment, 48 of 300 to 6000: heads of 64 (12) 6 warps 64.6, 8 65.7, 10 65.3; Q8_0 (16) 94.9,
    //     75.6, 81.2; heads of 128 (12) 3 warps 115, 4 110.7, 5 106.2; Q8_0 (16) 6 warps 137, 7 123, 8 109
    if (hd == 64)
        return two ? paged_attn_run<BF16, Q8, 64, 2, 8>(p, grid, s) : paged_attn_run<BF16, Q8, 64, 1, Q8 ? 12 : 10>(p, grid, s);
    if (two) return paged_attn_run<BF16, Q8, 128, 2, Q8 ? 8 : 4>(p, grid, s);
    return paged_attn_run<BF16, Q8, 128, 1, Q8 ? 12 : 7>(p, grid, s);
}

int bad(const char* what) { return set_error(NCM_EINVAL, what); }

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" ncm_status ncm_paged_append(const ncm_paged_kv* kv, int in_type, const void* q, int64_t q_stride, const void* k,
                                       int64_t k_stride, const void* v, int64_t v_stride, void* q_out, int q_out_type,
                                       int tokens, int heads, int batch, const int* cu_tokens, const int* lengths,
                                       const int* page_table, int table_width, const float* rope, int rope_len,
                                       int rope_half, int rope_style, int* err, void* stream) {
    if (const char* e = cache_error(kv)) return bad(e);
    const int hd = kv->head_dim, es = in_type == NCM_TYPE_F32 ? 4 : 2;
    if (in_type != NCM_TYPE_F32 && !is_16bit(in_type)) return bad("in_type must be F32, F16 or BF16");
    if (tokens < 0 || batch < 0 || heads < 0 || heads > 4096 || table_width < 0) return bad("bad append sizes");
    if (heads && !is_16bit(q_out_type)) return bad("q_out_type must be F16 or BF16");
    if (!cu_tokens && tokens != batch) return bad("without cu_tokens there is one token per sequence");
    if (rope_style != NCM_ROPE_PAIRS && rope_style != NCM_ROPE_HALVES) return bad("bad rope_style");
    if (rope && (rope_len < 1 || rope_half < 2 || rope_half % 2 || rope_half > hd / 2 || !aligned16(rope)))
        return bad("the rotation table needs rope_len >= 1, an even rope_half of at most head_dim / 2, 16-byte alignment");
    if (rope && rope_style == NCM_ROPE_HALVES && rope_half != hd / 2) return bad("NCM_ROPE_HALVES rotates the whole head");
    if (tokens == 0) return NCM_OK;
    if (!k || !v || !lengths || !page_table || (heads && (!q || !q_out))) return bad("null pointer");
    if (batch < 1 || table_width < 1 || table_width > (1 << 22)) return bad("bad append sizes");
    const int64_t wide[3] = {(int64_t)heads * hd, (int64_t)kv->kv_heads * hd, (int64_t)kv->kv_heads * hd};
    const void* src[3] = {heads ? q : nullptr, k, v};
    int64_t stride[3] = {q_stride, k_stride, v_stride};
    for (int i = 0; i < 3; ++i) {
        if (!stride[i]) stride[i] = wide[i];
        if (stride[i] < wide[i] || stride[i] * es % 16 || stride[i] > ((int64_t)1 << 40) || !aligned16(src[i]))
            return bad("q, k and v rows must be 16-byte aligned and at least a token apart");
    }
    if (!aligned16(q_out)) return bad("q_out must be 16-byte aligned");
    if (!aligned4(cu_tokens) || !aligned4(lengths) || !aligned4(page_table) || !aligned4(err)) return bad("int arrays must be 4-byte aligned");
    const void* check[] = {k, v, kv->k, kv->v, kv->k_scales, kv->v_scales, lengths, page_table, cu_tokens, rope, src[0],
                           heads ? q_out : nullptr, err};
    if (const char* e = device_pointers_error(check, sizeof check / sizeof *check)) return bad(e);
    AppendParams p;
    memset(&p, 0, sizeof p);
    p.q = src[0]; p.k = k; p.v = v; p.q_stride = stride[0]; p.k_stride = stride[1]; p.v_stride = stride[2];
    p.q_out = q_out; p.heads = heads; p.kv_heads = kv->kv_heads; p.hd = hd; p.tokens = tokens; p.batch = batch;
    p.cu = cu_tokens; p.lengths = lengths; p.table = page_table; p.table_width = table_width;
    p.log2ps = log2_of(kv->page_size); p.pages = kv->pages; p.page_stride = page_stride_of(kv);
    p.rope = reinterpret_cast<const float2*>(rope); p.rope_len = rope_len; p.rope_half = rope_half;
    p.halves = rope_style == NCM_ROPE_HALVES;
    p.kind = kv->type; p.out_bf16 = q_out_type == NCM_TYPE_BF16;
    p.kc = kv->k; p.vc = kv->v; p.ks = (__half*)kv->k_scales; p.vs = (__half*)kv->v_scales;
    p.err = err;
    // Few tokens: a thread for each 16 values, for latency (64 tokens of 32 + 16 heads: 3.0 us, with
    // 128 threads 4.1).  Many: 128 threads, so that more tokens are on the way at once (7062 tokens of
    // 32 + 16 f32 heads: 46.9 us with 384 threads, 42.8 with 192, 42.6 with 128, 43.1 with 64).
    const int threads = std::min(tokens < 4 * num_sms() ? 512 : 128, ((heads + 2 * kv->kv_heads) * (hd / 16) + 31) / 32 * 32);
    cudaStream_t s = (cudaStream_t)stream;
    if (in_type == NCM_TYPE_F32) paged_append_kernel<float><<<tokens, threads, 0, s>>>(p);
    else if (in_type == NCM_TYPE_F16) paged_append_kernel<__half><<<tokens, threads, 0, s>>>(p);
    else paged_append_kernel<__nv_bfloat16><<<tokens, threads, 0, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NCM_OK : set_error(NCM_ECUDA, cudaGetErrorString(e));
}

extern "C" ncm_status ncm_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes) {
    if (!bytes || heads < 1 || kv_heads < 1 || heads % kv_heads || (head_dim != 64 && head_dim != 128))
        return bad("bad paged attention sizes");
    int nchunk = 0;
    const int chunk = chunk_of(heads / kv_heads, &nchunk), grid = num_sms();
    *bytes = 4096 + (size_t)2 * grid * chunk * (head_dim + 2) * 4;
    return NCM_OK;
}

extern "C" ncm_status ncm_paged_attention(const ncm_paged_kv* kv, void* out, int64_t out_stride, const void* q,
                                          int64_t q_stride, int q_type, int batch, int heads, const int* lengths,
                                          const int* page_table, int table_width, float scale, void* workspace,
                                          size_t workspace_bytes, int* err, void* stream) {
    if (const char* e = cache_error(kv)) return bad(e);
    const int hd = kv->head_dim;
    if (!is_16bit(q_type)) return bad("q_type must be F16 or BF16");
    if (kv->type != NCM_TYPE_Q8_0 && kv->type != q_type) return bad("q and a 16-bit cache must be of one type");
    if (batch < 0 || heads < 1 || heads > 65536 || heads % kv->kv_heads || table_width < 0) return bad("bad attention sizes");
    if (!(scale >= 0.0f) || scale > 2.0e38f) return bad("scale must be positive, below 2e38 (0: 1 / sqrt(head_dim))");
    if (batch == 0) return NCM_OK;
    if (!out || !q || !lengths || !page_table || !workspace) return bad("null pointer");
    if (table_width < 1 || (int64_t)table_width * kv->page_size > (1 << 22))
        return bad("a sequence's pages must hold 1 to 2^22 tokens");
    const int64_t wide = (int64_t)heads * hd;
    if (!q_stride) q_stride = wide;
    if (!out_stride) out_stride = wide;
    if (q_stride < wide || out_stride < wide || q_stride % 8 || out_stride % 8 || q_stride > ((int64_t)1 << 40) ||
        out_stride > ((int64_t)1 << 40) || !aligned16(q) || !aligned16(out) || !aligned16(workspace))
        return bad("q and out rows must be 16-byte aligned and at least a token apart");
    if (!aligned4(lengths) || !aligned4(page_table) || !aligned4(err)) return bad("int arrays must be 4-byte aligned");
    size_t need = 0;
    if (ncm_paged_attention_workspace(heads, kv->kv_heads, hd, &need) || workspace_bytes < need)
        return bad("workspace smaller than ncm_paged_attention_workspace says");
    const void* check[] = {out, q, kv->k, kv->v, kv->k_scales, kv->v_scales, lengths, page_table, workspace, err};
    if (const char* e = device_pointers_error(check, sizeof check / sizeof *check)) return bad(e);
    PagedAttnParams p;
    memset(&p, 0, sizeof p);
    p.box_rows = std::min(kv->page_size, kUnit);
    if (paged_maps(kv, p.box_rows, p)) return set_error(NCM_ECUDA, "cuTensorMapEncodeTiled failed for the cache");
    const int grid = num_sms();
    if (grid > 1024) return set_error(NCM_EUNSUPPORTED, "more than 1024 SMs");
    p.q_stride = q_stride; p.out_stride = out_stride;
    p.table_width = table_width; p.heads = heads; p.kv_heads = kv->kv_heads; p.group = heads / kv->kv_heads;
    p.chunk = chunk_of(p.group, &p.nchunk);
    p.log2ps = log2_of(kv->page_size); p.pages = kv->pages;
    p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)hd)) * 1.4426950408889634f;
    p.counters = (unsigned*)workspace;
    p.part = (float*)((char*)workspace + 4096);
    p.err = err;
    // positions in the row of units, padded to pieces, fit 32 bits
    // 4 * 12: a piece
    const int64_t most = ((int64_t)table_width * kv->page_size / kUnit + 1 + 48) * kv->kv_heads * p.nchunk;
    const int step = (int)std::min<int64_t>(kPagedBatch, (int64_t)0x7fff0000 / most);
    if (step < 1) return set_error(NCM_EUNSUPPORTED, "a sequence's pages hold too many tokens for so many heads");
    cudaStream_t s = (cudaStream_t)stream;
    for (int b = 0; b < batch; b += step) {
        p.batch = std::min(step, batch - b);
        p.q = (const uint16_t*)q + b * q_stride;
        p.out = (uint16_t*)out + b * out_stride;
        p.lengths = lengths + b;
        p.table = page_table + (int64_t)b * table_width;
        const bool bf16 = q_type == NCM_TYPE_BF16, q8 = kv->type == NCM_TYPE_Q8_0;
        const int r = bf16 ? (q8 ? paged_attn_pick<true, true>(p, hd, grid, s) : paged_attn_pick<true, false>(p, hd, grid, s))
                           : (q8 ? paged_attn_pick<false, true>(p, hd, grid, s) : paged_attn_pick<false, false>(p, hd, grid, s));
        if (r) return set_error(NCM_ECUDA, cudaGetErrorString((cudaError_t)r));
    }
    return NCM_OK;
}
