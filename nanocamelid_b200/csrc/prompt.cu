// Attention over whole prompts: packed sequences of different lengths, grouped heads, causal
// or not, on the tcgen05 tensor cores.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j
//
// One CTA per SM walks over work items.  An item is one key-value head of one sequence and
// 2 x 128 query rows, a row being one (token, head of the group): all heads of a group share
// the K and V tiles, and a short prompt still fills the tile's rows.  Twelve warps:
//   0-3, 4-7  softmax of query tile 0 / 1, one thread per row: scores from TMEM, maximum,
//             exponentials, p back into TMEM (over the scores), and at the end the output;
//   8         TMA: queries, then K and V tiles of 128 keys into a ring;
//   9         issues the tensor-core products S = Q K^T and O += P V;
//   10, 11    look over the V tiles at the mask's edge: a key that a mask hides has p = 0, but
//             0 x infinity is not 0, so what is not finite there is taken out and given back
//             in the epilogue to the rows that do see it.
// While one tile's softmax runs, the tensor cores work on the other's products.  The softmax
// takes a tile's 128 keys in two steps of 64, whose p the tensor cores take one by one.
// TMEM columns: 128 x: S of tile x, and over it P, 64 h the step's; 256 + 128 x: O.
// What was slower, at one prompt of 8192 (32 / 8 heads of 128, 523 us then): an issuing warp for
// each tile (579), sixteen softmax warps (530), scores in units of 64 keys, double buffered (560:
// a product with N = 64 takes 50 cycles of the tensor cores, one with N = 128 64); and with heads
// of 64, where TMEM has room for it, P beside S, so that the next scores need not wait for the
// products (12 ragged prompts: 111 us against 102).
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

namespace ncm {
namespace {

constexpr int kRows = 128;               // query rows of a tile, and keys of a K or V tile
constexpr int kUnitKeys = 64;            // keys of one step of the softmax
constexpr int kPromptThreads = 384;
constexpr int kPromptBatch = 1024;       // sequences of one launch
// Exponentials of every eight that the FMA pipe computes: 0, 1, 2, 3 take 106.7, 103.7, 101.5, 102.7
// us for 12 ragged prompts, 32 / 8 heads of 64, in F16 and 108, 105 to 109, 101 to 105, 105 to 110 in BF16.
// With heads of 128 (4 chunks over 4000 keys, 64 / 8) the power cap moves each from 145 to 156 in BF16
// and from 162 to 182 in F16, and the four do not differ beyond that.
constexpr int kPolyOf8 = 2;
constexpr int kPromptSmem = 232448;
constexpr uint64_t kPromptWaitNs = 2000000000ull;

struct alignas(64) PromptParams {
    CUtensorMap qm;                      // {hd, group, kv_heads, tokens}, box {64, group, 1, tokens of a tile}
    CUtensorMap km, vm;                  // {hd, kv_heads, tokens}, box {64, 1, 128}
    void* out;
    const void* v;
    int64_t out_stride, v_stride;        // elements between tokens
    const int *cu_q, *cu_k;
    int batch, kv_heads, group, tokens;  // tokens: of a tile, 128 / group
    int before;                          // sequences of earlier launches, whose starts lie before cu_q
    int total_q, total_k, causal;
    float scale_log2;
    int* err;
};

__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// One lane of a converged warp, in a form that the compiler knows for one: the operands of the
// instructions under it stay in uniform registers.
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle, in units of 16 bytes.  Rows of 128 bytes
// in groups of eight (1024 bytes apart).  K-major (Q, K): the leading offset is not used.
// MN-major (V: keys x d, d contiguous): 64 values of d lie in one 128-byte row; the next 64 lie
// `lead` bytes on, the next eight keys 1024 bytes on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// Instruction descriptor of kind::f16: f32 accumulators, A and B f16 or bf16, M 128, N, B K-major or MN-major.
__host__ __device__ constexpr uint32_t inst_desc(bool bf16, int n, bool b_mn) {
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (b_mn ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t inst, bool add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(inst), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t inst, bool add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
        ::"r"(d), "r"(a), "l"(b), "r"(inst), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define NCM_R8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])
#define NCM_W8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define NCM_U8(r, i) "+r"((r)[i]), "+r"((r)[i + 1]), "+r"((r)[i + 2]), "+r"((r)[i + 3]), "+r"((r)[i + 4]), "+r"((r)[i + 5]), "+r"((r)[i + 6]), "+r"((r)[i + 7])
// Waits for this thread's TMEM loads.  It names what they loaded, so that no use of it is moved
// before the wait (`landed` does that for further registers).
__device__ __forceinline__ void wait_ld(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : NCM_U8(r, 0), NCM_U8(r, 8), NCM_U8(r, 16), NCM_U8(r, 24)::"memory");
}
__device__ __forceinline__ void landed(uint32_t* r) {
    asm volatile("" : NCM_U8(r, 0), NCM_U8(r, 8), NCM_U8(r, 16), NCM_U8(r, 24)::"memory");
}
// 32 columns of this warp's 32 lanes (one row per lane).
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : NCM_W8(r, 0), NCM_W8(r, 8), NCM_W8(r, 16), NCM_W8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::NCM_R8(r, 0), NCM_R8(r, 8), NCM_R8(r, 16), NCM_R8(r, 24), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::NCM_R8(r, 0), NCM_R8(r, 8), "r"(addr) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 in one 64-bit register, for the packed f32 instructions.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of two values at or below a few hundred, on the FMA pipe: x = n + f with f in [-1/2, 1/2]
// by adding and taking off 1.5 * 2^23, a minimax polynomial of 2^f (Remez exchange; relative
// error 7.5e-5 of degree 3, 2.6e-6 of degree 4, against roundings of 2^-9 and 2^-12 that
// follow), n added to the exponent.  Below 2^-126 it gives 2^-126.
template <bool BF16> __device__ __forceinline__ void ex2_poly(uint64_t x2, float& lo, float& hi) {
    float a, b;
    apart(x2, a, b);
    x2 = two(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const uint64_t t = add2(x2, two(12582912.0f, 12582912.0f));
    const uint64_t f = fma2(add2(t, two(-12582912.0f, -12582912.0f)), two(-1.0f, -1.0f), x2);
    uint64_t y;
    if (BF16) {
        y = two(0x1.c3f760p-5f, 0x1.c3f760p-5f);
        y = fma2(y, f, two(0x1.f0de1ap-3f, 0x1.f0de1ap-3f));
        y = fma2(y, f, two(0x1.62f31ap-1f, 0x1.62f31ap-1f));
        y = fma2(y, f, two(0x1.fff692p-1f, 0x1.fff692p-1f));
    } else {
        y = two(0x1.3997d6p-7f, 0x1.3997d6p-7f);
        y = fma2(y, f, two(0x1.ca1440p-5f, 0x1.ca1440p-5f));
        y = fma2(y, f, two(0x1.ec06dap-3f, 0x1.ec06dap-3f));
        y = fma2(y, f, two(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
        y = fma2(y, f, two(0x1.fffffep-1f, 0x1.fffffep-1f));
    }
    float n0, n1;
    apart(t, n0, n1);
    apart(y, lo, hi);
    lo = __uint_as_float(__float_as_uint(lo) + (__float_as_uint(n0) << 23));
    hi = __uint_as_float(__float_as_uint(hi) + (__float_as_uint(n1) << 23));
}
template <bool BF16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16> __device__ __forceinline__ float widen(uint16_t h) {
    return BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}
// Whether one of the 16-bit floats in w is infinite or NaN: its exponent's ones carry into bit 15.
template <bool BF16> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return BF16 ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// What every role knows of an item.
struct Item {
    int b, head;              // sequence, key-value head
    int q0, nq, k0, nk;       // first row and rows of the sequence in q and in k
    int t0;                   // first token of tile 0 within the sequence
    int shift;                // causal: token t sees keys up to t + shift
    int n0, n1;               // units of 64 keys of each query tile
    __device__ __forceinline__ int n(int x) const { return x ? n1 : n0; }
    __device__ __forceinline__ int tiles() const { return (max(n0, n1) + 1) / 2; }
    int seen;                 // keys that every row sees: what lies below is not cut by the mask
};
__device__ __forceinline__ Item item_at(const PromptParams& p, const int* prefix, int index) {
    const int *cu_q = prefix + p.batch + 1, *cu_k = cu_q + p.batch + 1;
    Item t;
    const int block = prefix[p.batch] - 1 - index / p.kv_heads;   // of a causal sequence the blocks that see most keys come first
    t.head = index % p.kv_heads;
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= block) lo = mid; else hi = mid;
    }
    t.b = lo;
    const int2 q = make_int2(cu_q[lo], cu_q[lo + 1]), k = make_int2(cu_k[lo], cu_k[lo + 1]);
    t.q0 = q.x; t.nq = q.y - q.x;
    t.k0 = min(max(k.x, 0), p.total_k); t.nk = min(max(k.y, t.k0), p.total_k) - t.k0;
    t.t0 = (block - prefix[lo]) * 2 * p.tokens;
    t.shift = t.nk - t.nq;
    int least = t.nk;                                             // keys that every row sees
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int first = t.t0 + x * p.tokens, last = min(first + p.tokens, t.nq) - 1;
        int end = 0;
        if (first <= last) {
            end = p.causal ? min(t.nk, last + t.shift + 1) : t.nk;
            if (p.causal) least = min(least, first + t.shift + 1);
        }
        (x ? t.n1 : t.n0) = end > 0 ? (end + kUnitKeys - 1) / kUnitKeys : 0;
    }
    t.seen = max(least, 0);
    // the same in all lanes: said in a form that the compiler knows, for uniform registers
    t.n0 = __shfl_sync(NCM_FULL, t.n0, 0);
    t.n1 = __shfl_sync(NCM_FULL, t.n1, 0);
    t.seen = __shfl_sync(NCM_FULL, t.seen, 0);
    return t;
}
// Items are CTAs of the grid.  A CTA that runs takes the next one that has not been launched
// instead of ending (cluster launch control): work is dealt out as it is finished, which no
// fixed deal matches when sequences differ (12 prompts of 17 to 2048 tokens: 110 -> 104 us),
// and what is set up once stays.  The TMA warp asks; all warps read the answer.
__device__ __forceinline__ void ask_next(uint4* answer, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int read_next(const uint4* answer) {   // -1: there are no more
    uint32_t yes, x;
    asm volatile(
        "{ .reg .b128 a; .reg .pred p; ld.shared.b128 a, [%2];"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a; selp.u32 %0, 1, 0, p; mov.u32 %1, 0;"
        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a; }"
        : "=r"(yes), "=r"(x) : "r"(smem_u32(answer)) : "memory");
    return yes ? (int)x : -1;
}

template <bool BF16, int HD>
struct Layout {
    static constexpr int kTile = kRows * HD * 2;            // bytes of a tile of Q, K or V
    static constexpr int kStages = HD == 128 ? 4 : 8;
    static constexpr int kRing = 2 * kTile;
    static constexpr int kBars = kRing + kStages * kTile;   // barriers, then a few words, then prefix
    static constexpr int kWords = kBars + 8 * (3 * kStages + 16);   // 16-byte aligned: NST is even
    static constexpr int kNext = kWords + 4 * 32;           // [2] answers of 16 bytes
    static constexpr int kStore = (kNext + 32 + 127) / 128 * 128;   // 2 KB per softmax warp: 32 rows of 32 values
    static constexpr int kPrefix = kStore + 8 * 2048;       // running sums of blocks, cu_q, cu_k: batch + 1 each
};

template <bool BF16, int HD>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attn_kernel(const __grid_constant__ PromptParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = Layout<BF16, HD>;
    constexpr int NST = L::kStages, SLABS = HD / 64, SLAB = kRows * 128;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t *empty = full + NST, *edge = empty + NST, *q_full = edge + NST, *q_empty = q_full + 1, *s_ready = q_empty + 1,
             *p_ready = s_ready + 2, *pv_done = p_ready + 4, *o_ready = pv_done + 2,   // [x], [2 x + h], [x], [x]
             *n_full = o_ready + 2, *n_empty = n_full + 2;
    // [0] TMEM address, [8..16) items with odd V, [16..28) sums
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::kWords);
    int* prefix = reinterpret_cast<int*>(smem + L::kPrefix);
    const int tid = threadIdx.x, warp = __shfl_sync(NCM_FULL, tid >> 5, 0), lane = tid & 31;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity, kPromptWaitNs)) {
            ok = false;
            set_dev_error(p.err, NCM_DEVERR_MBAR_TIMEOUT);
        }
        return ok;
    };
    // The same for a whole warp, which goes on together: the TMEM instructions want all lanes.
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        ok = __all_sync(NCM_FULL, wait(bar, parity));
        return ok;
    };

    // ---- the running sum of blocks of 2 tiles over the sequences
    if (tid < 8) words[8 + tid] = 0;
    {
        const int per = (p.batch + kPromptThreads - 1) / kPromptThreads, b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
        int* cu_q = prefix + p.batch + 1;
        auto blocks_of = [&](int rows) { return (rows + 2 * p.tokens - 1) / (2 * p.tokens); };
        int sum = 0, run;
        bool falls = false;   // starts in q out of order or range
        for (int b = b0; b < b1; ++b) {
            const int q0 = __ldg(p.cu_q + b), q1 = __ldg(p.cu_q + b + 1), k0 = __ldg(p.cu_k + b), k1 = __ldg(p.cu_k + b + 1);
            const bool bad_q = q0 < 0 || q1 < q0 || q1 > p.total_q;
            if (blockIdx.x == 0 && (bad_q || k0 < 0 || k1 < k0 || k1 > p.total_k)) set_dev_error(p.err, NCM_DEVERR_BAD_ARG);
            falls |= bad_q;
            prefix[b + 1] = bad_q ? 0 : blocks_of(q1 - q0);
            sum += prefix[b + 1];
        }
        for (int b = tid; b <= p.batch; b += kPromptThreads) {
            cu_q[b] = __ldg(p.cu_q + b);
            prefix[2 * (p.batch + 1) + b] = __ldg(p.cu_k + b);
        }
        for (int b = tid; b < p.before; b += kPromptThreads) falls |= __ldg(p.cu_q + b - p.before) > __ldg(p.cu_q);
        while (true) {
            run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(NCM_FULL, run, o);
                if (lane >= o) run += v;
            }
            if (lane == 31) words[16 + warp] = run;
            if (!__syncthreads_or(falls)) break;
            // Each start counts as the largest up to it, within the range: no row has two sequences, and there
            // are no more blocks than the grid was made for.
            if (warp == 0) {
                int top = 0;
                for (int b = lane; b < p.before; b += 32) top = max(top, __ldg(p.cu_q + b - p.before));
                top = __reduce_max_sync(NCM_FULL, top);
                for (int at = 0; at <= p.batch; at += 32) {
                    int v = at + lane <= p.batch ? max(top, cu_q[at + lane]) : top;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int w = __shfl_up_sync(NCM_FULL, v, o);
                        if (lane >= o) v = max(v, w);
                    }
                    if (at + lane <= p.batch) cu_q[at + lane] = min(v, p.total_q);
                    top = __shfl_sync(NCM_FULL, v, 31);
                }
            }
            __syncthreads();
            sum = 0;
            for (int b = b0; b < b1; ++b) {
                prefix[b + 1] = blocks_of(cu_q[b + 1] - cu_q[b]);
                sum += prefix[b + 1];
            }
            falls = false;
        }
        run -= sum;
        for (int w = 0; w < warp; ++w) run += words[16 + w];
        if (tid == 0) prefix[0] = 0;
        for (int b = b0; b < b1; ++b) { run += prefix[b + 1]; prefix[b + 1] = run; }
        __syncthreads();
    }
    const int items = __shfl_sync(NCM_FULL, prefix[p.batch] * p.kv_heads, 0);
    if ((int)blockIdx.x >= items) return;   // the grid is as large as the items could be many
    // ---- barriers, TMEM
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(words)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < NST; ++i) { mbar_init(full + i, 2); mbar_init(empty + i, 1); mbar_init(edge + i, 1); }
        mbar_init(q_full, 1); mbar_init(q_empty, 1);
        for (int i = 0; i < 4; ++i) mbar_init(p_ready + i, 4);
        for (int x = 0; x < 2; ++x) {
            mbar_init(s_ready + x, 1); mbar_init(pv_done + x, 1); mbar_init(o_ready + x, 1);
            mbar_init(n_full + x, 1); mbar_init(n_empty + x, kPromptThreads / 32);
        }
        fence_mbar_init();
    }
    fence_before();
    __syncthreads();
    fence_after();
    // Every role walks over the same items: `index`, and how many came before it.
    uint4* answers = reinterpret_cast<uint4*>(smem + L::kNext);
    int index = blockIdx.x;
    uint32_t it = 0;
    auto advance = [&]() {
        if (!wait_all(n_full + (it & 1), (it >> 1) & 1)) { index = -1; return; }
        index = __shfl_sync(NCM_FULL, read_next(answers + (it & 1)), 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // read before it is written again
        __syncwarp();
        if (lane == 0) mbar_arrive(n_empty + (it & 1));
        ++it;
    };
    const uint32_t tmem = __shfl_sync(NCM_FULL, words[0], 0);
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + L::kRing;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ---- TMA
            uint32_t slot = 0, round = 0, quse = 0;
            // A V tile at the mask's edge goes to warps 10 and 11, which pass it on: `full` takes
            // their two arrivals, or two from here.
            auto load = [&](const CUtensorMap* m, const Item& t, int j, bool at_edge) {
                if (!wait_all(empty + slot, (round & 1) ^ 1)) return;
                uint64_t* bar = (at_edge ? edge : full) + slot;
                if (elected()) {
                    if (!at_edge) mbar_arrive(bar);
                    mbar_arrive_expect_tx(bar, L::kTile);
                    for (int s = 0; s < SLABS; ++s) tma3(ring + slot * L::kTile + s * SLAB, m, bar, 64 * s, t.head, t.k0 + j * kRows);
                }
                __syncwarp();
                if (++slot == NST) { slot = 0; ++round; }
            };
            for (; ok && index >= 0; advance()) {
                if (!wait_all(n_empty + (it & 1), ((it >> 1) & 1) ^ 1)) break;
                if (elected()) ask_next(answers + (it & 1), n_full + (it & 1));
                __syncwarp();
                if (index >= items) continue;
                const Item t = item_at(p, prefix, index);
                const int n = t.tiles();
                if (n == 0) continue;
                if (!wait_all(q_empty, (quse & 1) ^ 1)) break;
                ++quse;
                const int box = p.tokens * p.group * 128;
                if (elected()) {
                    mbar_arrive_expect_tx(q_full, ((t.n0 > 0) + (t.n1 > 0)) * SLABS * box);
                    for (int x = 0; x < 2; ++x)
                        if (t.n(x) > 0)
                            for (int s = 0; s < SLABS; ++s)
                                tma4(q_smem + x * L::kTile + s * SLAB, &p.qm, q_full, 64 * s, 0, t.head, t.q0 + t.t0 + x * p.tokens);
                }
                __syncwarp();
                for (int j = 0; j < n && ok; ++j) { load(&p.km, t, j, false); load(&p.vm, t, j, j >= t.seen / kRows); }
            }
            // every stage is given back before the CTA ends
            for (int i = 0; i < NST && ok; ++i) {
                wait_all(empty + slot, (round & 1) ^ 1);
                if (++slot == NST) { slot = 0; ++round; }
            }
            wait_all(q_empty, (quse & 1) ^ 1);
        } else if (warp == 9) {
            // ---- products
            constexpr uint32_t inst_s = inst_desc(BF16, kRows, false), inst_o = inst_desc(BF16, HD, true);
            uint32_t base = 0, quse = 0, phases = 0;   // bit 2 x + h: parity of p_ready's next phase
            auto slot_of = [&](uint32_t i) { return (base + i) % NST; };   // K and V tile j: places 2 j and 2 j + 1
            auto arrived = [&](uint32_t i) { return wait_all(full + slot_of(i), ((base + i) / NST) & 1); };
            auto scores = [&](int x, uint32_t i) {
                const uint32_t a = q_smem + x * L::kTile, b = ring + slot_of(i) * L::kTile;
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = (k / 4) * SLAB + (k % 4) * 32;
                        mma_ss(tmem + x * 128, smem_desc(a + off, 16), smem_desc(b + off, 16), inst_s, k > 0);
                    }
                    mma_commit(s_ready + x);
                }
                __syncwarp();
            };
            auto give_back = [&](uint64_t* bar) {
                if (elected()) mma_commit(bar);
                __syncwarp();
            };
            for (; ok && index >= 0; advance()) {
                if (index >= items) continue;
                const Item t = item_at(p, prefix, index);
                const int n = t.tiles();
                if (n == 0) continue;
                if (!wait_all(q_full, quse & 1)) break;
                ++quse;
                if (!arrived(0)) break;
                fence_after();
                if (t.n0 > 0) scores(0, 0);
                if (t.n1 > 0) scores(1, 0);
                give_back(empty + slot_of(0));
                if (n == 1) give_back(q_empty);
                // V of tile j and K of tile j + 1 are waited for a step ahead, while the products of
                // query tile 0 run: the ring holds both beside the two in use.
                static_assert(NST >= 4, "the ring holds two tiles of K and of V");
                if (!arrived(1) || (n > 1 && !arrived(2))) break;
                for (int j = 0; j < n && ok; ++j) {
                    const uint32_t v = ring + slot_of(2 * j + 1) * L::kTile;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int u = 2 * j + h;
                            if (u >= t.n(x) || !wait_all(p_ready + 2 * x + h, (phases >> (2 * x + h)) & 1)) continue;
                            phases ^= 1u << (2 * x + h);
                            fence_after();
                            if (elected()) {
#pragma unroll
                                for (int k = 0; k < kUnitKeys / 16; ++k)
                                    mma_ts(tmem + 256 + x * 128, tmem + x * 128 + h * 64 + 8 * k, smem_desc(v + (4 * h + k) * 2048, SLAB), inst_o,
                                           u > 0 || k > 0);
                                mma_commit(pv_done + x);
                                if (u + 1 == t.n(x)) mma_commit(o_ready + x);
                            }
                            __syncwarp();
                            if (h == 1 && u + 1 < t.n(x)) scores(x, 2 * j + 2);
                        }
                        if (x == 0) {
                            if (j + 1 < n) arrived(2 * j + 3);
                            if (j + 2 < n) arrived(2 * j + 4);
                        }
                    }
                    if (elected()) {
                        mma_commit(empty + slot_of(2 * j + 1));
                        if (j + 1 < n) mma_commit(empty + slot_of(2 * j + 2));
                        if (j + 2 == n) mma_commit(q_empty);
                    }
                    __syncwarp();
                }
                base += 2 * n;
            }
        } else if (warp >= 10) {
            // ---- V tiles at the mask's edge
            uint32_t base = 0, phases = 0;   // bit s: parity of edge[s]'s next phase
            for (; ok && index >= 0; advance()) {
                if (index >= items) continue;
                const Item t = item_at(p, prefix, index);
                const int n = t.tiles();
                for (int j = t.seen / kRows; j < n && ok; ++j) {
                    const uint32_t s = (base + 2 * j + 1) % NST;
                    if (!wait_all(edge + s, (phases >> s) & 1)) break;
                    phases ^= 1u << s;
                    const int from = max(t.seen - j * kRows, 0);   // rows before it are seen by all
#pragma unroll 1
                    for (int slab = 0; slab < SLABS; ++slab) {
                        uint4* tile = reinterpret_cast<uint4*>(smem + L::kRing + s * L::kTile + slab * SLAB);
                        uint32_t odd = 0;
#pragma unroll 8
                        for (int e = from * 8 + (warp - 10) * 32 + lane; e < kRows * 8; e += 64) {
                            const uint4 w = tile[e];
                            odd |= not_finite<BF16>(w.x) | not_finite<BF16>(w.y) | not_finite<BF16>(w.z) | not_finite<BF16>(w.w);
                        }
                        if (!__any_sync(NCM_FULL, odd)) continue;
                        for (int e = from * 8 + (warp - 10) * 32 + lane; e < kRows * 8; e += 64) {
                            uint32_t* w = reinterpret_cast<uint32_t*>(tile + e);
                            for (int c = 0; c < 4; ++c) {
                                const uint32_t bits = not_finite<BF16>(w[c]);
                                if (bits & 0x8000u) w[c] &= 0xffff0000u;
                                if (bits & 0x80000000u) w[c] &= 0x0000ffffu;
                            }
                        }
                        if (lane == 0) words[8 + (it & 7)] = it + 1;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + s);
                }
                base += 2 * n;
            }
        }
    } else {
        // ---- softmax, one row per thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // p and its sum times 2^7 in f16: 2^15 at most then, and what is below 2^-14 of the largest, where
        // f16's steps no longer shrink, is held 2^7 times finer.
        constexpr float kLift = BF16 ? 0.0f : 7.0f;
        const int x = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // 32 lanes per warp, in bits 16 and up
        const uint32_t s_at = tmem + x * 128 + lanes, o_at = tmem + 256 + x * 128 + lanes;
        const int token = row / p.group, member = row % p.group;
        uint32_t phases = 0, used = 0, handed = 0;   // of s_ready, of o_ready; units given to the products
        for (; ok && index >= 0; advance()) {
            if (index >= items) continue;
            const Item t = item_at(p, prefix, index);
            const int at = t.t0 + x * p.tokens + token;                 // token within the sequence
            const bool mine = token < p.tokens && at < t.nq;
            const int limit = !mine ? -1 : p.causal ? min(at + t.shift, t.nk - 1) : t.nk - 1;   // last key seen
            const int units = t.n(x);
            float top = -INFINITY, sum = 0.0f;                          // running maximum (times scale, log2), sum of p
            for (int u = 0; u < units; ++u) {
                const int h = u & 1;
                const uint32_t s_unit = s_at + 64 * h;
                if (h == 0) {
                    if (!wait_all(s_ready + x, phases & 1)) break;
                    ++phases;
                    fence_after();
                }
                uint32_t s[64];
                tmem_ld32(s, s_unit);
                tmem_ld32(s + 32, s_unit + 32);
                wait_ld(s);
                landed(s + 32);
                const bool masked = (u + 1) * kUnitKeys > t.seen;
                if (masked) {
                    const int left = limit - u * kUnitKeys;             // columns up to this one are seen
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (c > left) s[c] = 0xff800000u;
                }
                float m[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) m[c] = max3(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1]), -INFINITY);
#pragma unroll
                for (int c = 8; c < 64; c += 2) m[(c >> 1) & 3] = max3(m[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                const float now = max3(max3(m[0], m[1], m[2]), m[3], -INFINITY) * p.scale_log2;
                // The maximum is moved only where a score has passed it by more than 2^8, so that
                // the sums in TMEM are rarely rescaled; p stays below 2^8.  A score that is NaN or
                // infinite makes the row NaN.  Rows of no token (behind the sequence, or where the group
                // does not divide 128, whose queries are whatever lay there) have no say.
                const bool over = mine && !(now <= top + 8.0f);
                if (__any_sync(NCM_FULL, over)) {
                    const float a = !over ? 1.0f : now < INFINITY ? ex2(top - now) : NAN;
                    if (over && now < INFINITY) top = now;
                    sum *= a;
                    if (!(now < INFINITY)) sum = NAN;
                    // O is at rest once the last unit's products are complete (those before it are: S is here)
                    if (u > 0) {
                        if (!wait_all(pv_done + x, (handed - 1) & 1)) break;
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(o, o_at + c);
                            wait_ld(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                            tmem_st32(o_at + c, o);
                        }
                    }
                }
                const float shift = top == -INFINITY ? 0.0f : kLift - top;
                const uint64_t scale2 = two(p.scale_log2, p.scale_log2), shift2 = two(shift, shift);
                uint64_t l0 = 0, l1 = 0;
                // p of 32 columns; with a mask by ex2 alone, which gives 0 where it hides
                auto part = [&](int c, bool plain) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint64_t v = fma2(two(__uint_as_float(s[32 * c + 2 * i]), __uint_as_float(s[32 * c + 2 * i + 1])), scale2, shift2);
                        float a, b;
                        if (!plain && (i & 7) < kPolyOf8) {
                            ex2_poly<BF16>(v, a, b);
                        } else {
                            apart(v, a, b);
                            a = ex2(a); b = ex2(b);
                        }
                        (i & 1 ? l1 : l0) = add2(i & 1 ? l1 : l0, two(a, b));
                        w[i] = pack<BF16>(a, b);
                    }
                    tmem_st16(s_unit + 16 * c, w);
                };
                if (masked) { part(0, true); part(1, true); } else { part(0, false); part(1, false); }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + 2 * x + h);
                ++handed;
                float la, lb, lc, ld;
                apart(l0, la, lb);
                apart(l1, lc, ld);
                sum += (la + lb) + (lc + ld);
            }
            if (units > 0) {
                if (!wait_all(o_ready + x, used & 1)) break;
                ++used;
                fence_after();
            }
            const bool odd = words[8 + (it & 7)] == it + 1;
            // A row without keys, or with none that scores above -infinity: zeros (what ex2_poly made of
            // such scores is in its sum).  The sum is at least one otherwise, or NaN.
            const float inv = top == -INFINITY && sum == sum ? 0.0f : 1.0f / sum;
            // Rows leave through shared memory, 32 columns at a time: four lanes then write 64
            // bytes of a row, where one lane per row would touch 32 lines with every store.
            uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)(t.q0 + at) * p.out_stride + (int64_t)(t.head * p.group + member) * HD;
            uint8_t* stage = smem + L::kStore + warp * 2048;
            const uint32_t rows = __ballot_sync(NCM_FULL, mine);
            uint16_t* dst[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                dst[i] = reinterpret_cast<uint16_t*>(__shfl_sync(NCM_FULL, reinterpret_cast<unsigned long long>(out), 8 * i + (lane >> 2))) + 8 * (lane & 3);
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (units > 0) {
                    tmem_ld32(o, o_at + c);
                    wait_ld(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (odd && mine) {
                    // infinities and NaN that were taken out of V, for the rows that see their keys
                    const uint16_t* v = static_cast<const uint16_t*>(p.v) + (int64_t)t.k0 * p.v_stride + t.head * HD + c;
                    for (int key = t.seen; key <= limit; ++key)
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const uint16_t h = __ldg(v + key * p.v_stride + i);
                            if (not_finite<BF16>(h)) o[i] = __float_as_uint(__uint_as_float(o[i]) + widen<BF16>(h));
                        }
                }
                // (zero times a value that is not finite is not zero)
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = inv == 0.0f ? 0u : o[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = pack<BF16>(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 8 * i + (lane >> 2);
                    const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
                    if (rows >> r & 1) *reinterpret_cast<uint4*>(dst[i] + c) = w;
                }
            }
            fence_before();   // O is read before the next item's products overwrite it
            __syncwarp();
        }
    }
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------------ host side
bool aligned16(const void* p) { return (((uintptr_t)p) & 15) == 0; }
bool aligned4(const void* p) { return (((uintptr_t)p) & 3) == 0; }
int bad(const char* what) { return set_error(NCM_EINVAL, what); }

bool kv_map(CUtensorMap* m, const void* base, int hd, int kv_heads, int tokens, int64_t stride) {
    const cuuint64_t dim[3] = {(cuuint64_t)hd, (cuuint64_t)kv_heads, (cuuint64_t)tokens};
    const cuuint64_t step[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, 1, kRows}, one[3] = {1, 1, 1};
    return encode_tiled_fn()(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dim, step, box, one,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool q_map(CUtensorMap* m, const void* base, int hd, int group, int kv_heads, int tokens, int64_t stride, int box_tokens) {
    const cuuint64_t dim[4] = {(cuuint64_t)hd, (cuuint64_t)group, (cuuint64_t)kv_heads, (cuuint64_t)tokens};
    const cuuint64_t step[3] = {(cuuint64_t)hd * 2, (cuuint64_t)group * hd * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)box_tokens}, one[4] = {1, 1, 1, 1};
    return encode_tiled_fn()(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dim, step, box, one,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, int HD>
int prompt_run(const PromptParams& p, int grid, cudaStream_t s) {
    const int bytes = Layout<BF16, HD>::kPrefix + 12 * (p.batch + 1);
    auto fn = prompt_attn_kernel<BF16, HD>;
    if (int r = set_smem_limit((const void*)fn, kPromptSmem)) return r;
    fn<<<grid, kPromptThreads, bytes, s>>>(p);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" ncm_status ncm_prompt_attention(void* out, int64_t out_stride, const void* q, int64_t q_stride, const void* k,
                                           int64_t k_stride, const void* v, int64_t v_stride, int type, int total_q,
                                           int total_k, int batch, int heads, int kv_heads, int head_dim, const int* cu_q,
                                           const int* cu_k, int causal, float scale, int* err, void* stream) {
    if (type != NCM_TYPE_F16 && type != NCM_TYPE_BF16) return bad("type must be F16 or BF16");
    if (head_dim != 64 && head_dim != 128) return bad("head_dim must be 64 or 128");
    if (heads < 1 || kv_heads < 1 || kv_heads > 1024 || heads % kv_heads || heads / kv_heads > 128)
        return bad("heads must be a multiple of kv_heads, 128 to one at most");
    if (total_q < 0 || total_k < 0 || batch < 0 || total_q > (1 << 30) || total_k > (1 << 30)) return bad("bad prompt sizes");
    if (!(scale >= 0.0f) || scale > 2.0e38f) return bad("scale must be positive, below 2e38 (0: 1 / sqrt(head_dim))");
    if (total_q == 0 || batch == 0) return NCM_OK;
    if (!out || !q || !cu_q || !cu_k || (total_k && (!k || !v))) return bad("null pointer");
    const int64_t wide_q = (int64_t)heads * head_dim, wide_k = (int64_t)kv_heads * head_dim;
    int64_t* stride[4] = {&out_stride, &q_stride, &k_stride, &v_stride};
    const void* at[4] = {out, q, k, v};
    for (int i = 0; i < 4; ++i) {
        const int64_t wide = i < 2 ? wide_q : wide_k;
        if (!*stride[i]) *stride[i] = wide;
        if (*stride[i] < wide || *stride[i] % 8 || *stride[i] > ((int64_t)1 << 38) || !aligned16(at[i]))
            return bad("rows must be 16-byte aligned and at least a token apart");
    }
    if (!aligned4(cu_q) || !aligned4(cu_k) || !aligned4(err)) return bad("int arrays must be 4-byte aligned");
    if (total_k == 0) { k = q; v = q; k_stride = q_stride; v_stride = q_stride; }   // never read: no row sees a key
    const void* check[] = {out, q, k, v, cu_q, cu_k, err};
    if (const char* e = device_pointers_error(check, sizeof check / sizeof *check)) return bad(e);
    if (!encode_tiled_fn()) return set_error(NCM_ECUDA, "cuTensorMapEncodeTiled not available");
    PromptParams p;
    memset(&p, 0, sizeof p);
    p.group = heads / kv_heads;
    p.tokens = kRows / p.group;
    if (!q_map(&p.qm, q, head_dim, p.group, kv_heads, total_q, q_stride, p.tokens) ||
        !kv_map(&p.km, k, head_dim, kv_heads, std::max(total_k, 1), k_stride) ||
        !kv_map(&p.vm, v, head_dim, kv_heads, std::max(total_k, 1), v_stride))
        return set_error(NCM_ECUDA, "cuTensorMapEncodeTiled failed for the prompt");
    p.out = out; p.v = v; p.out_stride = out_stride; p.v_stride = v_stride;
    p.kv_heads = kv_heads; p.total_q = total_q; p.total_k = total_k; p.causal = causal != 0;
    p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f;
    p.err = err;
    cudaStream_t s = (cudaStream_t)stream;
    for (int b = 0; b < batch; b += kPromptBatch) {
        p.batch = std::min(kPromptBatch, batch - b);
        p.before = b;
        p.cu_q = cu_q + b; p.cu_k = cu_k + b;
        const int64_t most = ((int64_t)total_q / (2 * p.tokens) + p.batch) * kv_heads;
        if (most > (1 << 30)) return set_error(NCM_EUNSUPPORTED, "too many blocks of queries");
        const int grid = (int)most;
        int r;
        if (type == NCM_TYPE_BF16) r = head_dim == 64 ? prompt_run<true, 64>(p, grid, s) : prompt_run<true, 128>(p, grid, s);
        else r = head_dim == 64 ? prompt_run<false, 64>(p, grid, s) : prompt_run<false, 128>(p, grid, s);
        if (r) return set_error(NCM_ECUDA, cudaGetErrorString((cudaError_t)r));
    }
    return NCM_OK;
}
