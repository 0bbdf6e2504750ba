// Low-rank adapters of many requests beside a projection that they share, and their gradients (contract:
// include/qwen4_moe_b200.h; no counterpart in the reference).
//
//   h_t = scale_s A_s x_t       y_t  = base_t + B_s h_t
//   g_t = scale_s B_s^T dy_t    dx_t = base_t + A_s^T g_t     dA_s = sum_t g_t x_t^T     dB_s = sum_t dy_t h_t^T
//
// Three products, each a grouped GEMM whose groups are the tokens of one slot (adapter_lists_kernel sorts them):
//   shrink  [128 tokens] x [width] -> [128 tokens, rank]      A x and B^T dy: contracts a wide axis, cut over a cluster's CTAs
//   expand  [rank] -> [128 tokens, 128 columns]               B h and A^T g: contracts the rank, adds base, streams rows in and out
//   outer   [tokens of a slot] -> [128 columns, rank]         dA and dB: contracts the tokens, cut over a cluster's CTAs
// All on tcgen05 with FP32 accumulators in TMEM.  An FP32 value enters as three bf16 values, its 24 bits cut in three (each
// a truncation, so their sum is the value exactly); F16 adapters as two, BF16 ones as they are.  Products of planes i and j are formed for
// i + j <= 2; what is left out is below 2^-21 of a product of two FP32 values, 2^-25 on average.
//
// Operands are written to shared memory by the CTA's threads, which cut them on the way, as 8 x 16-byte core matrices without
// swizzle: [8 columns][8 rows][16 bytes], so that rows of the source can be the rows of either major-ness.  Column groups
// lie 16 bytes further apart than they are long: eight lanes that write one row's eight groups then meet in no bank.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <pthread.h>
#include <stdint.h>

#include "cuda_shim.h"

extern "C" int qw4sh_note_launch(const char *name);
extern "C" int qw4sh_allow_smem(const void *kernel, size_t smem);

namespace {

constexpr uint32_t THREADS = 256, TM = 128;                  // tokens per tile: tcgen05's M (shrink) or most N (expand)
constexpr uint32_t KC = 64;                                  // shrink: columns per step
constexpr uint32_t TC = 64;                                  // outer: tokens per step

// ---- PTX ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// The fence orders the initialisation, a store like any other, before what bulk copies and commits do to the barrier.
__device__ __forceinline__ void bar_init(uint32_t bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n fence.mbarrier_init.release.cluster;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded (about a second): whoever gives up records it, and the launch goes on to its end without that product.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, uint32_t *status) {
    if (bar_try(bar, parity)) return;
    const uint32_t start = (uint32_t)clock();
    while (!bar_try(bar, parity))
        if ((uint32_t)clock() - start > (1u << 31)) { atomicOr(status, QW4SH_ERR_STATE); return; }
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_alloc(uint32_t at, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
// sixteen accumulator columns of the thread's lane
__device__ __forceinline__ void tc_load16(uint32_t addr, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
                   "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t addr, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
                 "tcgen05.wait::st.sync.aligned;"
                 ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
                   "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
                 : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// As in balance.cu: nothing that the launch ahead wrote is read before the wait, or through a __restrict__ pointer to const.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kind::f16 with bf16 operands and FP32 accumulators
__host__ __device__ constexpr uint32_t idesc_of(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | (n >> 3 << 17) | (m >> 4 << 24);
}

// ---- operand tiles in shared memory -----------------------------------------------------------------------------------------
// ROWS x COLS bf16, a source row being a tile row: element (r, c) at c / 8 * GROUP + r * 16 + c % 8 * 2.  Where the rows are the
// operand's M or N axis the tile is K-major, where they are its K axis MN-major; LBO is the step along K and SBO the one along M
// or N, from one core matrix to the next.
template <uint32_t ROWS, uint32_t COLS, uint32_t PLANES> struct Tile {
    static constexpr uint32_t GROUP = ROWS * 16 + 16, PLANE = COLS / 8 * GROUP, BYTES = PLANES * PLANE;
    static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) { return (c >> 3) * GROUP + r * 16 + (c & 7) * 2; }
    static __device__ __forceinline__ uint64_t desc(uint32_t addr, bool mn) {
        const uint32_t along_k = mn ? 128 : GROUP, along_mn = mn ? GROUP : 128;
        return (uint64_t)(addr >> 4 & 0x3fffu) | (uint64_t)(along_k >> 4) << 16 | (uint64_t)(along_mn >> 4) << 32 | 1ull << 46;
    }
    static __host__ __device__ constexpr uint32_t k16(bool mn) { return mn ? 256 : 2 * GROUP; }          // bytes to the next sixteen of K
};

// The result of shrink, rows of RP values cut in three planes, lies in memory as it is read: core matrices of eight rows x eight values, the
// matrices of eight rows behind one another.  A slot's rows start at a multiple of sixteen and end at one, zeros behind the
// last, so a run of rows is one copy to a plane, and an operand with either axis as K.
template <uint32_t ROWS, uint32_t RP> struct Rank {
    static constexpr uint32_t PLANE = ROWS * RP * 2, BYTES = 3 * PLANE;
    static __device__ __forceinline__ uint64_t desc(uint32_t addr, bool mn) {
        const uint32_t along_k = mn ? RP * 16 : 128, along_mn = mn ? 128 : RP * 16;
        return (uint64_t)(addr >> 4 & 0x3fffu) | (uint64_t)(along_k >> 4) << 16 | (uint64_t)(along_mn >> 4) << 32 | 1ull << 46;
    }
    static __host__ __device__ constexpr uint32_t k16(bool mn) { return mn ? 2 * RP * 16 : 256; }
};
// Sixteen-row runs of its three planes to shared memory, by one thread; `bar` learns of their arrival.
template <uint32_t ROWS, uint32_t RP>
__device__ __forceinline__ void copy_rank(uint32_t dst, const __nv_bfloat16 *planes, uint64_t plane, uint32_t first, uint32_t rows16, uint32_t bar) {
    const uint32_t bytes = rows16 * RP * 2;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(3 * bytes) : "memory");
#pragma unroll
    for (uint32_t p = 0; p < 3; p++)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(dst + p * Rank<ROWS, RP>::PLANE), "l"(planes + p * plane + (uint64_t)first * RP), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void put8(uint32_t addr, uint32_t a, uint32_t b) { asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory"); }

// The upper sixteen bits of two values, and what they leave of them.
__device__ __forceinline__ uint32_t cut2(float &a, float &b) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    a -= __uint_as_float(x & 0xffff0000u);
    b -= __uint_as_float(y & 0xffff0000u);
    return __byte_perm(x, y, 0x7632);
}
// Four values into PLANES planes `step` bytes apart.
template <int PLANES> __device__ __forceinline__ void put_cut(uint32_t addr, uint32_t step, float4 v) {
#pragma unroll
    for (int p = 0; p < PLANES; p++) {
        const uint32_t a = cut2(v.x, v.y), b = cut2(v.z, v.w);
        put8(addr + p * step, a, b);
    }
}

// Four neighbouring values of a row as they are in memory.  Loads have no condition (a branch around one makes its result wait at the
// join, and the loads of a step then follow one another): places that do not exist are read at the last one that does, and zeroed
// (`keep`) when they are cut.
template <typename W> struct Four;
template <> struct Four<float> {
    static constexpr int PLANES = 3;
    float4 v;
    __device__ __forceinline__ void load4(const float *p) { v = *(const float4 *)p; }
    __device__ __forceinline__ void load1(const float *row, uint32_t c, uint32_t last) {
        v = make_float4(row[min(c, last)], row[min(c + 1, last)], row[min(c + 2, last)], row[min(c + 3, last)]);
    }
    __device__ __forceinline__ void keep(int valid) {
        if (valid < 1) v.x = 0;
        if (valid < 2) v.y = 0;
        if (valid < 3) v.z = 0;
        if (valid < 4) v.w = 0;
    }
    __device__ __forceinline__ void take(uint32_t addr) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    }
    __device__ __forceinline__ void put(uint32_t addr, uint32_t step) const { put_cut<3>(addr, step, v); }
};
template <typename H> struct Four16 {
    uint2 v;
    __device__ __forceinline__ void take(uint32_t addr) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory"); }
    __device__ __forceinline__ void load4(const H *p) { v = *(const uint2 *)p; }
    __device__ __forceinline__ void load1(const H *q, uint32_t c, uint32_t last) {
        const uint16_t *row = (const uint16_t *)q;
        v = make_uint2(row[min(c, last)] | (uint32_t)row[min(c + 1, last)] << 16, row[min(c + 2, last)] | (uint32_t)row[min(c + 3, last)] << 16);
    }
    __device__ __forceinline__ void keep(int valid) {
        v.x &= valid < 1 ? 0u : valid < 2 ? 0xffffu : 0xffffffffu;
        v.y &= valid < 3 ? 0u : valid < 4 ? 0xffffu : 0xffffffffu;
    }
};
template <> struct Four<__nv_bfloat16> : Four16<__nv_bfloat16> {
    static constexpr int PLANES = 1;
    __device__ __forceinline__ void put(uint32_t addr, uint32_t) const { put8(addr, v.x, v.y); }
};
template <> struct Four<__half> : Four16<__half> {
    static constexpr int PLANES = 2;                         // eleven bits
    __device__ __forceinline__ void put(uint32_t addr, uint32_t step) const {
        const float2 a = __half22float2(*(const __half2 *)&v.x), b = __half22float2(*(const __half2 *)&v.y);
        put_cut<2>(addr, step, make_float4(a.x, a.y, b.x, b.y));
    }
};
// Copies to shared memory that the thread itself waits for: the first `there` of BYTES bytes, zeros behind them.
template <uint32_t BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void *src, uint32_t there) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(there), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// How many of four places from c on lie before `end`.
__device__ __forceinline__ int places(uint32_t c, uint32_t end) { return c < end ? (int)min(4u, end - c) : 0; }

// The adapters of all slots as [rank, width] matrices: wide: rows of the rank axis (A), else rows of the wide axis (B).  `fours`: rows
// start on a boundary of four values and end on one.
template <typename W> struct Mat { const W *p; uint64_t slot; uint32_t rank, width; bool wide, fours; };

// A run of LEN columns of a slot's matrix (rank padded to RP) on its way into the operand tiles Wide (RP x LEN) or Tall (LEN x RP).
// Where runs of four lie on their boundaries a thread keeps the places it reads in such runs (and `copy` moves them on from run to run).
template <typename W, uint32_t RP, uint32_t LEN> struct MatRun {
    static constexpr uint32_t ALL = RP * LEN / 4, UNITS = (ALL + THREADS - 1) / THREADS, PLANES = Four<W>::PLANES;
    using Wide = Tile<RP, LEN, PLANES>;
    using Tall = Tile<LEN, RP, PLANES>;
    static constexpr uint32_t BYTES = Wide::BYTES > Tall::BYTES ? Wide::BYTES : Tall::BYTES;
    Four<W> v[UNITS];
    uint32_t at[UNITS];
    static_assert(ALL >= THREADS, "no thread without a run of four");
    static __device__ __forceinline__ uint32_t wide_r(uint32_t i) { return (threadIdx.x + i * THREADS) / (LEN / 4); }
    static __device__ __forceinline__ uint32_t wide_c(uint32_t i) { return (threadIdx.x + i * THREADS) % (LEN / 4) * 4; }
    static __device__ __forceinline__ uint32_t tall_c(uint32_t i) { return (threadIdx.x + i * THREADS) / (RP / 4); }
    static __device__ __forceinline__ uint32_t tall_r(uint32_t i) { return (threadIdx.x + i * THREADS) % (RP / 4) * 4; }
    __device__ __forceinline__ void begin(const Mat<W> &m, uint32_t c0) {
#pragma unroll
        for (uint32_t i = 0; i < UNITS; i++)
            at[i] = m.wide ? (min(wide_r(i), m.rank - 1) * m.width + c0 + wide_c(i)) / 4 : ((c0 + tall_c(i)) * m.rank + min(tall_r(i), (m.rank - 1) & ~3u)) / 4;
    }
    // columns c0 .. c0 + LEN of w, which end at `end`; where m.fours, the ones that `begin` was told
    __device__ __forceinline__ void load(const Mat<W> &m, const W *w, uint32_t c0, uint32_t end) {
        if (m.fours && c0 + LEN <= end) {
#pragma unroll
            for (uint32_t i = 0; i < UNITS; i++) v[i].load4(w + (uint64_t)at[i] * 4);
        } else if (m.wide) {
#pragma unroll 1
            for (uint32_t i = 0; i < UNITS; i++) {
                Four<W> f;
                f.load1(w + (uint64_t)min(wide_r(i), m.rank - 1) * m.width, c0 + wide_c(i), end - 1);
                set(i, f);
            }
        } else {
#pragma unroll 1
            for (uint32_t i = 0; i < UNITS; i++) {
                Four<W> f;
                f.load1(w + (uint64_t)min(c0 + tall_c(i), end - 1) * m.rank, tall_r(i), m.rank - 1);
                set(i, f);
            }
        }
    }
    // the same by way of the thread's own places in shared memory, UNITS of them `stride` bytes apart; only where m.fours
    __device__ __forceinline__ void copy(const Mat<W> &m, const W *w, uint32_t c0, uint32_t end, uint32_t to, uint32_t stride) {
        const uint32_t step = m.wide ? LEN / 4 : LEN / 4 * m.rank;
#pragma unroll
        for (uint32_t i = 0; i < UNITS; i++) {
            const bool there = m.wide ? c0 + wide_c(i) < end : c0 + tall_c(i) < end;
            copy_async<4 * sizeof(W)>(to + i * stride, there ? w + (uint64_t)at[i] * 4 : w, there ? 4 * sizeof(W) : 0);
            at[i] += step;
        }
    }
    __device__ __forceinline__ void take(uint32_t from, uint32_t stride) {
#pragma unroll
        for (uint32_t i = 0; i < UNITS; i++) v[i].take(from + i * stride);
    }
    __device__ __forceinline__ void set(uint32_t i, const Four<W> &f) {
#pragma unroll
        for (uint32_t j = 0; j < UNITS; j++) if (i == j) v[j] = f;
    }
    __device__ __forceinline__ void put(const Mat<W> &m, uint32_t c0, uint32_t end, uint32_t addr) {
        if (m.rank != RP || c0 + LEN > end)
#pragma unroll
            for (uint32_t i = 0; i < UNITS; i++) {
                if (m.wide) v[i].keep(wide_r(i) < m.rank ? places(c0 + wide_c(i), end) : 0);
                else v[i].keep(c0 + tall_c(i) < end ? places(tall_r(i), m.rank) : 0);
            }
        if (m.wide)
#pragma unroll
            for (uint32_t i = 0; i < UNITS; i++) v[i].put(addr + Wide::at(wide_r(i), wide_c(i)), Wide::PLANE);
        else
#pragma unroll
            for (uint32_t i = 0; i < UNITS; i++) v[i].put(addr + Tall::at(tall_c(i), tall_r(i)), Tall::PLANE);
    }
};

// ---- lists ------------------------------------------------------------------------------------------------------------------
// Tokens sorted by slot (tokens without one last, in the group `slots`), in the order of the batch inside a slot, every slot's from a
// multiple of sixteen on; tiles of up to 128 tokens of one slot.  One CTA: every warp counts a run of tokens, then places it.
struct ATile { uint32_t slot, first, rows, pad; };

__global__ void __launch_bounds__(1024) adapter_lists_kernel(const uint32_t *ids, uint32_t T, uint32_t S, uint32_t *__restrict__ order,
                                                             uint32_t *__restrict__ offsets /* [groups][start, tokens] */, ATile *__restrict__ tiles,
                                                             uint32_t *__restrict__ n_tiles, uint32_t *status) {
    extern __shared__ uint32_t counts[];                     // [warps][S + 1], then where the groups start [S + 1]
    __shared__ uint32_t sums[2][32];
    const uint32_t G = S + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t per = ((T + 31) / 32 + 31) & ~31u, first = min(T, warp * per), end = min(T, first + per);
    uint32_t *mine = counts + warp * G, *starts = counts + 32 * G;
    grid_go();                                               // the tiles' CTAs may take their places
    grid_wait();
    constexpr uint32_t LOADS = 8;                            // in flight
    uint32_t s[LOADS], same[LOADS];
    auto fetch = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) s[i] = t0 + 32 * i + lane < end ? ids[t0 + 32 * i + lane] : 0;
    };
    auto match = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) {
            const bool there = t0 + 32 * i + lane < end;
            if (there && s[i] >= S && s[i] != QW4CU_NO_ADAPTER) atomicOr(status, QW4SH_ERR_BOUNDS);
            s[i] = there ? min(s[i], S) : 0xffffffffu;
            same[i] = t0 + 32 * i < end ? __match_any_sync(0xffffffffu, s[i]) : 0;
        }
    };
    fetch(first);
    for (uint32_t i = threadIdx.x; i < 32 * G; i += 1024) counts[i] = 0;
    match(first);
    __syncthreads();
    for (uint32_t t0 = first; t0 < end; t0 += 32 * LOADS) {
        if (t0 != first) { fetch(t0); match(t0); }
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) {
            if (s[i] <= S && __ffs(same[i]) - 1 == (int)lane) mine[s[i]] += __popc(same[i]);
            __syncwarp();
        }
    }
    __syncthreads();
    // where each warp's run of a group starts inside it: a warp per group, a lane per run
    for (uint32_t g = warp; g < G; g += 32) {
        const uint32_t c = counts[lane * G + g];
        uint32_t sum = c;
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        counts[lane * G + g] = sum - c;
        if (lane == 31) starts[g] = sum;
    }
    __syncthreads();
    // where each group and its tiles start: two groups to a thread
    uint32_t total[2], room[2];
    for (uint32_t j = 0; j < 2; j++) {
        total[j] = 2 * threadIdx.x + j < G ? starts[2 * threadIdx.x + j] : 0;
        room[j] = (total[j] + 15) & ~15u;
    }
    uint32_t r = room[0] + room[1], n = (total[0] + TM - 1) / TM + (total[1] + TM - 1) / TM;
    const uint32_t own_r = r, own_n = n;
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) { r += a; n += b; }
    }
    if (lane == 31) { sums[0][warp] = r; sums[1][warp] = n; }
    __syncthreads();
    uint32_t at = __reduce_add_sync(0xffffffffu, lane < warp ? sums[0][lane] : 0) + r - own_r;
    uint32_t tile = __reduce_add_sync(0xffffffffu, lane < warp ? sums[1][lane] : 0) + n - own_n;
    for (uint32_t j = 0; j < 2; j++) {
        const uint32_t g = 2 * threadIdx.x + j;
        if (g >= G) break;
        starts[g] = at;
        offsets[2 * g] = at;
        offsets[2 * g + 1] = total[j];
        for (uint32_t i = 0; i < total[j]; i += TM) tiles[tile++] = ATile{g, at + i, min(TM, total[j] - i), 0};
        at += room[j];
        if (g == S) *n_tiles = tile;
    }
    __syncthreads();
    if (per > 32 * LOADS) { fetch(first); match(first); }    // else they are still there
    for (uint32_t t0 = first; t0 < end; t0 += 32 * LOADS) {
        if (t0 != first) { fetch(t0); match(t0); }
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) {
            const bool there = s[i] <= S;
            const uint32_t before = there ? mine[s[i]] : 0;
            __syncwarp();
            if (there) {
                order[starts[s[i]] + before + __popc(same[i] & ((1u << lane) - 1))] = t0 + 32 * i + lane;
                if (__ffs(same[i]) - 1 == (int)lane) mine[s[i]] = before + __popc(same[i]);
            }
            __syncwarp();
        }
    }
}

// ---- accumulators ---------------------------------------------------------------------------------------------------------
// An accumulator loses up to a bit's weight at every instruction that adds to it (additions in the tensor core truncate), always towards
// zero, so what counts is how many add to the same one.  Products of the leading planes go to two accumulators in turn, and
// the corrections, 2^-8 of them and less, to one of their own (`side`), where their truncations are as much smaller; the sums meet
// in FP32 when they are read.  Every FLUSH steps they are added to a fourth set of columns, rounded to nearest, and begun anew, so
// that neither the length of the sum nor how it is cut matters.  Measured with one accumulator for everything: dA of 8192 tokens off by
// 5.9e-6 of its norm (the plain form in FP32: 0.9e-6); with one for the leading planes and no flush up to 1.8e-6.
constexpr uint32_t FLUSH = 16;
template <uint32_t RP> struct Sums {
    static constexpr uint32_t MAINS = 2, SIDE = 2 * RP, TOTAL = 3 * RP, COLS = 4 * RP;
    static constexpr uint32_t CTAS = RP <= 32 ? 3 : RP == 64 ? 2 : 1;                // to an SM, which has 512 columns
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// The MMAs of one step: every sixteen of K, every pair of planes.
// One warp walks this, and one of its threads issues.  Whatever an instruction names has to be warp-uniform for the compiler as well (read
// from shared memory it is not, out of a reduction it is): otherwise every operand is moved to a uniform register first, and an
// instruction costs 87 cycles instead of 49 (N = 64) or 65 (N = 128; the same with and without a swizzle, K- and MN-major).
template <typename TA, typename TB, int PA, int PB, bool AMN, bool BMN, uint32_t MAINS, uint32_t K16S>
__device__ __forceinline__ void step_mma(uint32_t d, uint32_t d_step, uint32_t side, uint32_t a_at, uint32_t b_at, uint32_t idesc, bool first, uint32_t leader) {
    const uint64_t a = TA::desc(a_at, AMN), b = TB::desc(b_at, BMN);
    const uint32_t more = first ? 0 : 1;
    if (!leader) return;
    bool begun = false;
#pragma unroll
    for (int order = 2; order > 0; order--)                  // the smallest first
#pragma unroll
        for (uint32_t k = 0; k < K16S; k++)
#pragma unroll
            for (int i = 0; i < PA; i++) {
                const int j = order - i;
                if (j < 0 || j >= PB) continue;
                tc_mma(side, a + ((i * TA::PLANE + k * TA::k16(AMN)) >> 4), b + ((j * TB::PLANE + k * TB::k16(BMN)) >> 4), idesc, begun ? 1 : more);
                begun = true;
            }
#pragma unroll
    for (uint32_t k = 0; k < K16S; k++)
        tc_mma(d + k % MAINS * d_step, a + (k * TA::k16(AMN) >> 4), b + (k * TB::k16(BMN) >> 4), idesc, d_step == 0 || k >= MAINS ? 1 : more);
}
// Sixteen columns of a sum that lies in the accumulators of shrink and outer: what was added up since the last flush (`mains`: leading accumulators
// that are in use), and what was before it.
template <uint32_t RP> __device__ __forceinline__ void load_sum(uint32_t addr, float (&v)[16], uint32_t mains, bool flushed) {
    float u[16];
    tc_load16(addr, v);
    tc_load16(addr + Sums<RP>::SIDE, u);
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] += u[i];
    if (mains > 1) {
        tc_load16(addr + RP, u);
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] += u[i];
    }
    if (flushed) {
        tc_load16(addr + Sums<RP>::TOTAL, u);
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] += u[i];
    }
}
// By all warps, between the products of one step and the next: the accumulators to the total.
template <uint32_t RP> __device__ __forceinline__ void flush(uint32_t tmem, bool again) {
    const uint32_t warp = threadIdx.x >> 5, lanes = tmem + ((warp & 3) << 21);
    tc_after();
    for (uint32_t c = (warp >> 2) * 16; c < RP; c += 32) {
        float v[16];
        load_sum<RP>(lanes + c, v, Sums<RP>::MAINS, again);
        tc_store16(lanes + Sums<RP>::TOTAL + c, v);
    }
    tc_before();
}

// ---- shrink -----------------------------------------------------------------------------------------------------------------
struct Lists { const uint32_t *order, *offsets; const ATile *tiles; const uint32_t *n_tiles; };

template <typename W> struct ShrinkJob {
    Mat<W> w;
    const float *x;
    uint64_t pitch;
    bool x_fours;                                            // rows on boundaries of four values, no more than 2^32 such runs
    __nv_bfloat16 *planes;                                   // [3][rows x RP]: the result, rows in the lists' order
};
template <typename W> struct ShrinkArgs {
    ShrinkJob<W> job[2];
    Lists lists;
    const float *scale;
    uint64_t plane;                                          // elements from one plane of the result to the next
    uint32_t slots;
    uint32_t *status;
};

template <typename W, uint32_t RP> struct ShrinkMap {
    using X = Tile<TM, KC, 3>;                               // rows tokens: K-major
    using Run = MatRun<W, RP, KC>;                           // Wide: K-major, Tall: MN-major
    static constexpr uint32_t XU = TM * KC / 4 / THREADS;    // runs of four values of x per thread and step
    static constexpr uint32_t W_UNIT = THREADS * 4 * sizeof(W), SLOT = XU * THREADS * 16 + Run::UNITS * W_UNIT;
    static constexpr uint32_t OPERANDS = X::BYTES + Run::BYTES;
    static constexpr uint32_t ORDER = 64, STAGE = ORDER + TM * 4, RING = STAGE + OPERANDS, END = RING + SLOT;
    static constexpr uint32_t PITCH = RP + 4;                // floats per row of the exchanged accumulators
    static constexpr uint32_t ACC_END = STAGE + TM * PITCH * 4, TOTAL = END > ACC_END ? END : ACC_END;
};

// Values come in by asynchronous copies, a step before they are cut, each thread's own into places of its own: no barrier, no register and no line
// of L1 holds them meanwhile (through registers an SM had half as many bytes under way).
// Two CTAs to an SM up to rank 64 (F32: up to 32), one beyond: shared memory, 124 KB for F32 at rank 64.
template <typename W, uint32_t RP>
__global__ void __launch_bounds__(THREADS, RP <= 64 ? 2 : 1) adapter_shrink_kernel(const __grid_constant__ ShrinkArgs<W> a) {
    namespace cg = cooperative_groups;
    using M = ShrinkMap<W, RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    const ShrinkJob<W> &job = a.job[blockIdx.z];
    uint32_t *order = (uint32_t *)(smem + M::ORDER);
    cg::cluster_group cluster = cg::this_cluster();          // the CTAs of one tile, a run of columns each
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank();
    grid_wait();
    if (blockIdx.y >= *a.lists.n_tiles) return;              // the same for all CTAs of a cluster
    const ATile t = a.lists.tiles[blockIdx.y];
    if (t.slot >= a.slots) return;
    if (tid < 2) bar_init(base + 8 * tid);
    if (warp == 0) tc_alloc(base + 32, Sums<RP>::COLS);
    if (tid < TM) order[tid] = a.lists.order[t.first + min(tid, t.rows - 1)];
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(*(volatile uint32_t *)(smem + 32));
    const Mat<W> m = job.w;
    const uint32_t per = ((m.width + parts - 1) / parts + KC - 1) / KC * KC, c_first = min(m.width, part * per), c_end = min(m.width, c_first + per);
    const uint32_t steps = uniform((c_end - c_first + KC - 1) / KC);
    const W *w = m.p + t.slot * m.slot;

    constexpr uint32_t XU = M::XU, ROWS = THREADS / (KC / 4);                        // rows from one run of four to the thread's next
    const uint32_t x_row = tid / (KC / 4), x_col = tid % (KC / 4) * 4, mine = base + M::RING + tid * 16, mine_w = base + M::RING + XU * THREADS * 16 + tid * 4 * sizeof(W);
    uint32_t x_at[XU];                                       // places in runs of four
    typename M::Run wv;
#pragma unroll
    for (uint32_t i = 0; i < XU; i++) x_at[i] = (uint32_t)((order[x_row + i * ROWS] * job.pitch + c_first + x_col) / 4);
    wv.begin(m, c_first);
    const float *x = job.x;
    auto copy = [&](uint32_t s) {
        if (s < steps) {
            const uint32_t c = c_first + s * KC + x_col;
            const uint32_t valid = places(c, c_end);
            if (job.x_fours) {
#pragma unroll
                for (uint32_t i = 0; i < XU; i++) {
                    const bool there = x_row + i * ROWS < t.rows && valid;
                    copy_async<16>(mine + i * THREADS * 16, there ? x + (uint64_t)x_at[i] * 4 : x, there ? 4 * valid : 0);
                    x_at[i] += KC / 4;
                }
            } else {
#pragma unroll 1
                for (uint32_t i = 0; i < XU; i++) {
                    const float *row = x + order[x_row + i * ROWS] * job.pitch;
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        const bool there = x_row + i * ROWS < t.rows && j < valid;
                        copy_async<4>(mine + i * THREADS * 16 + 4 * j, there ? row + c + j : x, there ? 4 : 0);
                    }
                }
            }
            if (m.fours) wv.copy(m, w, c_first + s * KC, c_end, mine_w, M::W_UNIT);
        }
    };
    copy(0);
    const uint32_t idesc = idesc_of(TM, RP, false, !m.wide);
    for (uint32_t s = 0; s < steps; s++) {
        const uint32_t c0 = c_first + s * KC, at = base + M::STAGE, wat = at + M::X::BYTES;
        copies_wait();
        if (s) bar_wait(base, (s - 1) & 1, a.status);
        if (s && s % FLUSH == 0) flush<RP>(tmem, s > FLUSH);
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) {
            Four<float> xv;
            xv.take(mine + i * THREADS * 16);
            xv.put(at + M::X::at(x_row + i * ROWS, x_col), M::X::PLANE);
        }
        if (m.fours) wv.take(mine_w, M::W_UNIT); else wv.load(m, w, c0, c_end);
        wv.put(m, c0, c_end, wat);
        copy(s + 1);
        fence_async();
        __syncthreads();
        if (warp == 0) {
            tc_after();
            const uint32_t leader = elect();                 // the thread whose products the commit answers for
            if (m.wide) step_mma<typename M::X, typename M::Run::Wide, 3, M::Run::PLANES, false, false, Sums<RP>::MAINS, KC / 16>(tmem, RP, tmem + Sums<RP>::SIDE, at, wat, idesc, s % FLUSH == 0, leader);
            else step_mma<typename M::X, typename M::Run::Tall, 3, M::Run::PLANES, false, true, Sums<RP>::MAINS, KC / 16>(tmem, RP, tmem + Sums<RP>::SIDE, at, wat, idesc, s % FLUSH == 0, leader);
            if (leader) tc_commit(base);
            __syncwarp();
        }
    }
    copies_wait();
    if (steps) bar_wait(base, (steps - 1) & 1, a.status);
    tc_after();
    grid_go();                                               // not before: CTAs of the next launch would crowd onto the SMs that are done first
    // accumulators to shared memory, summed over the cluster's CTAs in their order, scaled, cut and stored
    float *acc = (float *)(smem + M::STAGE);
    for (uint32_t c = (warp >> 2) * 16; c < RP; c += 32) {
        float v[16];
        load_sum<RP>(tmem + ((warp & 3) << 21) + c, v, Sums<RP>::MAINS, steps > FLUSH);
        float *row = acc + ((warp & 3) * 32 + lane) * M::PITCH + c;
#pragma unroll
        for (int i = 0; i < 16; i += 4) *(float4 *)(row + i) = steps ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_float4(0, 0, 0, 0);
    }
    // TMEM goes back before the CTAs wait for one another: two clusters that each held columns which a CTA of the other was waiting for
    // would wait for good
    tc_before();
    __syncthreads();
    if (warp == 0) { tc_after(); tc_free(tmem, Sums<RP>::COLS); }
    cluster.sync();
    const float scale = a.scale ? a.scale[t.slot] : 1.0f;
    const uint32_t rows = TM / parts, rows16 = (t.rows + 15) & ~15u;
    for (uint32_t u = tid; u < rows * (RP / 4); u += THREADS) {
        // two threads to eight values of a row, eight rows to 128 bytes of the result
        const uint32_t row = part * rows + u / (2 * RP) * 8 + (u >> 1 & 7), c = (u >> 4) % (RP / 8) * 8 + (u & 1) * 4;
        if (row >= rows16) break;
        float4 v[8], sum = make_float4(0, 0, 0, 0);
        for (uint32_t q = 0; q < parts; q += 8) {
#pragma unroll
            for (uint32_t p = 0; p < 8; p++) if (q + p < parts) v[p] = *(const float4 *)(cluster.map_shared_rank(acc, q + p) + row * M::PITCH + c);
#pragma unroll
            for (uint32_t p = 0; p < 8; p++) if (q + p < parts) { sum.x += v[p].x; sum.y += v[p].y; sum.z += v[p].z; sum.w += v[p].w; }
        }
        const bool there = row < t.rows;
        sum = make_float4(there ? sum.x * scale : 0, there ? sum.y * scale : 0, there ? sum.z * scale : 0, there ? sum.w * scale : 0);
        __nv_bfloat16 *to = job.planes + (uint64_t)((t.first + row) >> 3) * (8 * RP) + (c >> 3) * 64 + (row & 7) * 8 + (c & 7);
#pragma unroll
        for (int p = 0; p < 3; p++) {
            const uint32_t lo = cut2(sum.x, sum.y), hi = cut2(sum.z, sum.w);
            *(uint2 *)(to + p * a.plane) = make_uint2(lo, hi);
        }
    }
    cluster.sync();                                          // nobody leaves while its sums are read
}

// ---- expand -----------------------------------------------------------------------------------------------------------------
template <typename W> struct ExpandArgs {
    Mat<W> w;
    const __nv_bfloat16 *planes;                             // of shrink
    uint64_t plane;
    Lists lists;
    uint32_t slots;
    const float *base;
    uint64_t base_pitch;
    float *y;
    uint64_t y_pitch;
    uint32_t *status;
};
template <typename W, uint32_t RP> struct ExpandMap {
    using H = Rank<TM, RP>;                                  // rows tokens: K-major
    using Run = MatRun<W, RP, 128>;                          // Tall: K-major, Wide: MN-major
    static constexpr uint32_t PLACES = 64, H_AT = PLACES + TM * 16, W_AT = H_AT + H::BYTES, NEED = W_AT + Run::BYTES;
    // Never more than four CTAs on an SM, which have its 512 columns of TMEM: a fifth would hold its place waiting for columns (233472
    // bytes of shared memory to an SM, 1024 of them the system's for each CTA).
    static constexpr uint32_t TOTAL = NEED < 46080 ? 46080 : NEED, CTAS = TOTAL < 75000 ? 3 : TOTAL < 115000 ? 2 : 1;
    static_assert(5 * (TOTAL + 1024) > 233472 && TM == 128, "at most four CTAs of 128 TMEM columns");
};

// Columns of the projection are the accumulator's lanes and tokens its columns, so that a warp's 32 lanes hold 32 neighbouring values
// of a token's row.  base is read a batch of sixteen rows ahead of the one that is added.
template <typename W, uint32_t RP>
__global__ void __launch_bounds__(THREADS, ExpandMap<W, RP>::CTAS) adapter_expand_kernel(const __grid_constant__ ExpandArgs<W> a) {
    using M = ExpandMap<W, RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    struct Place { uint64_t b, y; };                         // bytes from the first row of base and of y
    Place *place = (Place *)(smem + M::PLACES);
    grid_go();
    // The lists are there: the launch before this one, whose end grid_wait waits for, let this one start after its own wait for them.
    if (blockIdx.y >= *a.lists.n_tiles) { grid_wait(); return; }                 // no launch ends before the one that it waits for
    const ATile t = a.lists.tiles[blockIdx.y];
    const bool none = t.slot >= a.slots;
    if (none && a.base == a.y) { grid_wait(); return; }
    const Mat<W> m = a.w;
    const uint32_t c0 = blockIdx.x * 128, c = c0 + (warp & 3) * 32 + lane;
    if (tid < 2) bar_init(base + 8 * tid);                   // products, rows of shrink
    if (tid < TM) {
        const uint64_t row = a.lists.order[t.first + min(tid, t.rows - 1)];
        place[tid] = Place{row * a.base_pitch * 4, row * a.y_pitch * 4};
    }
    const W *w = m.p + t.slot * m.slot;
    typename M::Run wv;
    const uint32_t n = uniform((t.rows + 15) & ~15u);
    if (!none) {
        wv.begin(m, c0);
        wv.load(m, w, c0, m.width);
    }
    if (warp == 0) tc_alloc(base + 32, TM);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(*(volatile uint32_t *)(smem + 32));
    if (tid == THREADS - 1) {
        grid_wait();
        if (!none) copy_rank<TM, RP>(base + M::H_AT, a.planes, a.plane, t.first, n, base + 8);
    }
    const uint32_t idesc = idesc_of(128, n, m.wide, false);
    const uint32_t t_first = (warp >> 2) * 64, t_last = min(t.rows, t_first + 64), d = tmem + ((warp & 3) << 21);
    const bool added = a.base != nullptr;
    const char *b_col = (const char *)(a.base + min(c, m.width - 1));
    char *y_col = (char *)(a.y + c);
    float b[16], v[16];
    auto fetch = [&](uint32_t j) {
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) b[i] = *(const float *)(b_col + place[j + i].b);
    };
    if (added && t_first < t_last) fetch(t_first);
    if (!none) {
        wv.put(m, c0, m.width, base + M::W_AT);
        fence_async();
        tc_before();
        __syncthreads();
        if (warp == 0) {
            tc_after();
            bar_wait(base + 8, 0, a.status);
            __syncwarp();
            const uint32_t leader = elect();
            if (m.wide) step_mma<typename M::Run::Wide, typename M::H, M::Run::PLANES, 3, true, false, 1, RP / 16>(tmem, 0, tmem, base + M::W_AT, base + M::H_AT, idesc, true, leader);
            else step_mma<typename M::Run::Tall, typename M::H, M::Run::PLANES, 3, false, false, 1, RP / 16>(tmem, 0, tmem, base + M::W_AT, base + M::H_AT, idesc, true, leader);
            if (leader) tc_commit(base);
            __syncwarp();
        }
        bar_wait(base, 0, a.status);
        tc_after();
    }
    for (uint32_t j = t_first; j < t_last; j += 16) {
        if (none) {
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) v[i] = 0;
        } else tc_load16(d + j, v);
        if (added)
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) v[i] = none ? b[i] : b[i] + v[i];
        if (added && j + 16 < t_last) fetch(j + 16);
        if (c < m.width)
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) if (j + i < t_last) *(float *)(y_col + place[j + i].y) = v[i];
    }
    tc_before();
    __syncthreads();
    if (warp == 0) tc_free(tmem, TM);
}

// ---- outer ------------------------------------------------------------------------------------------------------------------
struct OuterJob {
    const float *x;
    uint64_t pitch;
    uint32_t width;
    bool x_fours;
    const __nv_bfloat16 *planes;                             // of shrink
    float *d;                                                // [slots][rank * width]: (r, c) at r * sr + c * sc
    uint32_t sr, sc;
    uint32_t blocks;                                         // of 128 columns
};
struct OuterArgs {
    OuterJob job[2];
    Lists lists;
    uint64_t plane;
    uint32_t rank;
    uint32_t *status;
};
template <uint32_t RP> struct OuterMap {
    using X = Tile<TC, 128, 3>;                              // rows tokens: MN-major
    using H = Rank<TC, RP>;                                  // rows tokens: MN-major
    static constexpr uint32_t STAGE = 64, H_AT = STAGE + X::BYTES, END = H_AT + H::BYTES;
    static constexpr uint32_t PITCH = 132;                   // floats per r of the exchanged accumulators
    static constexpr uint32_t ACC_END = STAGE + RP * PITCH * 4, TOTAL = END > ACC_END ? END : ACC_END;
};

template <uint32_t RP>
__global__ void __launch_bounds__(THREADS, Sums<RP>::CTAS) adapter_outer_kernel(const __grid_constant__ OuterArgs a) {
    namespace cg = cooperative_groups;
    using M = OuterMap<RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    cg::cluster_group cluster = cg::this_cluster();          // a slot's tokens, a run to each CTA
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank(), slot = blockIdx.z;
    const bool second = blockIdx.y >= a.job[0].blocks;
    const OuterJob &job = a.job[second];
    const uint32_t c0 = (blockIdx.y - (second ? a.job[0].blocks : 0)) * 128;
    // the lists are there, as for expand
    const uint32_t begin = a.lists.offsets[2 * slot], tokens = a.lists.offsets[2 * slot + 1];
    const uint32_t cols = min(128u, job.width - c0), sr = job.sr, sc = job.sc;
    float *d = job.d + (uint64_t)slot * a.rank * job.width + c0 * sc;
    if (!tokens) {
        grid_wait();
        for (uint32_t u = part * THREADS + tid; u < a.rank * cols; u += parts * THREADS) d[sc == 1 ? u / cols * sr + u % cols : u % a.rank * sr + u / a.rank * sc] = 0;
        return;                                              // the same for all CTAs of the cluster
    }
    if (tid < 2) bar_init(base + 8 * tid);                   // products, rows of shrink
    if (warp == 0) tc_alloc(base + 32, Sums<RP>::COLS);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(*(volatile uint32_t *)(smem + 32));
    const uint32_t per = ((tokens + parts - 1) / parts + TC - 1) / TC * TC, from = min(tokens, part * per), to = min(tokens, from + per);
    const uint32_t steps = uniform((to - from + TC - 1) / TC);
    constexpr uint32_t XU = TC * 128 / 4 / THREADS;
    const uint32_t x_row = tid / 32, x_col = lane * 4;
    const float *x = job.x + c0;
    Four<float> xv[XU];
    uint32_t ids[XU];                                        // tokens of the step after the one that is fetched
    auto fetch_ids = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) ids[i] = a.lists.order[begin + min(t0 + x_row + i * 8, to - 1)];
    };
    auto fetch = [&](uint32_t t0) {
        if (job.x_fours && cols == 128) {
#pragma unroll
            for (uint32_t i = 0; i < XU; i++) xv[i].load4(x + ids[i] * job.pitch + x_col);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < XU; i++) xv[i].load1(x + ids[i] * job.pitch, x_col, cols - 1);
        }
        if (t0 + TC < to) fetch_ids(t0 + TC);
    };
    if (steps) { fetch_ids(from); fetch(from); }
    grid_wait();
    constexpr uint32_t idesc = idesc_of(128, RP, true, true);
    for (uint32_t s = 0; s < steps; s++) {
        const uint32_t t0 = from + s * TC;
        if (s) bar_wait(base, (s - 1) & 1, a.status);
        if (s && s % FLUSH == 0) flush<RP>(tmem, s > FLUSH);
        const uint32_t rows16 = uniform((min(to - t0, TC) + 15) & ~15u);
        if (tid == 0) copy_rank<TC, RP>(base + M::H_AT, job.planes, a.plane, begin + t0, rows16, base + 8);       // out of L2, while x is cut
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) xv[i].put(base + M::STAGE + M::X::at(x_row + i * 8, x_col), M::X::PLANE);
        fence_async();
        __syncthreads();
        if (warp == 0) {
            tc_after();
            bar_wait(base + 8, s & 1, a.status);
            __syncwarp();
            const uint32_t leader = elect();
            if (rows16 == TC)
                step_mma<typename M::X, typename M::H, 3, 3, true, true, Sums<RP>::MAINS, TC / 16>(tmem, RP, tmem + Sums<RP>::SIDE, base + M::STAGE, base + M::H_AT, idesc, s % FLUSH == 0, leader);
            else                                             // the last tokens; into one of the leading accumulators alone, the others as they are
                for (uint32_t k = 0; k < rows16 / 16; k++)
                    step_mma<typename M::X, typename M::H, 3, 3, true, true, 1, 1>(tmem, RP, tmem + Sums<RP>::SIDE, base + M::STAGE + k * M::X::k16(true),
                                                                                    base + M::H_AT + k * M::H::k16(true), idesc, s % FLUSH == 0 && k == 0, leader);
            if (leader) tc_commit(base);
            __syncwarp();
        }
        if (s + 1 < steps) fetch(t0 + TC);
    }
    if (steps) bar_wait(base, (steps - 1) & 1, a.status);
    tc_after();
    grid_go();
    // the last tokens alone, if no whole step came before them since the last flush, are in one leading accumulator
    const uint32_t mains = steps && to - from - (steps - 1) / FLUSH * (FLUSH * TC) + 15 < TC ? 1 : Sums<RP>::MAINS;
    float *acc = (float *)(smem + M::STAGE);
    for (uint32_t c = (warp >> 2) * 16; c < RP; c += 32) {
        float v[16];
        load_sum<RP>(tmem + ((warp & 3) << 21) + c, v, mains, steps > FLUSH);
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) acc[(c + i) * M::PITCH + (warp & 3) * 32 + lane] = steps ? v[i] : 0.0f;
    }
    // TMEM goes back before the CTAs wait for one another: two clusters that each held columns which a CTA of the other was waiting for
    // would wait for good
    tc_before();
    __syncthreads();
    if (warp == 0) { tc_after(); tc_free(tmem, Sums<RP>::COLS); }
    cluster.sync();
    for (uint32_t u = part * THREADS + tid; u < RP * 32; u += parts * THREADS) {
        // neighbouring threads: neighbouring columns of dA, neighbouring r of dB
        const uint32_t r = sc == 1 ? u / 32 : u % RP, c = (sc == 1 ? u % 32 : u / RP) * 4;
        if (r >= a.rank || c >= cols) continue;
        float4 v[8], sum = make_float4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t p = 0; p < 8; p++) if (p < parts) v[p] = *(const float4 *)(cluster.map_shared_rank(acc, p) + r * M::PITCH + c);
#pragma unroll
        for (uint32_t p = 0; p < 8; p++) if (p < parts) { sum.x += v[p].x; sum.y += v[p].y; sum.z += v[p].z; sum.w += v[p].w; }
        float *to_at = d + r * sr + c * sc;
        to_at[0] = sum.x;
        if (c + 1 < cols) to_at[sc] = sum.y;
        if (c + 2 < cols) to_at[2 * sc] = sum.z;
        if (c + 3 < cols) to_at[3 * sc] = sum.w;
    }
    cluster.sync();
}

// ---- a few tokens -----------------------------------------------------------------------------------------------------------
// One cluster of eight CTAs to a token, whatever its slot: A x with a run of columns of x to each CTA, the eight partial sums of every r
// to all of them (distributed shared memory), B h with a run of y's columns to each.  Everything is read once and one launch is all
// there is.  What bounds it is latency: the id, then A, the exchange, then the sum; B and base are on their way meanwhile.
constexpr uint32_t FEW_CTAS = 8;

template <typename W> struct FewArgs {
    const W *a, *b;
    uint32_t slots, rank, k, n;
    const float *scale, *x;
    uint64_t x_pitch;
    const uint32_t *ids;
    const float *base;
    uint64_t base_pitch;
    float *y;
    uint64_t y_pitch;
    bool x_fours;
    uint32_t *status;
};

// V neighbouring values of a row in one load, and their products with floats.
template <typename W, int V> struct Run;
template <int V> struct Run<float, V> {
    float v[V];
    __device__ __forceinline__ void load(const float *p) {
        if (V == 4) { const float4 u = *(const float4 *)p; v[0] = u.x; v[V / 4] = u.y; v[V / 2] = u.z; v[V - 1] = u.w; }
        else v[0] = *p;
    }
    __device__ __forceinline__ float dot(const float *f, float sum) const {
#pragma unroll
        for (int i = 0; i < V; i++) sum = fmaf(v[i], f[i], sum);
        return sum;
    }
};
__device__ __forceinline__ float2 pair_of(uint32_t u, const __nv_bfloat16 *) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ float2 pair_of(uint32_t u, const __half *) { return __half22float2(*(const __half2 *)&u); }
template <typename H, int V> struct Run16 {
    uint32_t v[V > 1 ? V / 2 : 1];
    __device__ __forceinline__ void load(const H *p) {
        if (V == 8) { const uint4 u = *(const uint4 *)p; v[0] = u.x; v[V / 8] = u.y; v[V / 4] = u.z; v[V / 2 - 1] = u.w; }
        else if (V == 4) { const uint2 u = *(const uint2 *)p; v[0] = u.x; v[V / 4] = u.y; }
        else v[0] = *(const uint16_t *)p;
    }
    __device__ __forceinline__ float dot(const float *f, float sum) const {
        if constexpr (V == 1) sum = fmaf(pair_of(v[0], (const H *)nullptr).x, f[0], sum);
        else
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                const float2 u = pair_of(v[i], (const H *)nullptr);
                sum = fmaf(u.y, f[2 * i + 1], fmaf(u.x, f[2 * i], sum));
            }
        return sum;
    }
};
template <int V> struct Run<__nv_bfloat16, V> : Run16<__nv_bfloat16, V> {};
template <int V> struct Run<__half, V> : Run16<__half, V> {};

template <typename W, int V>
__global__ void __launch_bounds__(THREADS, 4) adapter_few_kernel(const __grid_constant__ FewArgs<W> a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ float partial[FEW_CTAS][QW4CU_TUNE_MAX_RANK], h[QW4CU_TUNE_MAX_RANK];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, part = blockIdx.x, t = blockIdx.y, R = a.rank;
    grid_wait();
    const uint32_t s = a.ids[t];
    const uint32_t n_per = (a.n + FEW_CTAS - 1) / FEW_CTAS, n0 = min(a.n, part * n_per), n1 = min(a.n, n0 + n_per);
    const float *base = a.base ? a.base + t * a.base_pitch : nullptr;
    float *y = a.y + t * a.y_pitch;
    if (s >= a.slots) {                                      // the same for all CTAs of the cluster
        if (s != QW4CU_NO_ADAPTER && tid == 0) atomicOr(a.status, QW4SH_ERR_BOUNDS);
        if (base != y) for (uint32_t c = n0 + tid; c < n1; c += THREADS) y[c] = base ? base[c] : 0.0f;
        return;
    }
    const W *A = a.a + (uint64_t)s * R * a.k, *B = a.b + (uint64_t)s * R * a.n;
    const float *x = a.x + t * a.x_pitch;
    cluster.barrier_arrive();                                // whoever writes to another CTA's shared memory has to know that it has begun

    // rows of B: `span` lanes to a row, so that a load of a warp is one run of memory
    uint32_t span = 1;
    while (span < 32 && span * V < R) span *= 2;
    const uint32_t sub = lane % span, rows = 32 / span, n_first = n0 + warp * rows + lane / span, n_step = 8 * rows;
    constexpr int PASSES = 4;
    Run<W, V> bv[PASSES];
    float added[PASSES];
    auto fetch = [&](uint32_t n) {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const uint32_t row = min(n + i * n_step, a.n - 1);
            bv[i].load(B + (uint64_t)row * R + min(sub * V, R - V));
            added[i] = base ? base[row] : 0.0f;
        }
    };
    fetch(n_first);

    const uint32_t k_per = ((a.k + V - 1) / V + FEW_CTAS - 1) / FEW_CTAS * V, c0 = min(a.k, part * k_per), c1 = min(a.k, c0 + k_per);
    constexpr uint32_t RANKS = 4;                            // of a warp at a time
    for (uint32_t r0 = warp; r0 < R; r0 += 8 * RANKS) {
        float sum[RANKS] = {};
        for (uint32_t c = c0 + lane * V; c < c1; c += 32 * V) {
            float xv[V];
            Run<W, V> av[RANKS];
#pragma unroll
            for (uint32_t j = 0; j < RANKS; j++) av[j].load(A + (uint64_t)min(r0 + 8 * j, R - 1) * a.k + c);
            if (V >= 4 && a.x_fours) {
#pragma unroll
                for (int i = 0; i < V; i += 4) { const float4 u = *(const float4 *)(x + c + i); xv[i] = u.x; xv[(i + 1) % V] = u.y; xv[(i + 2) % V] = u.z; xv[(i + 3) % V] = u.w; }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) xv[i] = x[c + i];
            }
#pragma unroll
            for (uint32_t j = 0; j < RANKS; j++) sum[j] = av[j].dot(xv, sum[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < RANKS; j++)
#pragma unroll
            for (int o = 16; o; o >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
        if (r0 == warp) cluster.barrier_wait();
        if (lane < FEW_CTAS) {
            float *to = cluster.map_shared_rank(&partial[part][0], lane);
#pragma unroll
            for (uint32_t j = 0; j < RANKS; j++) if (r0 + 8 * j < R) to[r0 + 8 * j] = sum[j];
        }
    }
    if (warp >= R) cluster.barrier_wait();                   // a warp without an r
    cluster.sync();
    if (tid < R) {
        float sum = 0;
#pragma unroll
        for (uint32_t p = 0; p < FEW_CTAS; p++) sum += partial[p][tid];
        h[tid] = sum * (a.scale ? a.scale[s] : 1.0f);
    }
    __syncthreads();
    for (uint32_t n = n_first; n - lane / span < n1; n += PASSES * n_step) {
        if (n != n_first) fetch(n);
        float sum[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            sum[i] = sub * V < R ? bv[i].dot(h + sub * V, 0.0f) : 0.0f;
            for (uint32_t r = (sub + span) * V; r < R; r += span * V) {              // more values to a row than a warp has lanes for
                Run<W, V> more;
                more.load(B + (uint64_t)min(n + i * n_step, a.n - 1) * R + r);
                sum[i] = more.dot(h + r, sum[i]);
            }
        }
        for (uint32_t o = span / 2; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < PASSES; i++) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
#pragma unroll
        for (int i = 0; i < PASSES; i++) if (sub == 0 && n + i * n_step < n1) y[n + i * n_step] = added[i] + sum[i];
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <typename... A>
int launch(void (*kernel)(A...), const char *name, dim3 grid, uint32_t threads, size_t smem, uint32_t cluster, bool behind, cudaStream_t stream, A... args) {
    if (smem > 40u * 1024u && qw4sh_allow_smem((const void *)kernel, smem)) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    uint32_t n = 0;
    if (behind) { attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[n++].val.programmaticStreamSerializationAllowed = 1; }
    if (cluster) { attr[n].id = cudaLaunchAttributeClusterDimension; attr[n].val.clusterDim.x = cluster; attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1; n++; }
    cfg.attrs = attr; cfg.numAttrs = n;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    return qw4sh_note_launch(name);
}

bool fours(const void *p, size_t step, size_t element) { return (uintptr_t)p % (4 * element) == 0 && step % 4 == 0; }

constexpr uint32_t SMS = 148;

// Most CTAs to a cluster of this kernel: sixteen where the device has room for one (eight is what every device promises).
uint32_t most_ctas(const void *kernel, size_t smem) {
    static struct { const void *kernel; int device; uint32_t most; } have[64];
    static uint32_t n = 0;
    static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 8;
    pthread_mutex_lock(&lock);
    uint32_t i = 0, most = 8;
    while (i < n && (have[i].kernel != kernel || have[i].device != device)) i++;
    if (i < n) most = have[i].most;
    else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(16); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension; attr.val.clusterDim.x = 16; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess && !qw4sh_allow_smem(kernel, smem) &&
            cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters >= 4) most = 16;
        (void)cudaGetLastError();
        if (n < 64) { have[n].kernel = kernel; have[n].device = device; have[n++].most = most; }
    }
    pthread_mutex_unlock(&lock);
    return most;
}
struct Shape {
    uint32_t T, S, R, RP, tiles;                             // tiles: most that there can be
    Lists lists;
    const float *scale;
    uint32_t *status;
    uint64_t plane;
    cudaStream_t stream;
};

int make_lists(const QW4ShTune *tune, const QW4CuAdapters *ad, const uint32_t *slots, size_t T, cudaStream_t stream, Shape &s) {
    s.T = (uint32_t)T; s.S = ad->slots; s.R = ad->rank; s.RP = qw4sh_adapter_rank(ad->rank);
    s.tiles = (uint32_t)qw4sh_adapter_tiles(T, s.S);
    s.lists = {tune->order, tune->offsets, (const ATile *)tune->tiles, tune->n_tiles};
    s.scale = ad->scale; s.status = tune->status; s.plane = qw4sh_adapter_rows(T, s.S) * s.RP; s.stream = stream;
    return launch(adapter_lists_kernel, "adapter_lists_kernel", dim3(1), 1024, (size_t)33 * (s.S + 1) * 4, 0, true, stream, slots, s.T, s.S, tune->order,
                  tune->offsets, (ATile *)tune->tiles, tune->n_tiles, tune->status);
}

// CTAs to a cluster: as many as `ctas` has room for, with a run of `least` each at least.
uint32_t cluster_of(uint64_t items, uint64_t length, uint32_t least, uint32_t ctas, uint32_t most = 8) {
    uint32_t c = 1;
    while (c < most && items * 2 * c <= ctas && length / (2 * c) >= least) c *= 2;
    return c;
}

template <typename W, uint32_t RP>
int shrink(const ShrinkJob<W> *jobs, uint32_t all, uint32_t n, const Shape &s) {
    // cut as for all the jobs that there may be: the bits of one do not depend on whether the other was asked for
    ShrinkArgs<W> a = {};
    uint64_t width = 0;
    for (uint32_t i = 0; i < all; i++) { a.job[i] = jobs[i]; if (jobs[i].w.width > width) width = jobs[i].w.width; }
    a.lists = s.lists; a.scale = s.scale; a.plane = s.plane; a.slots = s.S; a.status = s.status;
    const uint32_t c = cluster_of((uint64_t)(s.T + TM - 1) / TM * all, width, 128, 2 * SMS, most_ctas((const void *)adapter_shrink_kernel<W, RP>, ShrinkMap<W, RP>::TOTAL));
    return launch(adapter_shrink_kernel<W, RP>, "adapter_shrink_kernel", dim3(c, s.tiles, n), THREADS, ShrinkMap<W, RP>::TOTAL, c, true, s.stream, a);
}
template <typename W, uint32_t RP>
int expand(const Mat<W> &w, const __nv_bfloat16 *planes, const float *base, size_t base_pitch, float *y, size_t y_pitch, const Shape &s) {
    const ExpandArgs<W> a = {w, planes, s.plane, s.lists, s.S, base, base_pitch, y, y_pitch, s.status};
    return launch(adapter_expand_kernel<W, RP>, "adapter_expand_kernel", dim3((w.width + 127) / 128, s.tiles), THREADS, ExpandMap<W, RP>::TOTAL, 0, true, s.stream, a);
}
template <uint32_t RP>
int outer(const OuterJob *jobs, const Shape &s) {
    OuterArgs a = {{jobs[0], jobs[1]}, s.lists, s.plane, s.R, s.status};
    const uint32_t blocks = jobs[0].blocks + jobs[1].blocks;
    const uint32_t c = cluster_of((uint64_t)blocks * ((s.T + 1023) / 1024 < s.S ? (s.T + 1023) / 1024 : s.S), s.T, TC, 4 * SMS);
    return launch(adapter_outer_kernel<RP>, "adapter_outer_kernel", dim3(c, blocks, s.S), THREADS, OuterMap<RP>::TOTAL, c, true, s.stream, a);
}

template <typename W> Mat<W> mat_a(const QW4CuAdapters *ad) { return {(const W *)ad->a, ad->rank * ad->k, ad->rank, (uint32_t)ad->k, true, fours(ad->a, ad->k, sizeof(W))}; }
template <typename W> Mat<W> mat_b(const QW4CuAdapters *ad) { return {(const W *)ad->b, ad->rank * ad->n, ad->rank, (uint32_t)ad->n, false, fours(ad->b, ad->rank, sizeof(W))}; }

struct Rows { const float *p; size_t pitch; };
bool runs(Rows x, uint64_t T) { return fours(x.p, x.pitch, 4) && T * x.pitch < 1ull << 34; }

template <typename W>
int few(const QW4ShTune *tune, const QW4CuAdapters *ad, Rows x, const uint32_t *slots, Rows base, float *y, size_t y_pitch, size_t T, cudaStream_t stream) {
    const FewArgs<W> a = {(const W *)ad->a, (const W *)ad->b, ad->slots, ad->rank, (uint32_t)ad->k, (uint32_t)ad->n, ad->scale, x.p, x.pitch, slots,
                          base.p, base.pitch, y, y_pitch, fours(x.p, x.pitch, 4), tune->status};
    constexpr int MOST = 16 / sizeof(W);
    auto runs_of = [&](uint32_t v) { return ad->k % v == 0 && ad->rank % v == 0 && (((uintptr_t)ad->a | (uintptr_t)ad->b) & (v * sizeof(W) - 1)) == 0; };
    const auto kernel = runs_of(MOST) ? adapter_few_kernel<W, MOST> : runs_of(4) ? adapter_few_kernel<W, 4> : adapter_few_kernel<W, 1>;
    return launch(kernel, "adapter_few_kernel", dim3(FEW_CTAS, (unsigned)T), THREADS, 0, FEW_CTAS, true, stream, a);
}
template <typename W, uint32_t RP>
int forward(const QW4ShTune *tune, const QW4CuAdapters *ad, Rows x, Rows base, float *y, size_t y_pitch, const Shape &s) {
    const ShrinkJob<W> job = {mat_a<W>(ad), x.p, x.pitch, runs(x, s.T), (__nv_bfloat16 *)tune->h};
    if (const int rc = shrink<W, RP>(&job, 1, 1, s)) return rc;
    return expand<W, RP>(mat_b<W>(ad), job.planes, base.p, base.pitch, y, y_pitch, s);
}
template <typename W, uint32_t RP>
int backward(const QW4ShTune *tune, const QW4CuAdapters *ad, Rows x, Rows dy, Rows base, float *dx, size_t dx_pitch, float *da, float *db, const Shape &s) {
    const ShrinkJob<W> jobs[2] = {{mat_b<W>(ad), dy.p, dy.pitch, runs(dy, s.T), (__nv_bfloat16 *)tune->g},
                                  {mat_a<W>(ad), x.p, x.pitch, runs(x, s.T), (__nv_bfloat16 *)tune->h}};
    int rc;
    if ((rc = shrink<W, RP>(jobs, 2, da ? 2 : 1, s))) return rc;
    const OuterJob outers[2] = {{x.p, x.pitch, (uint32_t)ad->k, jobs[1].x_fours, jobs[0].planes, da, (uint32_t)ad->k, 1, (uint32_t)((ad->k + 127) / 128)},
                                {dy.p, dy.pitch, (uint32_t)ad->n, jobs[0].x_fours, jobs[1].planes, db, 1, ad->rank, (uint32_t)((ad->n + 127) / 128)}};
    // dA and dB behind shrink, which has just read what they read
    if (da && (rc = outer<RP>(outers, s))) return rc;
    return dx ? expand<W, RP>(mat_a<W>(ad), jobs[0].planes, base.p, base.pitch, dx, dx_pitch, s) : 0;
}

#define BY_RANK(f, W, ...) (s.RP == 16 ? f<W, 16>(__VA_ARGS__) : s.RP == 32 ? f<W, 32>(__VA_ARGS__) : s.RP == 64 ? f<W, 64>(__VA_ARGS__) : f<W, 128>(__VA_ARGS__))
#define BY_TYPE(f, ...) (ad->type == 0 ? BY_RANK(f, float, __VA_ARGS__) : ad->type == 1 ? BY_RANK(f, __half, __VA_ARGS__) : BY_RANK(f, __nv_bfloat16, __VA_ARGS__))

}  // namespace

extern "C" uint32_t qw4sh_adapter_rank(uint32_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }
// Places of the sorted tokens: every group rounded up to sixteen.
extern "C" size_t qw4sh_adapter_rows(size_t tokens, uint32_t slots) {
    const size_t groups = tokens < slots + 1u ? tokens : slots + 1u;
    return (tokens + 15 * groups + 15) & ~(size_t)15;
}
// Most tiles that there can be: a token in each group, and then whole tiles.
extern "C" size_t qw4sh_adapter_tiles(size_t tokens, uint32_t slots) {
    const size_t groups = tokens < slots + 1u ? tokens : slots + 1u;
    return (tokens - groups) / TM + groups;
}

extern "C" int qw4sh_adapter_forward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                                     const float *base, size_t base_pitch, float *y, size_t y_pitch, size_t tokens, void *stream) {
    const Rows xr = {x, x_pitch}, br = {base, base_pitch};
    // A cluster per token costs a token its adapter out of L2 every time, the grouped products three launches and a tile of 128 rows for every adapter
    // in use.  us, cluster | grouped, BF16, 2048 -> 2048, tokens spread evenly over 8 slots: rank 16 128 tokens 10.2 | 15.7, 192 tokens 14.8 | 16.1;
    // rank 32 128 tokens 12.4 | 16.2, 192 tokens 17.7 | 16.8; rank 64 64 tokens 12.4 | 17.1, 80 tokens 17.4 | 17.2, 96 tokens 19.7 | 17.1; rank 128 64 tokens
    // 20.5 | 26.2, 80 tokens 28.4 | 26.3.  With one slot, and 2048 -> 512 and 512 -> 2048, the rule's choice is at most 27% behind the other.
    // It takes adapters to be shared: the more of them are in use the later the crossing comes (rank 64, 192 tokens: 31 | 28 with 24, 31 | 49 with 48 in use).
    if (tokens <= 64 || (tokens <= 192 && tokens * ad->rank <= 5120))
        return (ad->type == 0 ? few<float> : ad->type == 1 ? few<__half> : few<__nv_bfloat16>)(tune, ad, xr, slots, br, y, y_pitch, tokens, (cudaStream_t)stream);
    Shape s;
    if (const int rc = make_lists(tune, ad, slots, tokens, (cudaStream_t)stream, s)) return rc;
    return BY_TYPE(forward, tune, ad, xr, br, y, y_pitch, s);
}

extern "C" int qw4sh_adapter_backward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                                      const float *dy, size_t dy_pitch, const float *base, size_t base_pitch, float *dx, size_t dx_pitch,
                                      float *da, float *db, size_t tokens, void *stream) {
    if (!tokens) {
        if (!da) return 0;
        const size_t a = (size_t)ad->slots * ad->rank * ad->k * 4, b = (size_t)ad->slots * ad->rank * ad->n * 4;
        return qw4sh_memset_async(da, 0, a, stream) || qw4sh_memset_async(db, 0, b, stream);
    }
    Shape s;
    if (const int rc = make_lists(tune, ad, slots, tokens, (cudaStream_t)stream, s)) return rc;
    const Rows xr = {x, x_pitch}, dr = {dy, dy_pitch}, br = {base, base_pitch};
    return BY_TYPE(backward, tune, ad, xr, dr, br, dx, dx_pitch, da, db, s);
}
