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
// i + j <= 2; what is left out is below 2^-24 of a product.
//
// Operands are written to shared memory by the CTA's threads, which cut them on the way, as 8 x 16-byte core matrices without
// swizzle: [8 columns][8 rows][16 bytes], so that rows of the source can be the rows of either major-ness.  Column groups
// lie 16 bytes further apart than they are long: eight lanes that write one row's eight groups then meet in no bank.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cuda_shim.h"

extern "C" int qw4sh_note_launch(const char *name);
extern "C" int qw4sh_fail_text(const char *text);
extern "C" int qw4sh_allow_smem(const void *kernel, size_t smem);

namespace {

constexpr uint32_t THREADS = 256, TM = 128;                  // tokens per tile: tcgen05's M (shrink) or most N (expand)
constexpr uint32_t KC = 64;                                  // shrink: columns per step
constexpr uint32_t TC = 32;                                  // outer: tokens per step

// ---- PTX ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
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
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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

__device__ __forceinline__ void put8(uint32_t addr, uint32_t a, uint32_t b) { asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory"); }
__device__ __forceinline__ void put16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

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

// Four neighbouring values of a row as they are in memory; `valid` of them exist.  `wide`: rows start on a boundary of four values.
template <typename W> struct Four;
template <> struct Four<float> {
    static constexpr int PLANES = 3;
    float4 v;
    __device__ __forceinline__ void load(const float *p, int valid, bool wide) {
        if (valid >= 4 && wide) { v = *(const float4 *)p; return; }
        v = make_float4(0, 0, 0, 0);
        if (valid > 0) v.x = p[0];
        if (valid > 1) v.y = p[1];
        if (valid > 2) v.z = p[2];
        if (valid > 3) v.w = p[3];
    }
    __device__ __forceinline__ void put(uint32_t addr, uint32_t step) const { put_cut<3>(addr, step, v); }
};
template <typename H> struct Four16 {
    uint2 v;
    __device__ __forceinline__ void load(const H *q, int valid, bool wide) {
        const uint16_t *p = (const uint16_t *)q;
        if (valid >= 4 && wide) { v = *(const uint2 *)p; return; }
        v = make_uint2(0, 0);
        if (valid > 0) v.x = p[0];
        if (valid > 1) v.x |= (uint32_t)p[1] << 16;
        if (valid > 2) v.y = p[2];
        if (valid > 3) v.y |= (uint32_t)p[3] << 16;
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

// The adapters of all slots as [rank, width] matrices: WIDE: rows of the rank axis (A), else rows of the wide axis (B).
template <typename W> struct Mat { const W *p; uint64_t slot; uint32_t rank; uint64_t width; bool wide; };

// ---- lists ------------------------------------------------------------------------------------------------------------------
// Tokens sorted by slot (tokens without one last, in the group `slots`), in the order of the batch inside a slot; tiles of up to
// 128 tokens of one slot.  One CTA: every warp counts a run of tokens, then places it.
struct ATile { uint32_t slot, first, rows, pad; };

__global__ void __launch_bounds__(1024) adapter_lists_kernel(const uint32_t *__restrict__ ids, uint32_t T, uint32_t S, uint32_t *__restrict__ order,
                                                             uint32_t *__restrict__ offsets, ATile *__restrict__ tiles, uint32_t *__restrict__ n_tiles,
                                                             uint32_t *status) {
    extern __shared__ uint32_t counts[];                     // [warps][S + 1]
    __shared__ uint32_t sums[2][32];
    const uint32_t G = S + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t per = ((T + 31) / 32 + 31) & ~31u, first = warp * per, end = min(T, first + per);
    for (uint32_t i = threadIdx.x; i < 32 * G; i += 1024) counts[i] = 0;
    __syncthreads();
    uint32_t *mine = counts + warp * G;
    for (uint32_t t = first + lane; t - lane < end; t += 32) {
        uint32_t s = 0xffffffffu;
        if (t < end) {
            s = ids[t];
            if (s >= S) {
                if (s != QW4CU_NO_ADAPTER) atomicOr(status, QW4SH_ERR_BOUNDS);
                s = S;
            }
        }
        const uint32_t same = __match_any_sync(0xffffffffu, s);
        if (t < end && __ffs(same) - 1 == (int)lane) mine[s] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // a thread per group (two where there are more than 1024): where the group and its tiles start
    uint32_t total[2] = {0, 0}, rows_before = 0, tiles_before = 0;
    for (uint32_t j = 0; j < 2; j++) {
        const uint32_t g = 2 * threadIdx.x + j;
        if (g < G) for (uint32_t w = 0; w < 32; w++) { const uint32_t c = counts[w * G + g]; counts[w * G + g] = total[j]; total[j] += c; }
    }
    uint32_t r = total[0] + total[1], n = (total[0] + TM - 1) / TM + (total[1] + TM - 1) / TM;
    const uint32_t own_r = r, own_n = n;
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) { r += a; n += b; }
    }
    if (lane == 31) { sums[0][warp] = r; sums[1][warp] = n; }
    __syncthreads();
    for (uint32_t w = 0; w < warp; w++) { rows_before += sums[0][w]; tiles_before += sums[1][w]; }
    rows_before += r - own_r;
    tiles_before += n - own_n;
    for (uint32_t j = 0; j < 2; j++) {
        const uint32_t g = 2 * threadIdx.x + j;
        if (g >= G) break;
        for (uint32_t w = 0; w < 32; w++) counts[w * G + g] += rows_before;
        offsets[g] = rows_before;
        for (uint32_t at = 0; at < total[j]; at += TM) tiles[tiles_before++] = ATile{g, rows_before + at, min(TM, total[j] - at), 0};
        rows_before += total[j];
        if (g == S) { offsets[G] = rows_before; *n_tiles = tiles_before; }
    }
    __syncthreads();
    for (uint32_t t = first + lane; t - lane < end; t += 32) {
        uint32_t s = 0xffffffffu;
        if (t < end) s = min(ids[t], S);
        const uint32_t same = __match_any_sync(0xffffffffu, s);
        uint32_t at = 0;
        if (t < end) at = mine[s];
        __syncwarp();
        if (t < end) {
            order[at + __popc(same & ((1u << lane) - 1))] = t;
            if (__ffs(same) - 1 == (int)lane) mine[s] = at + __popc(same);
        }
        __syncwarp();
    }
}

// ---- accumulators ---------------------------------------------------------------------------------------------------------
template <uint32_t RP> struct Sums {
    static constexpr uint32_t MAINS = RP <= 64 ? 2 : 1, SIDE = MAINS * RP, NEED = SIDE + RP;
    static constexpr uint32_t COLS = NEED <= 64 ? 64 : NEED <= 128 ? 128 : 256;                      // TMEM is handed out in powers of two
};

// ---- shrink -----------------------------------------------------------------------------------------------------------------
struct Lists { const uint32_t *order, *offsets; const ATile *tiles; const uint32_t *n_tiles; };

template <typename W> struct ShrinkJob {
    Mat<W> w;
    const float *x;
    uint64_t pitch;
    bool x_wide, w_wide;                                     // rows on boundaries of four values
    __nv_bfloat16 *planes;                                   // [3][rows][RP]: the result cut in three, rows in the lists' order
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
    static constexpr int WP = Four<W>::PLANES;
    using X = Tile<TM, KC, 3>;
    using WideW = Tile<RP, KC, WP>;                          // rows r, columns of the wide axis: K-major
    using TallW = Tile<KC, RP, WP>;                          // rows of the wide axis, columns r: MN-major
    static constexpr uint32_t W_BYTES = WideW::BYTES > TallW::BYTES ? WideW::BYTES : TallW::BYTES;
    static constexpr uint32_t STAGE = (X::BYTES + W_BYTES + 15) & ~15u;
    static constexpr uint32_t ORDER = 64, STAGES_AT = ORDER + TM * 4;
    static constexpr uint32_t TOTAL = STAGES_AT + 2 * STAGE;
    static constexpr uint32_t PITCH = RP + 4;                // floats per row of the exchanged accumulators
    static_assert(TM * PITCH * 4 <= 2 * STAGE, "accumulators fit the stages");
    static constexpr uint32_t COLS = Sums<RP>::COLS;
};

// An accumulator loses up to a bit's weight at every instruction that adds to it (additions in the tensor core truncate), always towards
// zero, so what counts is how many add to the same one.  Products of the leading planes go to MAINS accumulators in turn, and
// the corrections, 2^-8 of them and less, to one of their own (`side`), where their truncations are as much smaller; the sums meet
// in FP32 when they are read.  With all six products in one accumulator dA of 8192 tokens was 5.9e-6 off, as the plain form in FP32 is
// 0.9e-6.
template <typename TA, typename TB, int PA, int PB, bool AMN, bool BMN, uint32_t MAINS>
__device__ __forceinline__ void step_mma(uint32_t d, uint32_t d_step, uint32_t side, uint32_t a, uint32_t b, uint32_t idesc, uint32_t k16s, bool first, uint32_t leader) {
    uint32_t accumulate = first ? 0 : 1;
#pragma unroll
    for (int order = 2; order > 0; order--)                  // the smallest first
        for (uint32_t k = 0; k < k16s; k++)
#pragma unroll
            for (int i = 0; i < PA; i++) {
                const int j = order - i;
                if (j < 0 || j >= PB) continue;
                if (leader) tc_mma(side, TA::desc(a + i * TA::PLANE + k * TA::k16(AMN), AMN), TB::desc(b + j * TB::PLANE + k * TB::k16(BMN), BMN), idesc, accumulate);
                accumulate = 1;
            }
    for (uint32_t k = 0; k < k16s; k++) {
        const uint32_t to = d + k % MAINS * d_step;
        if (leader) tc_mma(to, TA::desc(a + k * TA::k16(AMN), AMN), TB::desc(b + k * TB::k16(BMN), BMN), idesc, to == side || !first || k >= MAINS);
    }
}
// Sixteen columns of a sum that lies in the accumulators of shrink and outer.
template <uint32_t RP, uint32_t MAINS> __device__ __forceinline__ void load_sum(uint32_t addr, float (&v)[16]) {
    float u[16];
    tc_load16(addr, v);
#pragma unroll
    for (uint32_t m = 1; m <= MAINS; m++) {
        tc_load16(addr + m * RP, u);
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] += u[i];
    }
}
template <typename W, uint32_t RP>
__global__ void __launch_bounds__(THREADS) adapter_shrink_kernel(const __grid_constant__ ShrinkArgs<W> a) {
    namespace cg = cooperative_groups;
    using M = ShrinkMap<W, RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    const ShrinkJob<W> &job = a.job[blockIdx.z];
    uint32_t *order = (uint32_t *)(smem + M::ORDER);
    cg::cluster_group cluster = cg::this_cluster();          // the CTAs of one tile, a run of columns each
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank();
    grid_wait();
    grid_go();
    const uint32_t tile = blockIdx.y;
    if (tile >= *a.lists.n_tiles) return;                    // the same for all CTAs of a cluster
    const ATile t = a.lists.tiles[tile];
    if (t.slot >= a.slots) return;
    const uint32_t rank = job.w.rank;
    if (tid < 2) bar_init(base + 8 * tid);
    if (warp == 0) tc_alloc(base + 32, M::COLS);
    if (tid < TM) order[tid] = tid < t.rows ? a.lists.order[t.first + tid] : 0;
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *(volatile uint32_t *)(smem + 32);
    const uint64_t width = job.w.width;
    const uint64_t per = ((width + parts - 1) / parts + KC - 1) / KC * KC, c_first = min(width, part * per), c_end = min(width, c_first + per);
    const uint32_t steps = (uint32_t)((c_end - c_first + KC - 1) / KC);
    const W *w = job.w.p + t.slot * job.w.slot;

    constexpr uint32_t XU = TM * KC / 4 / THREADS, WU = RP * KC / 4 / THREADS;       // runs of four values per thread
    Four<float> xv[XU];
    Four<W> wv[WU];
    const uint32_t x_row = tid / (KC / 4), x_col = tid % (KC / 4) * 4;
    auto fetch = [&](uint64_t c0) {
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) {
            const uint32_t row = x_row + i * (THREADS / (KC / 4));
            if (row < t.rows) xv[i].load(job.x + order[row] * job.pitch + c0 + x_col, (int)min((uint64_t)4, c_end - min(c_end, c0 + x_col)), job.x_wide);
        }
#pragma unroll
        for (uint32_t i = 0; i < WU; i++) {
            const uint32_t u = tid + i * THREADS;
            if (job.w.wide) {
                const uint32_t r = u / (KC / 4);
                const uint64_t c = c0 + u % (KC / 4) * 4;
                wv[i].load(w + r * width + c, r < rank ? (int)min((uint64_t)4, c_end - min(c_end, c)) : 0, job.w_wide);
            } else {
                const uint64_t c = c0 + u / (RP / 4);
                const uint32_t r = u % (RP / 4) * 4;
                wv[i].load(w + c * rank + r, c < c_end ? (int)min(4u, rank - min(rank, r)) : 0, job.w_wide);
            }
        }
    };
    if (steps) fetch(c_first);
    const uint32_t idesc = idesc_of(TM, RP, false, !job.w.wide);
    for (uint32_t s = 0; s < steps; s++) {
        const uint32_t at = base + M::STAGES_AT + (s & 1) * M::STAGE, wat = at + M::X::BYTES;
        if (s >= 2) bar_wait(base + 8 * (s & 1), (s / 2 - 1) & 1, a.status);
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) {
            const uint32_t row = x_row + i * (THREADS / (KC / 4));
            if (row < t.rows) xv[i].put(at + M::X::at(row, x_col), M::X::PLANE);
        }
#pragma unroll
        for (uint32_t i = 0; i < WU; i++) {
            const uint32_t u = tid + i * THREADS;
            if (job.w.wide) wv[i].put(wat + M::WideW::at(u / (KC / 4), u % (KC / 4) * 4), M::WideW::PLANE);
            else wv[i].put(wat + M::TallW::at(u / (RP / 4), u % (RP / 4) * 4), M::TallW::PLANE);
        }
        if (s + 1 < steps) fetch(c_first + (uint64_t)(s + 1) * KC);
        fence_async();
        __syncthreads();
        if (warp == 0) {
            tc_after();
            const uint32_t leader = elect();                 // the thread whose products the commit answers for
            if (job.w.wide) step_mma<typename M::X, typename M::WideW, 3, M::WP, false, false, Sums<RP>::MAINS>(tmem, RP, tmem + Sums<RP>::SIDE, at, wat, idesc, KC / 16, s == 0, leader);
            else step_mma<typename M::X, typename M::TallW, 3, M::WP, false, true, Sums<RP>::MAINS>(tmem, RP, tmem + Sums<RP>::SIDE, at, wat, idesc, KC / 16, s == 0, leader);
            if (leader) tc_commit(base + 8 * (s & 1));
        }
    }
    if (steps) bar_wait(base + 8 * ((steps - 1) & 1), ((steps - 1) / 2) & 1, a.status);
    tc_after();
    // accumulators to shared memory, summed over the cluster's CTAs in their order, scaled, cut and stored
    float *acc = (float *)(smem + M::STAGES_AT);
    for (uint32_t c = (warp >> 2) * 16; c < RP; c += 32) {
        float v[16];
        load_sum<RP, Sums<RP>::MAINS>(tmem + ((warp & 3) << 21) + c, v);
        float *row = acc + ((warp & 3) * 32 + lane) * M::PITCH + c;
#pragma unroll
        for (int i = 0; i < 16; i += 4) *(float4 *)(row + i) = steps ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_float4(0, 0, 0, 0);
    }
    tc_before();
    cluster.sync();
    tc_after();
    if (warp == 0) tc_free(tmem, M::COLS);
    const float scale = a.scale ? a.scale[t.slot] : 1.0f;
    const uint32_t rows = TM / parts;
    for (uint32_t u = tid; u < rows * (RP / 4); u += THREADS) {
        const uint32_t row = part * rows + u / (RP / 4), c = u % (RP / 4) * 4;
        if (row >= t.rows) break;
        float4 sum = make_float4(0, 0, 0, 0);
        for (uint32_t p = 0; p < parts; p++) {
            const float4 v = *(const float4 *)(cluster.map_shared_rank(acc, p) + row * M::PITCH + c);
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        sum.x *= scale; sum.y *= scale; sum.z *= scale; sum.w *= scale;
#pragma unroll
        for (int p = 0; p < 3; p++) {
            const uint32_t lo = cut2(sum.x, sum.y), hi = cut2(sum.z, sum.w);
            *(uint2 *)(job.planes + p * a.plane + (uint64_t)(t.first + row) * RP + c) = make_uint2(lo, hi);
        }
    }
    cluster.sync();                                          // nobody leaves while its sums are read
}

// ---- expand -----------------------------------------------------------------------------------------------------------------
template <typename W> struct ExpandArgs {
    Mat<W> w;
    bool w_wide;
    const __nv_bfloat16 *planes;                             // [3][rows][RP], of shrink
    uint64_t plane;
    Lists lists;
    uint32_t slots, blocks;                                  // blocks of 128 columns per CTA
    const float *base;
    uint64_t base_pitch;
    float *y;
    uint64_t y_pitch;
    uint32_t *status;
};
template <typename W, uint32_t RP> struct ExpandMap {
    static constexpr int WP = Four<W>::PLANES;
    using H = Tile<TM, RP, 3>;                               // rows tokens: K-major
    using TallW = Tile<128, RP, WP>;                         // rows of the wide axis: K-major
    using WideW = Tile<RP, 128, WP>;                         // rows r: MN-major
    static constexpr uint32_t W_BYTES = WideW::BYTES > TallW::BYTES ? WideW::BYTES : TallW::BYTES;
    static constexpr uint32_t ORDER = 64, H_AT = ORDER + TM * 4, W_AT = H_AT + ((H::BYTES + 15) & ~15u), NEED = W_AT + W_BYTES;
    // Never more than four CTAs on an SM, which have its 512 columns of TMEM: a fifth would hold its place waiting for columns (233472
    // bytes of shared memory to an SM, 1024 of them the system's for each CTA).
    static constexpr uint32_t TOTAL = NEED < 46080 ? 46080 : NEED;
    static_assert(5 * (TOTAL + 1024) > 233472 && TM == 128, "at most four CTAs of 128 TMEM columns");
};

// Columns of the projection are the accumulator's lanes and tokens its columns, so that a warp's 32 lanes hold 32 neighbouring values
// of a token's row.
template <typename W, uint32_t RP>
__global__ void __launch_bounds__(THREADS) adapter_expand_kernel(const __grid_constant__ ExpandArgs<W> a) {
    using M = ExpandMap<W, RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    uint32_t *order = (uint32_t *)(smem + M::ORDER);
    grid_wait();
    grid_go();
    if (blockIdx.y >= *a.lists.n_tiles) return;
    const ATile t = a.lists.tiles[blockIdx.y];
    const bool none = t.slot >= a.slots;
    if (none && a.base == a.y) return;
    const uint64_t width = a.w.width;
    const uint32_t rank = a.w.rank;
    const uint32_t first = blockIdx.x * a.blocks, last = (uint32_t)min((width + 127) / 128, (uint64_t)first + a.blocks);
    if (tid == 0) bar_init(base);
    if (warp == 0) tc_alloc(base + 32, TM);
    if (tid < TM) order[tid] = tid < t.rows ? a.lists.order[t.first + tid] : 0;
    const W *w = a.w.p + t.slot * a.w.slot;
    constexpr uint32_t WU = RP * 128 / 4 / THREADS;
    Four<W> wv[WU];
    auto fetch = [&](uint32_t block) {
        const uint64_t c0 = (uint64_t)block * 128;
#pragma unroll
        for (uint32_t i = 0; i < WU; i++) {
            const uint32_t u = tid + i * THREADS;
            if (a.w.wide) {
                const uint32_t r = u / 32;
                const uint64_t c = c0 + u % 32 * 4;
                wv[i].load(w + r * width + c, r < rank ? (int)min((uint64_t)4, width - min(width, c)) : 0, a.w_wide);
            } else {
                const uint64_t c = c0 + u / (RP / 4);
                const uint32_t r = u % (RP / 4) * 4;
                wv[i].load(w + c * rank + r, c < width ? (int)min(4u, rank - min(rank, r)) : 0, a.w_wide);
            }
        }
    };
    const uint32_t n = (t.rows + 15) & ~15u;
    if (!none) {
        fetch(first);
        for (uint32_t u = tid; u < 3 * t.rows * (RP / 8); u += THREADS) {
            const uint32_t p = u / (t.rows * (RP / 8)), v = u % (t.rows * (RP / 8)), row = v / (RP / 8), c = v % (RP / 8) * 8;
            put16(base + M::H_AT + p * M::H::PLANE + M::H::at(row, c), *(const uint4 *)(a.planes + p * a.plane + (uint64_t)(t.first + row) * RP + c));
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *(volatile uint32_t *)(smem + 32);
    const uint32_t idesc = idesc_of(128, n, a.w.wide, false);
    for (uint32_t block = first; block < last; block++) {
        if (!none) {
#pragma unroll
            for (uint32_t i = 0; i < WU; i++) {
                const uint32_t u = tid + i * THREADS;
                if (a.w.wide) wv[i].put(base + M::W_AT + M::WideW::at(u / 32, u % 32 * 4), M::WideW::PLANE);
                else wv[i].put(base + M::W_AT + M::TallW::at(u / (RP / 4), u % (RP / 4) * 4), M::TallW::PLANE);
            }
            if (block + 1 < last) fetch(block + 1);
            fence_async();
            tc_before();
            __syncthreads();
            if (warp == 0) {
                tc_after();
                const uint32_t leader = elect();
                if (a.w.wide) step_mma<typename M::WideW, typename M::H, M::WP, 3, true, false, 1>(tmem, 0, tmem, base + M::W_AT, base + M::H_AT, idesc, RP / 16, true, leader);
                else step_mma<typename M::TallW, typename M::H, M::WP, 3, false, false, 1>(tmem, 0, tmem, base + M::W_AT, base + M::H_AT, idesc, RP / 16, true, leader);
                if (leader) tc_commit(base);
            }
        }
        const uint64_t c = (uint64_t)block * 128 + (warp & 3) * 32 + lane;
        const bool mine = c < width;
        const uint32_t t_first = (warp >> 2) * 64, t_last = min(t.rows, t_first + 64);
        bool waited = none;
        for (uint32_t j = t_first; j < t_last; j += 16) {
            float b[16], v[16];
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) b[i] = a.base && mine && j + i < t_last ? a.base[order[j + i] * a.base_pitch + c] : 0.0f;
            if (!waited) { bar_wait(base, (block - first) & 1, a.status); tc_after(); waited = true; }
            if (!none) tc_load16(tmem + ((warp & 3) << 21) + j, v);
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) if (mine && j + i < t_last) a.y[order[j + i] * a.y_pitch + c] = none ? b[i] : b[i] + v[i];
        }
        if (!waited) bar_wait(base, (block - first) & 1, a.status);          // the tile's columns of weights are written again only then
    }
    tc_before();
    __syncthreads();
    if (warp == 0) tc_free(tmem, TM);
}

// ---- outer ------------------------------------------------------------------------------------------------------------------
struct OuterJob {
    const float *x;
    uint64_t pitch, width;
    bool x_wide;
    const __nv_bfloat16 *planes;                             // [3][rows][RP]
    float *d;                                                // [slots][rank * width]: (r, c) at r * sr + c * sc
    uint64_t sr, sc;
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
    using H = Tile<TC, RP, 3>;                               // rows tokens: MN-major
    static constexpr uint32_t STAGE = (X::BYTES + H::BYTES + 15) & ~15u, STAGES_AT = 64;
    static constexpr uint32_t PITCH = 129;                   // floats per r of the exchanged accumulators
    static constexpr uint32_t ACC = RP * PITCH * 4;
    static constexpr uint32_t TOTAL = STAGES_AT + (2 * STAGE > ACC ? 2 * STAGE : ACC);
    static constexpr uint32_t COLS = Sums<RP>::COLS;
};

template <uint32_t RP>
__global__ void __launch_bounds__(THREADS) adapter_outer_kernel(const __grid_constant__ OuterArgs a) {
    namespace cg = cooperative_groups;
    using M = OuterMap<RP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = smem_u32(smem);
    cg::cluster_group cluster = cg::this_cluster();          // a slot's tokens, a run to each CTA
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank(), slot = blockIdx.z;
    const bool second = blockIdx.y >= a.job[0].blocks;
    const OuterJob &job = a.job[second];
    const uint64_t c0 = (uint64_t)(blockIdx.y - (second ? a.job[0].blocks : 0)) * 128;
    grid_wait();
    grid_go();
    const uint32_t begin = a.lists.offsets[slot], tokens = a.lists.offsets[slot + 1] - begin;
    const uint32_t cols = (uint32_t)min((uint64_t)128, job.width - c0);
    float *d = job.d + slot * (a.rank * job.width) + c0 * job.sc;
    if (!tokens) {
        for (uint32_t u = part * THREADS + tid; u < a.rank * cols; u += parts * THREADS)
            d[job.sc == 1 ? u / cols * job.sr + u % cols : u % a.rank * job.sr + u / a.rank * job.sc] = 0;
        return;                                              // the same for all CTAs of the cluster
    }
    if (tid < 2) bar_init(base + 8 * tid);
    if (warp == 0) tc_alloc(base + 32, M::COLS);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *(volatile uint32_t *)(smem + 32);
    const uint32_t per = ((tokens + parts - 1) / parts + TC - 1) / TC * TC, from = min(tokens, part * per), to = min(tokens, from + per);
    const uint32_t steps = (to - from + TC - 1) / TC;
    constexpr uint32_t XU = TC * 128 / 4 / THREADS, HU = (3 * TC * RP / 8 + THREADS - 1) / THREADS;
    Four<float> xv[XU];
    uint4 hv[HU];
    const uint32_t x_row = tid / 32, x_col = lane * 4;
    auto fetch = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) {
            const uint32_t t = t0 + x_row + i * 8;
            const int valid = t < to ? (int)cols - (int)x_col : 0;
            xv[i].load(valid > 0 ? job.x + a.lists.order[begin + t] * job.pitch + c0 + x_col : nullptr, valid, job.x_wide);
        }
#pragma unroll
        for (uint32_t i = 0; i < HU; i++) {
            const uint32_t u = tid + i * THREADS, p = u / (TC * RP / 8), v = u % (TC * RP / 8), t = t0 + v / (RP / 8);
            hv[i] = p < 3 && t < to ? *(const uint4 *)(job.planes + p * a.plane + (uint64_t)(begin + t) * RP + v % (RP / 8) * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    if (steps) fetch(from);
    constexpr uint32_t idesc = idesc_of(128, RP, true, true);
    for (uint32_t s = 0; s < steps; s++) {
        const uint32_t at = base + M::STAGES_AT + (s & 1) * M::STAGE, hat = at + M::X::BYTES;
        if (s >= 2) bar_wait(base + 8 * (s & 1), (s / 2 - 1) & 1, a.status);
#pragma unroll
        for (uint32_t i = 0; i < XU; i++) xv[i].put(at + M::X::at(x_row + i * 8, x_col), M::X::PLANE);
#pragma unroll
        for (uint32_t i = 0; i < HU; i++) {
            const uint32_t u = tid + i * THREADS, p = u / (TC * RP / 8), v = u % (TC * RP / 8);
            if (p < 3) put16(hat + p * M::H::PLANE + M::H::at(v / (RP / 8), v % (RP / 8) * 8), hv[i]);
        }
        if (s + 1 < steps) fetch(from + (s + 1) * TC);
        fence_async();
        __syncthreads();
        if (warp == 0) {
            tc_after();
            const uint32_t leader = elect();
            step_mma<typename M::X, typename M::H, 3, 3, true, true, Sums<RP>::MAINS>(tmem, RP, tmem + Sums<RP>::SIDE, at, hat, idesc, TC / 16, s == 0, leader);
            if (leader) tc_commit(base + 8 * (s & 1));
        }
    }
    if (steps) bar_wait(base + 8 * ((steps - 1) & 1), ((steps - 1) / 2) & 1, a.status);
    tc_after();
    float *acc = (float *)(smem + M::STAGES_AT);
    for (uint32_t c = (warp >> 2) * 16; c < RP; c += 32) {
        float v[16];
        load_sum<RP, Sums<RP>::MAINS>(tmem + ((warp & 3) << 21) + c, v);
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) acc[(c + i) * M::PITCH + (warp & 3) * 32 + lane] = steps ? v[i] : 0.0f;
    }
    tc_before();
    cluster.sync();
    tc_after();
    if (warp == 0) tc_free(tmem, M::COLS);
    for (uint32_t u = part * THREADS + tid; u < a.rank * cols; u += parts * THREADS) {
        const uint32_t r = job.sc == 1 ? u / cols : u % a.rank, c = job.sc == 1 ? u % cols : u / a.rank;
        float sum = 0;
        for (uint32_t p = 0; p < parts; p++) sum += cluster.map_shared_rank(acc, p)[r * M::PITCH + c];
        d[r * job.sr + c * job.sc] = sum;
    }
    cluster.sync();
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
    s.scale = ad->scale; s.status = tune->status; s.plane = (uint64_t)T * s.RP; s.stream = stream;
    return launch(adapter_lists_kernel, "adapter_lists_kernel", dim3(1), 1024, (size_t)32 * (s.S + 1) * 4, 0, false, stream, slots, s.T, s.S, tune->order,
                  tune->offsets, (ATile *)tune->tiles, tune->n_tiles, tune->status);
}

// As many CTAs to a tile as give every SM two, a run of 128 columns each at least.
uint32_t cluster_of(uint64_t items, uint64_t length, uint32_t least) {
    uint32_t c = 1;
    while (c < 8 && items * c < 2 * SMS && length / (2 * c) >= least) c *= 2;
    return c;
}

template <typename W, uint32_t RP>
int shrink(const ShrinkJob<W> *jobs, uint32_t n, const Shape &s) {
    ShrinkArgs<W> a = {};
    uint64_t width = 0;
    for (uint32_t i = 0; i < n; i++) { a.job[i] = jobs[i]; if (jobs[i].w.width > width) width = jobs[i].w.width; }
    a.lists = s.lists; a.scale = s.scale; a.plane = s.plane; a.slots = s.S; a.status = s.status;
    const uint32_t c = cluster_of((uint64_t)(s.T + TM - 1) / TM * n, width, 128);
    return launch(adapter_shrink_kernel<W, RP>, "adapter_shrink_kernel", dim3(c, s.tiles, n), THREADS, ShrinkMap<W, RP>::TOTAL, c, true, s.stream, a);
}
template <typename W, uint32_t RP>
int expand(const Mat<W> &w, bool w_wide, const __nv_bfloat16 *planes, const float *base, size_t base_pitch, float *y, size_t y_pitch, const Shape &s) {
    ExpandArgs<W> a = {w, w_wide, planes, s.plane, s.lists, s.S, 1, base, base_pitch, y, y_pitch, s.status};
    const uint64_t blocks = (w.width + 127) / 128, tiles = (s.T + TM - 1) / TM;
    a.blocks = (uint32_t)((blocks * tiles + 3 * SMS - 1) / (3 * SMS));
    if (a.blocks > blocks) a.blocks = (uint32_t)blocks;
    return launch(adapter_expand_kernel<W, RP>, "adapter_expand_kernel", dim3((unsigned)((blocks + a.blocks - 1) / a.blocks), s.tiles), THREADS,
                  ExpandMap<W, RP>::TOTAL, 0, true, s.stream, a);
}
template <uint32_t RP>
int outer(const OuterJob *jobs, const Shape &s) {
    OuterArgs a = {{jobs[0], jobs[1]}, s.lists, s.plane, s.R, s.status};
    const uint32_t blocks = jobs[0].blocks + jobs[1].blocks;
    const uint32_t c = cluster_of(blocks, s.T, TC);
    return launch(adapter_outer_kernel<RP>, "adapter_outer_kernel", dim3(c, blocks, s.S), THREADS, OuterMap<RP>::TOTAL, c, true, s.stream, a);
}

template <typename W> Mat<W> mat_a(const QW4CuAdapters *ad) { return {(const W *)ad->a, ad->rank * ad->k, ad->rank, ad->k, true}; }
template <typename W> Mat<W> mat_b(const QW4CuAdapters *ad) { return {(const W *)ad->b, ad->rank * ad->n, ad->rank, ad->n, false}; }
template <typename W> bool wide_a(const QW4CuAdapters *ad) { return fours(ad->a, ad->k, sizeof(W)); }
template <typename W> bool wide_b(const QW4CuAdapters *ad) { return fours(ad->b, ad->rank, sizeof(W)); }

struct Rows { const float *p; size_t pitch; };

template <typename W, uint32_t RP>
int forward(const QW4ShTune *tune, const QW4CuAdapters *ad, Rows x, Rows base, float *y, size_t y_pitch, const Shape &s) {
    const ShrinkJob<W> job = {mat_a<W>(ad), x.p, x.pitch, fours(x.p, x.pitch, 4), wide_a<W>(ad), (__nv_bfloat16 *)tune->h};
    if (const int rc = shrink<W, RP>(&job, 1, s)) return rc;
    return expand<W, RP>(mat_b<W>(ad), wide_b<W>(ad), job.planes, base.p, base.pitch, y, y_pitch, s);
}
template <typename W, uint32_t RP>
int backward(const QW4ShTune *tune, const QW4CuAdapters *ad, Rows x, Rows dy, Rows base, float *dx, size_t dx_pitch, float *da, float *db, const Shape &s) {
    const ShrinkJob<W> jobs[2] = {{mat_b<W>(ad), dy.p, dy.pitch, fours(dy.p, dy.pitch, 4), wide_b<W>(ad), (__nv_bfloat16 *)tune->g},
                                  {mat_a<W>(ad), x.p, x.pitch, fours(x.p, x.pitch, 4), wide_a<W>(ad), (__nv_bfloat16 *)tune->h}};
    int rc;
    if ((rc = shrink<W, RP>(jobs, da ? 2 : 1, s))) return rc;
    if (dx && (rc = expand<W, RP>(mat_a<W>(ad), wide_a<W>(ad), jobs[0].planes, base.p, base.pitch, dx, dx_pitch, s))) return rc;
    if (!da) return 0;
    const OuterJob outers[2] = {{x.p, x.pitch, ad->k, jobs[1].x_wide, jobs[0].planes, da, ad->k, 1, (uint32_t)((ad->k + 127) / 128)},
                                {dy.p, dy.pitch, ad->n, jobs[0].x_wide, jobs[1].planes, db, 1, ad->rank, (uint32_t)((ad->n + 127) / 128)}};
    return outer<RP>(outers, s);
}

#define BY_RANK(f, W, ...) (s.RP == 16 ? f<W, 16>(__VA_ARGS__) : s.RP == 32 ? f<W, 32>(__VA_ARGS__) : s.RP == 64 ? f<W, 64>(__VA_ARGS__) : f<W, 128>(__VA_ARGS__))
#define BY_TYPE(f, ...) (ad->type == 0 ? BY_RANK(f, float, __VA_ARGS__) : ad->type == 1 ? BY_RANK(f, __half, __VA_ARGS__) : BY_RANK(f, __nv_bfloat16, __VA_ARGS__))

}  // namespace

extern "C" uint32_t qw4sh_adapter_rank(uint32_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }
// Most tiles that there can be: a token in each group, and then whole tiles.
extern "C" size_t qw4sh_adapter_tiles(size_t tokens, uint32_t slots) {
    const size_t groups = tokens < slots + 1u ? tokens : slots + 1u;
    return (tokens - groups) / TM + groups;
}

extern "C" int qw4sh_adapter_forward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                                     const float *base, size_t base_pitch, float *y, size_t y_pitch, size_t tokens, void *stream) {
    Shape s;
    if (const int rc = make_lists(tune, ad, slots, tokens, (cudaStream_t)stream, s)) return rc;
    const Rows xr = {x, x_pitch}, br = {base, base_pitch};
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
