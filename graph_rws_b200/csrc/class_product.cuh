// Dense products on the 5th-generation tensor cores for the linear classifier's loss: A [M, K] B [K, N] with fp16 or bf16
// operands, fp32 accumulators in tensor memory and an epilogue per use (scores to statistics, scores to gradients, sums to
// an output), fed by TMA.
//
// Operands lie in memory with either axis contiguous: tiles of an operand whose inner axis K is contiguous are 128-byte
// swizzled rows of 64 elements of K; of one whose outer axis is contiguous, 64 x 64 pieces of 64 outer elements a line.  Both
// are read by the MMA as they are, so that no operand is ever transposed in memory.
//
// fp32 operands come as three bf16 planes (x = hi + mid + lo exactly to 24 bits): six products, hi hi, hi mid, mid hi, mid mid,
// hi lo, lo hi.  What is left out (mid lo and below) is 2^-24 of a product.  The tensor cores cut every sum off towards zero,
// so these sums are kept short: the five small pairs have an accumulator of their own, hi hi one for every two steps of the
// inner axis, and the epilogue adds them up in registers, rounding to nearest.  An infinite operand has planes of 0, and so has
// most of what it is multiplied with: where hi hi is not finite, it is the result, and the small pairs (inf 0) are left
// out.  Tiles have 128 columns, so that two of each
// accumulator fit and a thread's 64 sums stay in registers; a stage is one plane of both operands, which all products that
// need it read from where it lies.
//
// A persistent CTA (or a pair of CTAs that share the tile's columns, CG = 2) owns output tiles of 128 CG x up to 256; two
// accumulators alternate, so the epilogue of one tile runs under the MMAs of the next.  Warps: 0-7 epilogue (warp % 4
// is the quarter of tensor memory, warp / 4 takes every second 64 columns), 8 TMA, 9 MMA.  All waits are bounded.
//
// Outputs leave through shared memory as 32-row boxes of 128-byte lines (a warp's own 4 KB) and TMA stores, which also
// clip them: rows stored from registers reach memory as 32 separate 16-byte pieces per instruction, which held the
// gradient pass of 1,024 x 512 x 32,768 at 54 us.
#pragma once

#include <cuda.h>
#include <limits.h>

#include "class_loss.cuh"

namespace grws {
namespace prod {

using namespace cls;

constexpr int BM = 128, BK = 64;                    // rows per CTA, inner elements per stage
// How a product's sums are held.  WHOLE: the inner axis in one accumulator.  PLANES3: operands of three planes, as above.  CHAINS:
// 16-bit scores of wide rows, whose sum is taken off the tensor cores every CHAIN_STEPS steps; 128-column tiles for the
// same reason, two accumulators that take the chains in turn.
enum Kind : int { WHOLE = 0, PLANES3 = 1, CHAINS = 2 };
constexpr int tile_width(int kind) { return kind == WHOLE ? 256 : 128; }            // columns per tile at most
constexpr int MAX_STAGES = 8, SMEM_BYTES = 231936;        // 227 KB less what the barriers take
constexpr int EPILOGUE_WARPS = 8, TMA_WARP = 8, MMA_WARP = 9, THREADS = 320;
constexpr long long WAIT_LIMIT_CYCLES = 3000000000ll;   // about 1.5 to 2.5 s of SM clocks
constexpr int MAX_TASKS = 2;
constexpr int PIECE_BYTES = 64 * BK * 2;                // 64 of the outer axis of an operand: what one copy brings of B
constexpr int SUB_STEPS = 2;                            // PLANES3: steps of 64 inner elements whose hi hi is summed in tensor memory
constexpr int CHAIN_STEPS = 4;                          // CHAINS: steps of 64 inner elements in a chain

template <int CG, int KIND> struct Cfg {
    static constexpr bool SPLIT = KIND == PLANES3;
    static constexpr int BN = tile_width(KIND);
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN / CG * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
    // what a warp stores at once: 32 rows of 64 16-bit or 32 fp32 numbers, or of three planes of 32
    static constexpr int BOX_BYTES = SPLIT ? 3 * 32 * 64 : 32 * 128;
    static constexpr int STAGES = (SMEM_BYTES - 1024 - EPILOGUE_WARPS * BOX_BYTES) / STAGE_BYTES;          // (1,024: alignment of the first stage)
    static constexpr int SMEM = STAGES * STAGE_BYTES + EPILOGUE_WARPS * BOX_BYTES + 1024;
    static_assert(STAGES <= MAX_STAGES && STAGES >= 4, "stages");
};

enum Mode : int { STATS = 0, GRAD = 1, SUM = 2 };

// status codes: which wait ran out
enum : int { WAIT_OPERANDS = 1, WAIT_STAGE = 2, WAIT_ACCUMULATOR = 3, WAIT_TILE = 4 };

struct Task {
    int m_tiles, n_tiles, run, runs;      // a unit is one m tile and `run` n tiles
    int splits, k_blocks, k_len;          // parts of the inner axis, 64-element blocks in all and per part
    int bn;                               // columns per tile: a multiple of 64, or all of them in 32s
    int group;                            // m tiles side by side in the order of the units
    int a_outer, b_outer;                 // operand's outer axis contiguous
    int b_row0, b_k0;                     // first column / inner element of B within its tensor map
    int64_t M, N;
    // SUM: partial sums [splits][M][] in fp32 (added to what is there if `add`), or the output rounded to the operands' type,
    // through the map of the outputs; or to `out` with rows of ldo, where these are no multiple of 16 bytes apart or `turned`
    int rounded, add;
    void *out; int64_t ldo;
    bool turned;                          // `out` takes the transpose
    __host__ __device__ int units() const { return m_tiles * runs * splits; }
};

struct Params {
    Task task[MAX_TASKS];
    int tasks;
    int deal, deal_less, deal_more;       // see Walk
    int bf16;
    // STATS, GRAD
    const void *labels; int label_bytes;
    int64_t ignore_index, V, v0;          // number of classes, first class of column 0
    float2 *part;                         // STATS: [2 runs][M]
    float *label_score;                   // STATS: [M]
    int *done;                            // STATS: set to 0 for the kernel behind
    const float2 *state;
    int reduction;
    const float *grad, *count, *norm;
    float scale;                          // GRAD: power of two that keeps G within its type; SUM: its inverse
    int *status;
    long long wait_limit;
#ifdef GRWS_TC5_PROFILING
    int withhold;                         // self-test: stages that the first CTA fills before it stops filling (0: all)
#endif
};

struct alignas(64) Maps { CUtensorMap a[MAX_TASKS], b[MAX_TASKS], c[MAX_TASKS]; };       // operands, output

// ---------------------------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// address in the cluster's shared memory of what lies at `addr` in CTA `rank`
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    // (nothing but tensor memory is handed over, which tcgen05.fence orders: a release of the cluster's scope costs a
    // memory barrier per tile and warp)
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// bounded wait: gives up after `limit` SM clocks, or when another role of the CTA has
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, long long limit) {
    if (mbar_try_wait(bar, parity)) return true;
    long long t0 = 0;
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u) {
            if (*abort_flag) return false;
            const long long now = clock64();
            if (t0 == 0) t0 = now;
            if (now - t0 > limit) return false;
        }
    }
}
// the same wherever another role has given up already
__device__ __forceinline__ bool mbar_wait_drain(uint32_t bar, uint32_t parity, long long limit) {
    const long long t0 = clock64();
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u && clock64() - t0 > limit) return false;
    }
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
template <int CG> __device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// box of shared memory to its place in the output (what lies outside is dropped), or added to it
__device__ __forceinline__ void tma_store(const CUtensorMap *map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_add(const CUtensorMap *map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t smem_dst) {
    if constexpr (CG == 1) asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_dst) : "memory");
    else asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_dst) : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_relinquish() {
    if constexpr (CG == 1) asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    else asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
template <int CG> __device__ __forceinline__ void tmem_dealloc(uint32_t taddr) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int CG> __device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on `bar` (in both CTAs of a pair) when the MMAs issued so far have finished
template <int CG> __device__ __forceinline__ void umma_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// what was loaded is used behind this point only: the compiler sees no tie between the wait and the registers
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                      "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                      "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]));
    asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}

// shared-memory matrix descriptor, 128-byte swizzle.  Inner axis contiguous: 8-row groups 1,024 bytes apart, a step of 16
// inner elements is 32 bytes.  Outer axis contiguous: 64-element pieces of it `lbo` apart, groups of 8 inner elements 1,024
// bytes apart, a step of 16 inner elements is 2,048 bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, int outer) {
    const uint64_t lbo = outer ? (64 * BK * 2) >> 4 : 1, sbo = 1024 >> 4;
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (lbo << 16) | (sbo << 32) | (1ull << 46) | (2ull << 61);
}

// ---------------------------------------------------------------------------------------------
// order of the units: groups of `group` m tiles, within a group the n runs one after the other, so that the CTAs at work share
// the columns of B; parts of the inner axis outermost
// ---------------------------------------------------------------------------------------------
// columns that the MMA computes of a tile: the last one's in 32s (other tiles are multiples of 64, so that no box of 64 reaches
// into the next tile)
__device__ __forceinline__ int tile_columns(const Task &t, int n) { return (int)min((int64_t)t.bn, (t.N - (int64_t)n * t.bn + 31) & ~(int64_t)31); }

struct Unit { int task, m, n0, n1, split; };
__device__ __forceinline__ Unit unit_at(const Params &p, int u) {
    Unit r;
    r.task = 0;
    if (p.tasks > 1 && u >= p.task[0].units()) { u -= p.task[0].units(); r.task = 1; }
    const Task &t = p.task[r.task];
    const int per = t.m_tiles * t.runs;
    r.split = u / per;
    u -= r.split * per;
    const int g = u / (t.group * t.runs), first = g * t.group, size = min(t.group, t.m_tiles - first);
    u -= g * t.group * t.runs;
    const int run = u / size;
    r.m = first + (u - run * size);
    r.n0 = run * t.run;
    r.n1 = min(t.n_tiles, r.n0 + t.run);
    return r;
}

// The units of one CTA (pair) in order: every `ctas`-th one; or, where `deal` is set, every ctas-th of the first task and then
// of the second as many as leave all busy equally long: CTAs with one unit less of the first start on them `early` rounds sooner.
struct Walk {
    int u, step, left, end, phase, units, ctas, cta, many, early, rounds, second;
    __device__ __forceinline__ Walk(const Params &p, int all, int first, int n) : u(first - n), step(n), left(INT_MAX), end(all), phase(2), units(all), ctas(n),
                                                                                 cta(first), many(0), early(0), rounds(0), second(0) {
        if (!p.deal) return;
        end = second = p.task[0].units();
        phase = 0;
        many = end % n;                                     // CTAs that have one unit more of the first task
        early = p.deal_more - p.deal_less;
        rounds = p.deal_less;
    }
    __device__ __forceinline__ bool next() {
        for (;;) {
            if (left > 0) {
                --left;
                u += step;
                if (u < end) return true;
            }
            if (phase == 2) return false;
            const int others = ctas - many;
            if (phase++ == 0) { step = others; left = cta >= many ? early : 0; u = second + cta - many - step; }
            else { step = ctas; left = rounds; u = second + early * others + cta - step; }
            end = units;
        }
    }
};

struct Shared {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2], big_full[2], big_empty[2];
    uint32_t tmem;
    int abort_flag;
};

__device__ __forceinline__ void give_up(Shared *ss, const Params &p, int code) {
    ss->abort_flag = 1;
    if (p.status) atomicMax(p.status, code);
}

// a row's own factor: 0 for an ignored row, NaN for a label that is no class; and the factor of all rows
template <typename P> __device__ __forceinline__ float grad_row_factor(const P &p, int64_t row, int64_t label) {
    if (label == p.ignore_index) return 0.0f;
    if (label < 0 || label >= p.V) return NAN;
    if (p.reduction != RED_NONE) return 1.0f;
    const float norm = *p.norm, g = p.grad[row];
    return norm > 0.0f ? g / norm : g;
}
template <typename P> __device__ __forceinline__ float grad_alpha(const P &p) {
    if (p.reduction != RED_NONE) return loss_factor(p.grad, p.count, p.reduction);
    const float norm = *p.norm;
    return norm > 0.0f ? norm : 1.0f;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// v as three bf16 numbers: of a value past bf16's largest number (fp32's lowest, as a mask, is one) the first takes that number
// and the others the rest; what is not finite goes into the first alone
__device__ __forceinline__ void split3(float v, float &a, float &b, float &c) {
    constexpr float MOST = 3.3895313892515355e38f;          // (2 - 2^-7) 2^127
    const bool fin = fabsf(v) < INFINITY;
    a = __bfloat162float(__float2bfloat16_rn(fin ? fminf(fmaxf(v, -MOST), MOST) : v));
    const float r = fin ? v - a : 0.0f;
    b = __bfloat162float(__float2bfloat16_rn(r));
    c = r - b;
}

template <int CG, int MODE, int KIND> __global__ void __launch_bounds__(THREADS, 1) product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    using C = Cfg<CG, KIND>;
    constexpr bool SPLIT = C::SPLIT;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared shared;
    Shared *ss = &shared;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;      // (the same offset in both CTAs of a pair)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const int first = blockIdx.x / CG, stride = gridDim.x / CG;
    int units = p.task[0].units();
    if (p.tasks > 1) units += p.task[1].units();
    const long long limit = p.wait_limit;
    volatile int *abort_flag = &ss->abort_flag;

    if (threadIdx.x == 0) {
        ss->abort_flag = 0;
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(smem_u32(&ss->full[i]), 1); mbar_init(smem_u32(&ss->empty[i]), 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ss->acc_full[i]), 1); mbar_init(smem_u32(&ss->acc_empty[i]), EPILOGUE_WARPS * CG);
            mbar_init(smem_u32(&ss->big_full[i]), 1); mbar_init(smem_u32(&ss->big_empty[i]), EPILOGUE_WARPS * CG);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TMA_WARP && lane < p.tasks) {
        prefetch_map(&maps.a[lane]);
        prefetch_map(&maps.b[lane]);
    }
    if (warp == MMA_WARP) {
        tmem_alloc<CG>(smem_u32(&ss->tmem));
        tmem_relinquish<CG>();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&ss->tmem);
    wait_for_previous();
    let_next_start();
    if (MODE == STATS && blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;

    if (warp == TMA_WARP) {
        if (elect_one()) {
            // the pair's copies all count on the barriers of its first CTA, whose MMA warp issues for both.  (This thread's
            // instructions between a stage's release and its copies are time in which nothing is on the way.)
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            uint32_t full0 = smem_u32(&ss->full[0]);
            if constexpr (CG == 2) full0 = map_to_rank(full0, 0);
            constexpr int B_PIECES = C::BN / CG / 64, PLANES = SPLIT ? 3 : 1;
            for (Walk walk(p, units, first, stride); ok && walk.next();) {
                const Unit w = unit_at(p, walk.u);
                const Task &t = p.task[w.task];
                const CUtensorMap *ma = &maps.a[w.task], *mb = &maps.b[w.task];
                const int k0 = w.split * t.k_len, k1 = min(t.k_blocks, k0 + t.k_len), b_k0 = t.b_k0;
                const int a_row = (w.m * CG + (int)rank) * BM;
                const bool a_outer = t.a_outer, b_outer = t.b_outer;
                for (int n = w.n0; ok && n < w.n1; ++n) {
                    const int cols = tile_columns(t, n) / CG, b_row = t.b_row0 + n * t.bn + (int)rank * cols;
                    const int pieces = b_outer ? (cols + 63) >> 6 : B_PIECES;
                    const uint32_t bytes = CG * (C::A_BYTES + pieces * PIECE_BYTES);
                    for (int kb = k0; ok && kb < k1; ++kb) {
                        for (int plane = 0; plane < PLANES; ++plane) {
#ifdef GRWS_TC5_PROFILING
                            if (p.withhold > 0 && blockIdx.x == 0 && issued == p.withhold) { ok = false; break; }
#endif
                            if (!mbar_wait(smem_u32(&ss->empty[stage]), phase ^ 1u, abort_flag, limit)) { give_up(ss, p, WAIT_STAGE); ok = false; break; }
                            const uint32_t bar = full0 + stage * 8, a = ring + stage * C::STAGE_BYTES, b = a + C::A_BYTES;
                            const int ka = kb * BK, kB = b_k0 + ka;
                            if (rank == 0) mbar_expect_tx(smem_u32(&ss->full[stage]), bytes);
                            if (a_outer) {
#pragma unroll
                                for (int j = 0; j < BM / 64; ++j) tma_load<CG>(a + j * PIECE_BYTES, ma, bar, a_row + j * 64, ka, plane);
                            } else {
                                tma_load<CG>(a, ma, bar, ka, a_row, plane);
                            }
                            if (!b_outer) {
                                tma_load<CG>(b, mb, bar, kB, b_row, plane);
                            } else if (pieces == B_PIECES) {
#pragma unroll
                                for (int j = 0; j < B_PIECES; ++j) tma_load<CG>(b + j * PIECE_BYTES, mb, bar, b_row + j * 64, kB, plane);
                            } else {
                                for (int j = 0; j < pieces; ++j) tma_load<CG>(b + j * PIECE_BYTES, mb, bar, b_row + j * 64, kB, plane);
                            }
                            ++issued;
                            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                        }
                    }
                }
            }
            // every stage that was filled has been read (and, in a pair, the other CTA's commits have arrived here)
            // before this CTA may end
            const long long drain = ok ? limit : limit / 8;
            for (int i = 0; i < min(issued, (int)C::STAGES); ++i) {
                if (stage == 0) { stage = C::STAGES; phase ^= 1u; }
                --stage;
                if (rank == 0 && !ok) mbar_wait_drain(smem_u32(&ss->full[stage]), phase, drain);   // copies in flight
                if (ok && !mbar_wait(smem_u32(&ss->empty[stage]), phase, abort_flag, limit)) { give_up(ss, p, WAIT_STAGE); ok = false; }
            }
            if (!ok) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }          // the other CTA's copies
        }
        __syncwarp();
    } else if (warp == MMA_WARP) {
        if (rank == 0 && elect_one()) {
            int stage = 0;
            uint32_t phase = 0, tile = 0;
            [[maybe_unused]] uint32_t chain = 0;
            bool ok = true;
            for (Walk walk(p, units, first, stride); ok && walk.next();) {
                const Unit w = unit_at(p, walk.u);
                const Task &t = p.task[w.task];
                const int k0 = w.split * t.k_len, steps = min(t.k_blocks, k0 + t.k_len) - k0;
                const uint32_t idesc0 = (1u << 4) | ((uint32_t)p.bf16 << 7) | ((uint32_t)p.bf16 << 10) | ((uint32_t)t.a_outer << 15) |
                                        ((uint32_t)t.b_outer << 16) | ((uint32_t)(BM * CG >> 4) << 24);
                const uint64_t a_step = t.a_outer ? 2048 >> 4 : 32 >> 4, b_step = t.b_outer ? 2048 >> 4 : 32 >> 4;
                auto advance = [&]() { if (++stage == C::STAGES) { stage = 0; phase ^= 1u; } };
                auto wait_stage = [&](int at, uint32_t parity) {
                    if (mbar_wait(smem_u32(&ss->full[at]), parity, abort_flag, limit)) { tc_fence_after(); return true; }
                    give_up(ss, p, WAIT_OPERANDS);
                    return false;
                };
                auto wait_empty = [&](uint64_t *bar, uint32_t use) {
                    if (mbar_wait(smem_u32(&bar[use & 1u]), ((use >> 1) & 1u) ^ 1u, abort_flag, limit)) { tc_fence_after(); return true; }
                    give_up(ss, p, WAIT_ACCUMULATOR);
                    return false;
                };
                for (int n = w.n0; ok && n < w.n1; ++n, ++tile) {
                    const uint32_t idesc = idesc0 | ((uint32_t)(tile_columns(t, n) >> 3) << 17), d = tmem + (tile & 1u) * C::BN;
                    // the product of stage i's A and stage j's B; `add`: onto what is there
                    auto multiply = [&](uint32_t to, int i, int j, bool add) {
                        const uint64_t ad = smem_desc(ring + i * C::STAGE_BYTES, t.a_outer), bd = smem_desc(ring + j * C::STAGE_BYTES + C::A_BYTES, t.b_outer);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) umma<CG>(to, ad + k * a_step, bd + k * b_step, idesc, add || k > 0);
                    };
                    if constexpr (KIND != CHAINS) ok = wait_empty(ss->acc_empty, tile);
                    for (int k = 0; ok && k < steps; ++k) {
                        if constexpr (KIND == CHAINS) {
                            if (k % CHAIN_STEPS == 0 && !(ok = wait_empty(ss->big_empty, chain))) break;
                            if (!(ok = wait_stage(stage, phase))) break;
                            multiply(tmem + (chain & 1u) * C::BN, stage, stage, k % CHAIN_STEPS != 0);
                            umma_commit<CG>(smem_u32(&ss->empty[stage]));
                            advance();
                            if (k % CHAIN_STEPS == CHAIN_STEPS - 1 || k == steps - 1) { umma_commit<CG>(smem_u32(&ss->big_full[chain & 1u])); ++chain; }
                        } else if constexpr (!SPLIT) {
                            if (!(ok = wait_stage(stage, phase))) break;
                            multiply(d, stage, stage, k > 0);
                            umma_commit<CG>(smem_u32(&ss->empty[stage]));
                            advance();
                        } else {
                            const uint32_t db = tmem + 2 * C::BN + (chain & 1u) * C::BN;
                            const int hi = stage;
                            if (k % SUB_STEPS == 0 && !(ok = wait_empty(ss->big_empty, chain))) break;
                            if (!(ok = wait_stage(stage, phase))) break;
                            multiply(db, hi, hi, k % SUB_STEPS != 0);
                            advance();
                            const int mid = stage;
                            if (!(ok = wait_stage(stage, phase))) break;
                            multiply(d, hi, mid, k > 0);
                            multiply(d, mid, hi, true);
                            multiply(d, mid, mid, true);
                            advance();
                            const int lo = stage;
                            if (!(ok = wait_stage(stage, phase))) break;
                            multiply(d, hi, lo, true);
                            multiply(d, lo, hi, true);
                            advance();
                            umma_commit<CG>(smem_u32(&ss->empty[hi]));
                            umma_commit<CG>(smem_u32(&ss->empty[mid]));
                            umma_commit<CG>(smem_u32(&ss->empty[lo]));
                            if (k % SUB_STEPS == SUB_STEPS - 1 || k == steps - 1) { umma_commit<CG>(smem_u32(&ss->big_full[chain & 1u])); ++chain; }
                        }
                    }
                    if constexpr (KIND != CHAINS) {
                        if (ok) umma_commit<CG>(smem_u32(&ss->acc_full[tile & 1u]));
                    }
                }
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t box = ring + C::STAGES * C::STAGE_BYTES + warp * C::BOX_BYTES;
        uint32_t tile = 0;
        [[maybe_unused]] uint32_t chain = 0;
        bool ok = true, some = false;          // some: the warp has rows to store
        // waits for an accumulator's `use`-th sum, and gives it back
        auto wait_sum = [&](uint64_t *full, uint32_t use) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[use & 1u]), (use >> 1) & 1u, abort_flag, limit));
            if (!ok) give_up(ss, p, WAIT_TILE);
            tc_fence_after();
        };
        auto release_sum = [&](uint64_t *empty, uint32_t use) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = smem_u32(&empty[use & 1u]);
                if constexpr (CG == 2) mbar_arrive_cluster(map_to_rank(bar, 0));
                else mbar_arrive(bar);
            }
        };
        // 16 bytes of this lane's row of the box, swizzled as the store expects them
        auto put = [&](int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
            st_shared16(box + lane * 128 + ((piece ^ (lane & 7)) << 4), a, b, c, d);
        };
        auto box_free = [&]() {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
        };
        auto box_out = [&](const CUtensorMap *map, int x, int y, int z, bool add) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && some) {
                if (add) tma_add(map, box, x, y, z); else tma_store(map, box, x, y, z);
                bulk_commit();
            }
        };
        [[maybe_unused]] const float alpha = MODE == SUM ? grad_alpha(p) * p.scale : 0.0f;
        for (Walk walk(p, units, first, stride); ok && walk.next();) {
            const Unit w = unit_at(p, walk.u);
            const Task &t = p.task[w.task];
            const CUtensorMap *mc = &maps.c[w.task];
            const int row0 = (w.m * CG + (int)rank) * BM + quarter * 32;
            const int64_t row = row0 + lane;
            const bool in = row < t.M;
            some = row0 < t.M;
            [[maybe_unused]] float m = NEG_INF, s = 0.0f, factor = 0.0f, weight = 0.0f;
            [[maybe_unused]] int64_t label = -1;
            if constexpr (MODE != SUM) {
                if (in) label = load_index(p.labels, p.label_bytes, row);
            }
            if constexpr (MODE == GRAD) {
                if (in) {
                    const float2 st = p.state[row];
                    factor = grad_row_factor(p, row, label) * p.scale;
                    m = st.x;
                    weight = factor / st.y;
                }
                if (label == p.ignore_index) label = -1;
            }
            if constexpr (MODE == SUM) factor = t.rounded ? alpha : 1.0f;
            for (int n = w.n0; ok && n < w.n1; ++n) {
                const int64_t col0 = (int64_t)n * t.bn;
                const int cols = (int)min((int64_t)t.bn, t.N - col0);          // of this tile
                const int mine = (int)max((int64_t)-1, min((int64_t)C::BN, label - p.v0 - col0));    // label's column, if within
                (void)mine;
                // W columns from c on
                constexpr int W = SPLIT ? 32 : 64;
                auto put16 = [&](const float (&v)[W], uint32_t mask) {
                    if (p.bf16) {
#pragma unroll
                        for (int i = 0; i < W; i += 8)
                            put(i / 8, pack2<true>(v[i], v[i + 1]) & mask, pack2<true>(v[i + 2], v[i + 3]) & mask, pack2<true>(v[i + 4], v[i + 5]) & mask,
                                pack2<true>(v[i + 6], v[i + 7]) & mask);
                    } else {
#pragma unroll
                        for (int i = 0; i < W; i += 8)
                            put(i / 8, pack2<false>(v[i], v[i + 1]) & mask, pack2<false>(v[i + 2], v[i + 3]) & mask, pack2<false>(v[i + 4], v[i + 5]) & mask,
                                pack2<false>(v[i + 6], v[i + 7]) & mask);
                    }
                };
                auto use = [&](float (&v)[W], int c) {
                    if constexpr (MODE == STATS) {
                        if (__any_sync(0xffffffffu, mine >= c && mine < c + W)) {
                            float score = 0.0f;
#pragma unroll
                            for (int i = 0; i < W; ++i) if (mine == c + i) score = v[i];
                            if (in && mine >= c && mine < c + W && mine < cols) p.label_score[row] = score;
                        }
                        if (c + W > cols) {
#pragma unroll
                            for (int i = 0; i < W; ++i) if (c + i >= cols) v[i] = NEG_INF;
                        }
                        add_values<W>(m, s, v, LOG2E);
                    } else if constexpr (MODE == GRAD) {
                        const bool has = __any_sync(0xffffffffu, mine >= c && mine < c + W);
                        const uint64_t minus = pair2(-m, -m), cc = pair2(LOG2E, LOG2E), ww = pair2(weight, weight);
#pragma unroll
                        for (int i = 0; i < W; i += 2) unpair2(mul2(exp2_pair(v[i], v[i + 1], minus, cc), ww), v[i], v[i + 1]);
                        if (has) {
#pragma unroll
                            for (int i = 0; i < W; ++i) if (mine == c + i) v[i] -= factor;
                        }
                        box_free();
                        if constexpr (!SPLIT) {
                            // G in the operands' type, as the MMA wants both alike: dx and dw of 90,941 x 512 x 172 in bf16 are off by
                            // 1.9e-3 and 1.7e-3 of their size for it, instead of the 1.7e-3 of their own rounding
                            put16(v, factor == 0.0f ? 0u : ~0u);
                            box_out(mc, (int)col0 + c, row0, 0, false);
                        } else {
                            // the three planes: boxes of 64-byte lines, not swizzled
                            if (factor == 0.0f) {
#pragma unroll
                                for (int i = 0; i < W; ++i) v[i] = 0.0f;
                            }
#pragma unroll
                            for (int i = 0; i < W; i += 8) {
                                uint32_t q[3][4];
#pragma unroll
                                for (int j = 0; j < 8; j += 2) {
                                    float a[2], b[2], d[2];
                                    split3(v[i + j], a[0], b[0], d[0]);
                                    split3(v[i + j + 1], a[1], b[1], d[1]);
                                    q[0][j / 2] = pack2<true>(a[0], a[1]);
                                    q[1][j / 2] = pack2<true>(b[0], b[1]);
                                    q[2][j / 2] = pack2<true>(d[0], d[1]);
                                }
#pragma unroll
                                for (int k = 0; k < 3; ++k) st_shared16(box + k * 2048 + lane * 64 + i * 2, q[k][0], q[k][1], q[k][2], q[k][3]);
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0 && some) {
#pragma unroll
                                for (int k = 0; k < 3; ++k) tma_store(mc, box + k * 2048, (int)col0 + c, row0, k);
                                bulk_commit();
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < W; ++i) v[i] *= factor;
                        if (t.turned) {
                            // straight from the registers: a warp's 32 rows of one column lie side by side in `out`
                            if (!in) return;
                            const int64_t at = (col0 + c) * t.ldo + row;
                            if constexpr (SPLIT) {
                                float *o = static_cast<float *>(t.out) + at;
#pragma unroll
                                for (int i = 0; i < W; ++i, o += t.ldo) {
                                    if (c + i >= cols) break;
                                    *o = v[i];
                                }
                            } else {
                                uint16_t *o = static_cast<uint16_t *>(t.out) + at;
#pragma unroll
                                for (int i = 0; i < W; i += 2, o += 2 * t.ldo) {
                                    if (c + i >= cols) break;
                                    const uint32_t two = p.bf16 ? pack2<true>(v[i], v[i + 1]) : pack2<false>(v[i], v[i + 1]);
                                    o[0] = (uint16_t)two;
                                    if (c + i + 1 < cols) o[t.ldo] = (uint16_t)(two >> 16);
                                }
                            }
                            return;
                        }
                        if constexpr (!SPLIT) {
                            if (t.rounded) {
                                box_free();
                                put16(v, ~0u);
                                if (!t.out) { box_out(mc, (int)col0 + c, row0, 0, false); return; }
                                __syncwarp();
                                for (int r = 0; r < 32 && row0 + r < t.M; ++r) {
                                    const uint32_t two = ld_shared32(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                                    uint16_t *o = static_cast<uint16_t *>(t.out) + (row0 + r) * t.ldo + col0 + c + lane * 2;
                                    if (c + lane * 2 < cols) o[0] = (uint16_t)two;
                                    if (c + lane * 2 + 1 < cols) o[1] = (uint16_t)(two >> 16);
                                }
                                __syncwarp();
                                return;
                            }
                        }
#pragma unroll
                        for (int h = 0; h < W; h += 32) {
                            if (c + h >= cols) return;
                            box_free();
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                put(i / 4, __float_as_uint(v[h + i]), __float_as_uint(v[h + i + 1]), __float_as_uint(v[h + i + 2]), __float_as_uint(v[h + i + 3]));
                            if (!t.out) { box_out(mc, (int)col0 + c + h, row0, w.split, t.add); continue; }
                            __syncwarp();
                            for (int r = 0; r < 32 && row0 + r < t.M; ++r) {
                                const uint32_t one = ld_shared32(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                                if (c + h + lane < cols) static_cast<float *>(t.out)[(row0 + r) * t.ldo + col0 + c + h + lane] = __uint_as_float(one);
                            }
                            __syncwarp();
                        }
                    }
                };
                [[maybe_unused]] const uint32_t at = tmem + (tile & 1u) * C::BN + lanes;
                if constexpr (KIND == CHAINS) {
                    const int chains = (t.k_blocks + CHAIN_STEPS - 1) / CHAIN_STEPS, c = half * 64;
                    float acc[64];
#pragma unroll
                    for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
                    for (int sub = 0; sub < chains; ++sub, ++chain) {
                        wait_sum(ss->big_full, chain);
                        if (!ok) break;
                        if (c < cols) {
                            uint32_t r[32], r2[32];
                            const uint32_t from = tmem + (chain & 1u) * C::BN + lanes + c;
                            tmem_ld32(from, r);
                            tmem_ld32(from + 32, r2);
                            tmem_ld_wait();
                            loaded(r);
                            loaded(r2);
#pragma unroll
                            for (int i = 0; i < 32; ++i) { acc[i] += __uint_as_float(r[i]); acc[32 + i] += __uint_as_float(r2[i]); }
                        }
                        release_sum(ss->big_empty, chain);
                    }
                    if (!ok) break;
                    if (c < cols) use(acc, c);
                } else if constexpr (!SPLIT) {
                    wait_sum(ss->acc_full, tile);
                    if (!ok) break;
                    const int last = (cols - 1 - half * 64) >> 7;          // 64-column pieces of this warp, less one (-1: none)
                    if (last < 0) release_sum(ss->acc_empty, tile);
                    for (int k = 0; k <= last; ++k) {
                        const int c = half * 64 + k * 128;
                        float v[64];
                        uint32_t r[32], r2[32];
                        tmem_ld32(at + c, r);
                        tmem_ld32(at + c + 32, r2);
                        tmem_ld_wait();
                        loaded(r);
                        loaded(r2);
                        if (k == last) release_sum(ss->acc_empty, tile);
#pragma unroll
                        for (int i = 0; i < 32; ++i) { v[i] = __uint_as_float(r[i]); v[32 + i] = __uint_as_float(r2[i]); }
                        use(v, c);
                    }
                } else {
                    const int k0 = w.split * t.k_len, steps = min(t.k_blocks, k0 + t.k_len) - k0, chains = (steps + SUB_STEPS - 1) / SUB_STEPS;
                    const int c = half * 64;
                    float acc[2][W];
                    auto add_up = [&](uint32_t from, bool first, bool small) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            if (c + k * W >= cols) break;
                            uint32_t r[W];
                            tmem_ld32(from + c + k * W, r);
                            tmem_ld_wait();
                            loaded(r);
#pragma unroll
                            for (int i = 0; i < W; ++i) {
                                const float v = __uint_as_float(r[i]);
                                if (first) acc[k][i] = v;
                                else if (!small || fabsf(acc[k][i]) < INFINITY) acc[k][i] += v;
                            }
                        }
                    };
                    for (int sub = 0; sub < chains; ++sub, ++chain) {
                        wait_sum(ss->big_full, chain);
                        if (!ok) break;
                        add_up(tmem + 2 * C::BN + (chain & 1u) * C::BN + lanes, sub == 0, false);
                        release_sum(ss->big_empty, chain);
                    }
                    if (!ok) break;
                    wait_sum(ss->acc_full, tile);
                    if (!ok) break;
                    add_up(at, false, true);
                    release_sum(ss->acc_empty, tile);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (c + k * W < cols) use(acc[k], c + k * W);
                }
                ++tile;
            }
            if constexpr (MODE == STATS) {
                if (ok && in) p.part[(int64_t)((w.n0 / t.run) * 2 + half) * t.M + row] = make_float2(m, s);
            }
        }
        if (lane == 0) bulk_wait();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_dealloc<CG>(tmem);
    if constexpr (CG == 2) cluster_sync();
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
// Map of a [planes][rows][cols] matrix, cols contiguous, rows `ld` and planes `plane` elements apart; boxes of `box_cols`
// columns and `box_rows` rows, zeros outside; 128-byte swizzle where a box's line has 128 bytes.
inline int encode_map(CUtensorMap *map, const void *base, int dtype, int64_t cols, int64_t rows, int64_t ld, int planes, int64_t plane, int box_cols,
                      int box_rows) {
    typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);
    static EncodeFn encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<EncodeFn>(fn);
    }();
    if (!encode) return fail(GRWS_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t es = dtype_bytes(dtype);
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * es, (cuuint64_t)(planes > 1 ? plane : ld) * es};
    const cuuint32_t boxes[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == GRWS_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == GRWS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, type, 3, const_cast<void *>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box_cols * es == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GRWS_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return GRWS_OK;
}

template <int CG, int MODE, int KIND> static int launch_product(const Maps &maps, const Params &p, cudaStream_t st) {
    int64_t units = 0;
    for (int i = 0; i < p.tasks; ++i) units += p.task[i].units();
    const int64_t clusters = units < sm_count() / CG ? units : sm_count() / CG;
    using C = Cfg<CG, KIND>;
    static bool allowed[MAX_DEVICES];
    const int dev = current_device();
    if (dev < 0) return fail(GRWS_ERR_CUDA, "no current device");
    if (!__atomic_load_n(&allowed[dev], __ATOMIC_RELAXED)) {
        GRWS_CUDA_TRY(cudaFuncSetAttribute(product_kernel<CG, MODE, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        __atomic_store_n(&allowed[dev], true, __ATOMIC_RELAXED);
    }
    return launch_next(product_kernel<CG, MODE, KIND>, dim3((unsigned)(clusters * CG)), THREADS, C::SMEM, st, CG, maps, p);
}

}  // namespace prod
}  // namespace grws
