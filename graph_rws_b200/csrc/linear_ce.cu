// Softmax cross entropy of a linear classifier, without keeping the scores.  x [n, d], w [d, V], label y_i per row:
//
//     s_iv = sum_k x_ik w_kv      loss_i = log sum_v exp(s_iv) - s_i,y_i
//     G_iv = r_i (exp(s_iv - log sum) - [v = y_i])      dx = G w^T      dw = x^T G
//
// Forward keeps a row's maximum and sum of exponentials, nothing else.  Backward goes over the classes in pieces: the scores
// of a piece again, its G into a workspace, then the piece's part of dx and its columns of dw.
//
// r_i comes in two factors: alpha, one number for all rows, applied where dx and dw are rounded to their type, and a row's own
// factor in G, which is 1 (or 0 for an ignored row) where the loss is a mean or a sum.
#include <stdlib.h>

#include "class_product.cuh"

namespace grws {
namespace lce {

using namespace cls;

struct Problem {
    const void *x; int64_t ldx;
    const void *w; int64_t ldw;          // w(k, v) at k * ldw + v (class_major 0) or v * ldw + k (1)
    int class_major;
    const void *labels; int label_bytes;
    int64_t ignore_index;
    int64_t n, d, V;
    int dtype, reduction;
    const float2 *state;                 // [n]: maximum, sum of exponentials
    const float *grad, *count;           // backward: gradient of the loss, number of counted rows
    const float *norm;                   // backward without a reduction: largest |gradient| of a row that counts
    __host__ __device__ int64_t w_k() const { return class_major ? 1 : ldw; }
    __host__ __device__ int64_t w_v() const { return class_major ? ldw : 1; }
};

// largest finite |gradient| of a row that is not ignored: with it a row's factor is at most 1, whatever the scale of the loss
__global__ void __launch_bounds__(1024) grad_norm_kernel(const Problem p, float *norm) {
    __shared__ float red[32];
    float m = 0.0f;
    wait_for_previous();
    let_next_start();
    for (int64_t i = threadIdx.x; i < p.n; i += blockDim.x) {
        const float g = fabsf(p.grad[i]);
        if (g < INFINITY && load_index(p.labels, p.label_bytes, i) != p.ignore_index) m = fmaxf(m, g);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = red[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (threadIdx.x == 0) *norm = m;
    }
}

// Joins the parts of the rows' statistics and takes the rows' losses: GROUPS threads a row, in a fixed order.  The block that is
// done last adds the blocks' sums up; `done` was set to 0 by the kernel before.
template <int GROUPS> __global__ void __launch_bounds__(256) rows_kernel(const Problem p, const float2 *part, int parts,
                                                                         const float *label_score, float2 *__restrict__ state,
                                                                         float *__restrict__ loss, float *__restrict__ count, float2 *__restrict__ partial,
                                                                         int *__restrict__ done) {
    constexpr int ROWS = 256 / GROUPS;
    __shared__ float red[64];
    __shared__ float2 joined[GROUPS][ROWS];
    __shared__ bool last;
    const int at = threadIdx.x % ROWS, group = threadIdx.x / ROWS;
    const int64_t row = (int64_t)blockIdx.x * ROWS + at;
    float l = 0.0f, counted = 0.0f, m = NEG_INF, s = 0.0f, score = 0.0f;
    int64_t label = -1;
    wait_for_previous();
    if (row < p.n) {
        if (group == 0) {
            label = load_index(p.labels, p.label_bytes, row);
            score = label_score[row];          // (nothing was written there for a label that is no class)
        }
#pragma unroll 4
        for (int i = group; i < parts; i += GROUPS) {
            const float2 q = part[(int64_t)i * p.n + row];
            join_stats(m, s, q.x, q.y, LOG2E);
        }
    }
    if constexpr (GROUPS > 1) {
        joined[group][at] = make_float2(m, s);
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int i = 1; i < GROUPS; ++i) join_stats(m, s, joined[i][at].x, joined[i][at].y, LOG2E);
        }
    }
    if (group == 0 && row < p.n) {
        state[row] = make_float2(m, s);
        if (label != p.ignore_index) {
            l = label >= 0 && label < p.V ? logf(s) - (score - m) : NAN;
            counted = 1.0f;
        }
        if (p.reduction == RED_NONE) loss[row] = l;
    }
    if (p.reduction == RED_NONE) return;
    block_sum2(l, counted, red);
    if (threadIdx.x == 0) {
        partial[blockIdx.x] = make_float2(l, counted);
        __threadfence();
        last = atomicAdd(done, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    l = counted = 0.0f;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) { const float2 q = __ldcg(partial + i); l += q.x; counted += q.y; }
    block_sum2(l, counted, red);
    if (threadIdx.x == 0) finish_loss(l, counted, p.reduction, loss, count);
}
// eight threads a row where there are parts for them
static int rows_per_block(int64_t parts) { return parts > 4 ? 32 : 256; }

// ---------------------------------------------------------------------------------------------
// Small fp32 calls, in fp32 arithmetic on the general cores: 64 x 64 tiles, 16 deep, 4 x 4 a thread.
// ---------------------------------------------------------------------------------------------
constexpr int TM = 64, TN = 64, TK = 16, PAD = 4;

struct Tiles { float a[TK][TM + PAD], b[TK][TN + PAD]; };

__device__ __forceinline__ void tile_product(const float *A, int64_t am, int64_t ak, const float *B, int64_t bk, int64_t bn, int64_t M, int64_t N,
                                             int64_t m0, int64_t n0, int64_t k0, int64_t k1, Tiles &t, float (&acc)[4][4]) {
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    for (int64_t k = k0; k < k1; k += TK) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // neighbouring threads take neighbouring elements of memory
            const int e = tid + i * 256;
            const int am_i = ak == 1 ? e >> 4 : e & 63, ak_i = ak == 1 ? e & 15 : e >> 6;
            const int bn_i = bk == 1 ? e >> 4 : e & 63, bk_i = bk == 1 ? e & 15 : e >> 6;
            const int64_t ma = m0 + am_i, ka = k + ak_i, nb = n0 + bn_i, kb = k + bk_i;
            t.a[ak_i][am_i] = ma < M && ka < k1 ? A[ma * am + ka * ak] : 0.0f;
            t.b[bk_i][bn_i] = nb < N && kb < k1 ? B[kb * bk + nb * bn] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < TK; ++kk) {
            const float4 av = *reinterpret_cast<const float4 *>(&t.a[kk][ty * 4]), bv = *reinterpret_cast<const float4 *>(&t.b[kk][tx * 4]);
            const float a[4] = {av.x, av.y, av.z, av.w}, b[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
}

// statistics of 64 rows over the class tiles blockIdx.y, + gridDim.y, ...
__global__ void __launch_bounds__(256) plain_stats_kernel(const Problem p, float2 *__restrict__ part, float *__restrict__ label_score,
                                                                               int *__restrict__ done) {
    __shared__ __align__(16) Tiles t;
    wait_for_previous();
    let_next_start();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *done = 0;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int64_t m0 = (int64_t)blockIdx.x * TM;
    float m[4], s[4], acc[4][4];
    int64_t label[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + ty * 4 + i;
        m[i] = NEG_INF; s[i] = 0.0f;
        label[i] = row < p.n ? load_index(p.labels, p.label_bytes, row) : -1;
    }
    const int64_t tiles = (p.V + TN - 1) / TN;
    for (int64_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
        const int64_t n0 = tile * TN;
        tile_product(static_cast<const float *>(p.x), p.ldx, 1, static_cast<const float *>(p.w), p.w_k(), p.w_v(), p.n, p.V, m0, n0, 0, p.d, t, acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t v = n0 + tx * 4 + j;
                if (v == label[i] && v < p.V) label_score[m0 + ty * 4 + i] = acc[i][j];
                if (v >= p.V) acc[i][j] = NEG_INF;
            }
            add_values<4>(m[i], s[i], acc[i], LOG2E);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) join_stats(m[i], s[i], __shfl_xor_sync(0xffffffffu, m[i], o, 16), __shfl_xor_sync(0xffffffffu, s[i], o, 16), LOG2E);
        const int64_t row = m0 + ty * 4 + i;
        if (tx == 0 && row < p.n) part[(int64_t)blockIdx.y * p.n + row] = make_float2(m[i], s[i]);
    }
}

// G of the classes [v0, v0 + cols), fp32, rows of ldg
__global__ void __launch_bounds__(256) plain_grad_kernel(const Problem p, int64_t v0, int64_t cols, float *__restrict__ G, int64_t ldg) {
    __shared__ __align__(16) Tiles t;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int64_t m0 = (int64_t)blockIdx.x * TM, n0 = (int64_t)blockIdx.y * TN;
    float acc[4][4];
    wait_for_previous();
    let_next_start();
    tile_product(static_cast<const float *>(p.x), p.ldx, 1, static_cast<const float *>(p.w) + v0 * p.w_v(), p.w_k(), p.w_v(), p.n, cols, m0, n0, 0, p.d, t, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + ty * 4 + i;
        if (row >= p.n) continue;
        const int64_t label = load_index(p.labels, p.label_bytes, row);
        const float r = prod::grad_row_factor(p, row, label);
        const float2 st = p.state[row];
        const float inv = 1.0f / st.y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t c = n0 + tx * 4 + j;
            if (c >= cols) continue;
            const float q = exp2_approx((acc[i][j] - st.x) * LOG2E) * inv - (v0 + c == label ? 1.0f : 0.0f);
            G[row * ldg + c] = r == 0.0f ? 0.0f : r * q;
        }
    }
}

// A product A [M, K] B [K, N] in parts of K: element strides, tiles, and its plane of fp32 partial sums [parts][M][N], or (one
// part) the output itself at m * om + n * on
struct PlainTask {
    const float *a, *b;
    int64_t am, ak, bk, bn, M, N, K, k_part;
    int m_tiles, n_tiles, parts, add;
    float *sum, *out;
    int64_t om, on;
    __host__ __device__ int blocks() const { return m_tiles * n_tiles * parts; }
};

// dx = G w^T (task 0) and dw = x^T G (task 1) of one piece
__global__ void __launch_bounds__(256) plain_products_kernel(const Problem p, const PlainTask dx, const PlainTask dw) {
    __shared__ __align__(16) Tiles t;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    wait_for_previous();
    let_next_start();
    int i = blockIdx.x;
    const bool second = i >= dx.blocks();
    const PlainTask &q = second ? dw : dx;
    if (second) i -= dx.blocks();
    const int part = i / (q.m_tiles * q.n_tiles), tile = i - part * (q.m_tiles * q.n_tiles);
    const int64_t m0 = (int64_t)(tile % q.m_tiles) * TM, n0 = (int64_t)(tile / q.m_tiles) * TN, k0 = part * q.k_part, k1 = min(q.K, k0 + q.k_part);
    float acc[4][4];
    tile_product(q.a, q.am, q.ak, q.b, q.bk, q.bn, q.M, q.N, m0, n0, k0, k1, t, acc);
    const float alpha = q.out ? prod::grad_alpha(p) : 1.0f;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int64_t m = m0 + ty * 4 + a, n = n0 + tx * 4 + b;
            if (m >= q.M || n >= q.N) continue;
            if (q.out) {
                q.out[m * q.om + n * q.on] = acc[a][b] * alpha;
            } else {
                float *o = q.sum + ((int64_t)part * q.M + m) * q.N + n;
                *o = q.add ? *o + acc[a][b] : acc[a][b];
            }
        }
}

// out(m, n) = alpha * sum of the partial planes [parts][M][ldp] in order, rounded once to the output's type; out(m, n) at
// m * om + n * on.  Four columns a thread.
template <typename T> __global__ void __launch_bounds__(256) round_kernel(const Problem p, const float *part, int parts, int64_t M, int64_t N,
                                                                          int64_t ldp, float scale, T *__restrict__ out, int64_t om, int64_t on) {
    wait_for_previous();
    let_next_start();
    const float alpha = prod::grad_alpha(p) * scale;
    const int64_t per_row = (N + 3) / 4, total = M * per_row, plane = M * ldp;
    const bool vector = on == 1 && om % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0 && ldp % 4 == 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = total <= UINT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row, n = (i - m * per_row) * 4;
        const float *q = part + m * ldp + n;
        T *o = out + m * om + n * on;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (vector && n + 4 <= N) {
            for (int k = 0; k < parts; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(q + k * plane);
                s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
            }
            T r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = from_float<T>(s[j] * alpha);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(r);
            else *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(r);
        } else {
            for (int j = 0; j < 4 && n + j < N; ++j) {
                for (int k = 0; k < parts; ++k) s[j] += q[k * plane + j];
                o[j * on] = from_float<T>(s[j] * alpha);
            }
        }
    }
}

// Operands for the tensor cores from those whose rows no TMA copy can start at (or as three bf16 planes): rows of `ldp`
// elements, a multiple of 8.  A thread per 8 elements, both operands in one launch.
struct PackTask { const void *src; uint16_t *dst; int64_t ld, rows, cols, ldp; };

template <typename T, int PLANES> __device__ __forceinline__ void pack8(const PackTask &t, int64_t i) {
    const int64_t per_row = t.ldp / 8, row = i / per_row, c = (i - row * per_row) * 8, plane = t.rows * t.ldp;
    const T *s = static_cast<const T *>(t.src) + row * t.ld + c;
    uint16_t *d = t.dst + row * t.ldp + c;
    if constexpr (PLANES == 1) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = c + 2 * j < t.cols ? reinterpret_cast<const uint16_t *>(s)[2 * j] : 0;
            const uint32_t hi = c + 2 * j + 1 < t.cols ? reinterpret_cast<const uint16_t *>(s)[2 * j + 1] : 0;
            q[j] = lo | hi << 16;
        }
        *reinterpret_cast<uint4 *>(d) = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
        uint32_t q[3][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a[2], b[2], e[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) prod::split3(c + 2 * j + h < t.cols ? to_float(s[2 * j + h]) : 0.0f, a[h], b[h], e[h]);
            q[0][j] = prod::pack2<true>(a[0], a[1]);
            q[1][j] = prod::pack2<true>(b[0], b[1]);
            q[2][j] = prod::pack2<true>(e[0], e[1]);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4 *>(d + k * plane) = make_uint4(q[k][0], q[k][1], q[k][2], q[k][3]);
    }
}
template <typename T, int PLANES> __global__ void __launch_bounds__(256) pack_kernel(const PackTask a, const PackTask b) {
    const int64_t first = a.rows * (a.ldp / 8), total = first + b.rows * (b.ldp / 8);
    wait_for_previous();
    let_next_start();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        if (i < first) pack8<T, PLANES>(a, i); else pack8<T, PLANES>(b, i - first);
    }
}

// Worst status of a tensor-core launch on this device since it was last read
static __device__ int g_status;
static long long g_wait_limit = prod::WAIT_LIMIT_CYCLES;

// ---------------------------------------------------------------------------------------------
// plan: how a call is cut up, and where its workspace lies
// ---------------------------------------------------------------------------------------------
constexpr size_t PIECE_BYTES = 512ull << 20;       // workspace for G
constexpr int64_t PIECE_UNIT = 256;                // its columns come in whole tiles
// Rows of packed operands and of G are whole lines of 128 bytes: a copy's 128-byte line of another row start touches two lines
// of L2, and what an SM takes in from L2 bounds the products (5,003 x 301 x 49,999 in fp16: 842 us with rows of whole 16 bytes,
// 753 with these; 8,192 x 301 x 10,007 in bf16: 273 and 222; 8,192 x 2,048 x 10,007: 1,201 and 1,008)
constexpr int64_t LINE = 64;

struct Plan {
    bool tensor;
    int planes;                                    // of an operand: 1, or 3 of bf16 (see planes_of)
    int kind, score_kind;                          // how sums are held (prod::Kind), those of the scores
    bool pack_x, pack_w;
    int64_t ldx, ldw, ldg, ld_dx, ld_dw;           // rows of the operands as the tensor cores read them, of fp32 sums
    int64_t run, parts;                            // forward: class tiles per unit, parts of the class axis
    int64_t piece;                                 // backward: classes per piece
    int64_t dx_parts, dx_len, dw_parts, dw_len;    // parts of the two products' inner axes (classes of a piece, rows)
    bool sum_dx, sum_dw;                           // through planes of fp32 sums, even of one part
    bool turn_dw;                                  // dw of [d, V] as the transpose of G^T x
    size_t x, w;                                   // packed operands
    size_t stats, label_score, partial, done;      // forward scratch
    size_t norm, G, dx_sum, dw_sum;                // backward scratch
    size_t bytes;
};

static size_t place(size_t &at, size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
}
static void place_rows(size_t &at, int64_t n, Plan *q) {
    q->label_score = place(at, (size_t)n * sizeof(float));
    q->partial = place(at, (size_t)ceil_div(n, (int64_t)rows_per_block(q->parts)) * sizeof(float2));
    q->done = place(at, sizeof(int));
}
// parts of an inner axis of K so that `tiles` output tiles give every SM two blocks; none shorter than `least`
static void cut(int64_t tiles, int64_t K, int64_t least, int64_t unit, int64_t *parts, int64_t *len) {
    int64_t s = ceil_div((int64_t)sm_count() * 2, tiles > 0 ? tiles : 1);
    if (s > K / least) s = K / least;
    if (s < 1) s = 1;
    *len = ceil_div(ceil_div(K > 0 ? K : 1, s), unit) * unit;
    *parts = ceil_div(K > 0 ? K : 1, *len);
}

static int64_t in_32s(int64_t N) { return ceil_div(N, (int64_t)32) * 32; }
static int64_t column_tiles(int64_t N, int kind) { return ceil_div(N, (int64_t)prod::tile_width(kind)); }
static int columns_per_tile(int64_t N, int kind) {
    const int64_t tiles = column_tiles(N, kind);
    return (int)(tiles == 1 ? in_32s(N) : ceil_div(ceil_div(N, tiles), (int64_t)64) * 64);
}
static int64_t tiles_of(int64_t M, int64_t N, int cg, int kind) { return ceil_div(M, (int64_t)(prod::BM * cg)) * column_tiles(N, kind); }
// What 64 inner elements of a tile take, in steps of a 256 x 256 tile (some 0.4 us of a pair of SMs): fp32 has six products of half the width
static int64_t step_cost(int kind) { return kind == prod::PLANES3 ? 3 : 1; }

// CTAs that share a tile: pairs where there are more rows than one CTA's
static int cta_group(int64_t M) { return M > prod::BM ? 2 : 1; }

// Whether scores of 16-bit operands are summed in chains of 256 elements, which the epilogue adds up to nearest.  The tensor cores cut
// off every 16 products' sum towards zero: one sum over the width is off by some 1.5 * 2^-24 of itself per 16 elements where all have one
// sign (65,536 elements: a score of 18 came out 0.007 too small), and losses by 5e-7 (many classes) to 1.2e-6 (two) at a width of 1,024,
// 4.6e-6 at 4,096, where a chain leaves 1e-7 to 3e-7 at any width.  Tiles of half the columns are what it costs (forward,
// bf16, us, one sum and chains: 90,941 x 1,440 x 172 75 and 102, 2,000 x 1,440 x 30,000 166 and 208, 8,192 x 4,096 x 32,000 1,500 and
// 2,015), and nothing where the classes fit one (90,941 x 1,024 x 47 46 and 46, 20,000 x 768 x 100 18.6 and 20.6).  G is rounded to 16 bits, so its
// scores may be off by more, but not by more than that rounding: 2.4e-5 of a score at 4,096.
static bool in_chains(int64_t d, int64_t V, bool backward) {
    if (backward) return d > 4096;
    return d > (V <= prod::tile_width(prod::CHAINS) ? 768 : 1024);
}

static bool needs_packing(const void *p, int64_t ld, int planes) { return planes == 3 || !aligned16(p) || ld % 8 != 0; }

// fp32 operands are three bf16 planes.  So are fp16 ones (exactly), and with them G, in the backward pass of rows' losses
// without a reduction: rows' gradients may be decades apart, dw needs one scale for all rows, and a row's softmax, some 2^-16
// of its gradient where classes are many, would leave fp16's range from 10^-5 of the largest gradient on.  That is six
// products for one and up to two launches more: forward and backward of 1,024 x 512 x 32,768 497 us against 156 of the mean, 5,003
// x 301 x 49,999 2,914 against 647; 140 x 32 x 7 160 against 155.
static int planes_of(const Problem &p, bool backward) {
    return p.dtype == GRWS_F32 || (p.dtype == GRWS_F16 && backward && p.reduction == RED_NONE) ? 3 : 1;
}

// Class tiles that one unit of the scores takes: as many as leave the SMs equally busy.  A tile step takes about 0.4 us; a unit
// costs the latency of its rows' data (0.8 us) and, forward, a statistic per row (of two warps each) written and read at some
// 5 TB/s and a step of the loop that joins them.
static void cut_runs(int64_t n, int64_t m_tiles, int64_t n_tiles, int64_t steps, int64_t ctas, bool forward, int64_t *run, int64_t *runs) {
    int64_t best = 1;
    double best_us = 1e300;
    for (int64_t r = 1; r <= n_tiles && r <= 64; ++r) {
        const int64_t k = ceil_div(n_tiles, r);
        const double us = (double)ceil_div(m_tiles * k, ctas) * ((double)(r * steps) * 0.4 + 0.8) + (forward ? (double)(k * n) * 32.0 / 5.0e6 + 0.06 * (double)k : 0.0);
        if (us <= best_us) { best_us = us; best = r; }
    }
    *run = best;
    *runs = ceil_div(n_tiles, best);
}

// What a unit of `steps` takes, in steps: a tile's sums need about six to leave
static int64_t unit_time(int64_t steps) { return steps > 6 ? steps : 6; }

// Units of the second task for the CTAs that have one unit more (less) of the first, whose units are the longer ones, so that
// all are done at about the same time; returns that time in steps.
static int64_t deal_units(int64_t u0, int64_t l0, int64_t u1, int64_t l1, int64_t ctas, int *less, int *more) {
    const int64_t each = u0 / ctas, many = u0 % ctas;
    for (int64_t t = ceil_div(u0 * l0 + u1 * l1, ctas);; t += 1 + l1 / 16) {
        const int64_t left = t - (each + 1) * l0, right = t - each * l0;
        const int64_t a = left > 0 ? left / l1 : 0, b = right > 0 ? right / l1 : 0;
        if (many * a + (ctas - many) * b < u1) continue;
        if (less) *less = (int)a;
        if (more) *more = (int)b;
        const int64_t longest = (each + (many > 0)) * l0;
        return t > longest ? t : longest;
    }
}

// Parts of the inner axes of dx (classes of a piece) and dw (rows), which run in one launch: short units leave the CTAs equally
// busy, but every part is one more plane of fp32 sums through memory.  Costs are in
// units of one 64-element step of one tile, about 0.4 us of a pair of SMs; a launch that adds planes up takes some 6 us.
static double cut_products(int64_t tiles0, int64_t k0, double sums0, int64_t tiles1, int64_t k1, double sums1, int64_t step, int64_t ctas, int64_t *parts0,
                           int64_t *parts1) {
    static const int64_t tries[] = {1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 12, 14, 16, 18, 20, 24, 28, 32, 37, 48, 64, 74, 96, 128, 148};
    const double step_us = 0.4, plane_us = 8.0 / 2.5e6;          // an fp32 number written and read at 2.5 TB/s
    double best = 1e300;
    for (int64_t a : tries) {
        if (a > 1 && (k0 / a < 8 || tiles0 * a > 6 * ctas)) break;
        for (int64_t b : tries) {
            if (b > 1 && (k1 / b < 8 || tiles1 * b > 6 * ctas)) break;
            const int64_t l0 = ceil_div(k0, a), l1 = ceil_div(k1, b), u0 = tiles0 * a, u1 = tiles1 * b;
            const int64_t t0 = unit_time(l0 * step), t1 = unit_time(l1 * step);
            double cost = (double)(l1 >= l0 ? deal_units(u1, t1, u0, t0, ctas, nullptr, nullptr) : deal_units(u0, t0, u1, t1, ctas, nullptr, nullptr));
            if (a > 1) cost += (6.0 + (double)a * sums0 * plane_us) / step_us;
            if (b > 1) cost += (6.0 + (double)b * sums1 * plane_us) / step_us;
            if (cost < best) { best = cost; *parts0 = a; *parts1 = b; }
        }
    }
    return best;
}

// 16-bit operands always go to the tensor cores (140 x 32 x 7: 20.7 us against 24.7 on the general cores, 300 x 256 x 40: 23
// against 66), fp32 from 2^21 products on (128 x 128 x 128: 33 us against 43; 256 x 64 x 47: 35 against 33; 140 x 32 x 7: 29
// against 25, and five launches more).
static bool on_tensor_cores(int64_t n, int64_t d, int64_t V, int dtype) {
    return dtype != GRWS_F32 || (double)n * (double)d * (double)V >= (double)(1 << 21);
}

// dw of a [d, V] weight is x^T G, whose rows d come in tiles of 128 or 256, or the transpose of G^T x, whose columns d come in
// 32s, and which leaves the registers as 64-byte pieces of rows (128 of fp32).  The latter where it multiplies a quarter less
// (forward and backward, bf16: 5,003 x 301 x 49,999 in 580 us against 619, 30,000 x 100 x 49,999 in 2,358 against 2,609, 8,192 x
// 320 x 10,000 in 258 against 269; fp32: 8,192 x 96 x 49,999 in 2,284 against 2,745; a fifth less, bf16, 30,000 x 600 x 49,999:
// 6,931 against 6,840).
static bool turns(const Problem &p, int cg, int kind) {
    if (p.class_major) return false;
    const int64_t before = (column_tiles(p.d, kind) - 1) * columns_per_tile(p.d, kind), rows = (int64_t)prod::BM * cg;
    return 3 * ceil_div(p.d, rows) * rows >= 4 * (before + in_32s(p.d - before));
}

static Plan make_plan(const Problem &p, bool backward) {
    Plan q = {};
    const int64_t n = p.n, d = p.d, V = p.V;
    q.tensor = on_tensor_cores(n, d, V, p.dtype);
    size_t at = 0;
    if (!q.tensor) {
        const int64_t row_tiles = ceil_div(n, (int64_t)TM), class_tiles = ceil_div(V, (int64_t)TN), width_tiles = ceil_div(d, (int64_t)TN);
        if (!backward) {
            q.parts = ceil_div((int64_t)sm_count() * 2, row_tiles > 0 ? row_tiles : 1);
            if (q.parts > class_tiles) q.parts = class_tiles;
            q.stats = place(at, (size_t)q.parts * n * sizeof(float2));
            place_rows(at, n, &q);
        } else {
            q.piece = (int64_t)(PIECE_BYTES / sizeof(float)) / (n > 0 ? n : 1) / TN * TN;
            if (q.piece < TN) q.piece = TN;
            if (q.piece > 32768) q.piece = 32768;           // (a grid has at most 65,535 tiles in y)
            if (q.piece > V) q.piece = V;
            cut(row_tiles * width_tiles, q.piece, 128, TK, &q.dx_parts, &q.dx_len);
            cut(width_tiles * ceil_div(q.piece, (int64_t)TN), n, 128, TK, &q.dw_parts, &q.dw_len);
            q.norm = place(at, sizeof(float));
            q.G = place(at, (size_t)n * q.piece * sizeof(float));
            q.dx_sum = place(at, (size_t)q.dx_parts * n * d * sizeof(float));
            q.dw_sum = place(at, (size_t)q.dw_parts * d * q.piece * sizeof(float));
        }
        q.bytes = at;
        return q;
    }
    q.planes = planes_of(p, backward);
    q.kind = q.planes == 3 ? prod::PLANES3 : prod::WHOLE;
    q.score_kind = q.planes == 1 && in_chains(d, V, backward) ? prod::CHAINS : q.kind;
    const int64_t w_rows = p.class_major ? V : d, w_cols = p.class_major ? d : V;
    // x whose rows are no whole lines is packed for many classes, which read it as often (bf16, 8,192 x 1,000 x 50,000: 2,663 us
    // as it is, 2,430 packed; x 10,000: 479 and 462; 8,192 x 304 x 10,000: 210 and 211; x 1,000: 54 and 58); a copy of w, as
    // large as what dw writes, costs what it saves (8,192 x 1,000 x 50,000: 2,663 and 2,666; 1,000 rows: 329 and 387)
    q.pack_x = needs_packing(p.x, p.ldx, q.planes) || (p.ldx % LINE != 0 && V >= 16384);
    q.pack_w = needs_packing(p.w, p.ldw, q.planes);
    q.ldx = q.pack_x ? ceil_div(d, LINE) * LINE : p.ldx;
    q.ldw = q.pack_w ? ceil_div(w_cols, LINE) * LINE : p.ldw;
    if (q.pack_x) q.x = place(at, (size_t)q.planes * n * q.ldx * 2);
    if (q.pack_w) q.w = place(at, (size_t)q.planes * w_rows * q.ldw * 2);
    const int cg = cta_group(n);
    if (!backward) {
        const int64_t bn = columns_per_tile(V, q.score_kind);
        cut_runs(n, ceil_div(n, (int64_t)(prod::BM * cg)), ceil_div(V, bn), ceil_div(d, (int64_t)prod::BK) * step_cost(q.score_kind), sm_count() / cg, true, &q.run, &q.parts);
        q.stats = place(at, (size_t)q.parts * 2 * n * sizeof(float2));
        place_rows(at, n, &q);
    } else {
        int64_t most = (int64_t)(PIECE_BYTES / (2 * q.planes)) / n / PIECE_UNIT * PIECE_UNIT;
        if (most < PIECE_UNIT) most = PIECE_UNIT;
        const int pg = cta_group(n > d ? n : d);
        const int64_t k1 = ceil_div(n, (int64_t)prod::BK);
        // all classes at once if they fit; else the largest piece, or one down to half of it whose products leave the SMs more
        // equally busy
        const int64_t all = ceil_div(V, PIECE_UNIT) * PIECE_UNIT, top = most < all ? most : all;
        const bool summed = q.planes == 3 && p.dtype != GRWS_F32;          // (the kernel rounds to the type of its operands or to fp32)
        for (q.turn_dw = !summed && turns(p, pg, q.kind);; q.turn_dw = false) {
            double best = 1e300;
            for (int64_t k = 8; k >= (all <= most ? 8 : 4); --k) {
                const int64_t piece = ceil_div(top * k / 8, PIECE_UNIT) * PIECE_UNIT;
                const int64_t c = piece < V ? piece : V;
                const int64_t tiles0 = tiles_of(n, d, pg, q.kind), tiles1 = p.class_major || q.turn_dw ? tiles_of(c, d, pg, q.kind) : tiles_of(d, c, pg, q.kind);
                int64_t a, b;
                const double cost = (cut_products(tiles0, ceil_div(c, (int64_t)prod::BK), (double)n * d, tiles1, k1, (double)d * c, step_cost(q.kind), sm_count() / pg, &a, &b) +
                                     (c < V ? (double)n * d * 8.0 / 5.0e6 / 0.4 : 0.0)) * (double)ceil_div(V, c);
                if (cost < best) { best = cost; q.piece = c; q.dx_parts = a; q.dw_parts = b; }
            }
            if (!q.turn_dw || q.dw_parts == 1) break;          // (the sums of parts are added up as they lie)
        }
        q.ldg = ceil_div(q.piece, LINE) * LINE;
        const int64_t k0 = ceil_div(q.piece, (int64_t)prod::BK);
        q.dx_len = ceil_div(k0, q.dx_parts);
        q.dx_parts = ceil_div(k0, q.dx_len);
        q.dw_len = ceil_div(k1, q.dw_parts);
        q.dw_parts = ceil_div(k1, q.dw_len);
        q.ld_dx = ceil_div(d, (int64_t)4) * 4;
        q.ld_dw = ceil_div(p.class_major ? d : q.piece, (int64_t)4) * 4;
        q.norm = place(at, sizeof(float));
        q.G = place(at, (size_t)q.planes * n * q.ldg * 2);
        q.sum_dx = summed || q.dx_parts > 1 || q.piece < V;
        q.sum_dw = summed || q.dw_parts > 1;
        if (q.sum_dx) q.dx_sum = place(at, (size_t)q.dx_parts * n * q.ld_dx * sizeof(float));
        if (q.sum_dw) q.dw_sum = place(at, (size_t)q.dw_parts * (p.class_major ? q.piece : d) * q.ld_dw * sizeof(float));
    }
    q.bytes = at;
    return q;
}

template <typename T> static int launch_round(const Problem &p, const float *part, int64_t parts, int64_t M, int64_t N, int64_t ldp, float scale, void *out, int64_t om,
                                              int64_t on, cudaStream_t st) {
    int64_t g = ceil_div(M * ceil_div(N, (int64_t)4), (int64_t)256);
    const int64_t most = (int64_t)sm_count() * 8;
    if (g > most) g = most;
    return launch_next(round_kernel<T>, dim3((unsigned)g), 256, 0, st, 1, p, part, (int)parts, M, N, ldp, scale, static_cast<T *>(out), om, on);
}

// ---- the tensor cores' way ----
// an operand as it lies in memory: [planes][rows][cols], cols contiguous
struct View { const void *p; int64_t rows, cols, ld, plane; int planes; };
struct Operands { View x, w; int dtype; };

template <typename T> static int pack_operands(const Problem &p, const Plan &q, char *scratch, Operands *o, cudaStream_t st) {
    const int64_t w_rows = p.class_major ? p.V : p.d, w_cols = p.class_major ? p.d : p.V;
    o->x = View{q.pack_x ? scratch + q.x : p.x, p.n, p.d, q.ldx, p.n * q.ldx, q.planes};
    o->w = View{q.pack_w ? scratch + q.w : p.w, w_rows, w_cols, q.ldw, w_rows * q.ldw, q.planes};
    o->dtype = q.planes == 1 && p.dtype == GRWS_F16 ? GRWS_F16 : GRWS_BF16;
    PackTask a = {}, b = {};
    if (q.pack_x) a = PackTask{p.x, reinterpret_cast<uint16_t *>(scratch + q.x), p.ldx, p.n, p.d, q.ldx};
    if (q.pack_w) b = PackTask{p.w, reinterpret_cast<uint16_t *>(scratch + q.w), p.ldw, w_rows, w_cols, q.ldw};
    const int64_t blocks = ceil_div(a.rows * (a.ldp / 8) + b.rows * (b.ldp / 8), (int64_t)256), most = (int64_t)sm_count() * 8;
    if (blocks == 0) return GRWS_OK;
    void (*kernel)(const PackTask, const PackTask) = pack_kernel<T, sizeof(T) == 4 ? 3 : 1>;
    if constexpr (std::is_same<T, __half>::value) if (q.planes == 3) kernel = pack_kernel<T, 3>;
    return launch_next(kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, st, 1, a, b);
}

// sets a product up: its tile counts and the maps of its operands; `outer`: the operand's rows are the inner axis
static int set_task(prod::Task *t, CUtensorMap *ma, CUtensorMap *mb, int cg, int kind, int dtype, const View &a, int a_outer, const View &b, int b_outer, int64_t M,
                    int64_t N, int64_t K) {
    t->M = M; t->N = N;
    t->bn = columns_per_tile(N, kind);
    t->m_tiles = (int)ceil_div(M, (int64_t)(prod::BM * cg));
    t->n_tiles = (int)ceil_div(N, (int64_t)t->bn);
    t->run = 1; t->runs = t->n_tiles; t->splits = 1;
    t->k_blocks = t->k_len = (int)ceil_div(K, (int64_t)prod::BK);
    t->group = t->m_tiles < 16 ? t->m_tiles : 16;
    t->a_outer = a_outer; t->b_outer = b_outer;
    if (int rc = prod::encode_map(ma, a.p, dtype, a.cols, a.rows, a.ld, a.planes, a.plane, 64, a_outer ? prod::BK : prod::BM)) return rc;
    return prod::encode_map(mb, b.p, dtype, b.cols, b.rows, b.ld, b.planes, b.plane, 64, b_outer ? prod::BK : prod::tile_width(kind) / cg);
}

// where a SUM task's results go: planes of fp32 sums, or the rounded output
static int set_sums(prod::Task *t, CUtensorMap *mc, int64_t parts, float *sum, int64_t ld, bool add) {
    t->splits = (int)parts;
    t->add = add;
    return prod::encode_map(mc, sum, GRWS_F32, t->N, t->M, ld, (int)parts, t->M * ld, 32, 32);
}
static int set_rounded(prod::Task *t, CUtensorMap *mc, int dtype, void *out, int64_t ldo) {
    t->rounded = 1;
    if (!aligned16(out) || ldo * (int64_t)dtype_bytes(dtype) % 16 != 0) {         // no TMA store starts at such rows
        t->out = out;
        t->ldo = ldo;
        return GRWS_OK;
    }
    return prod::encode_map(mc, out, dtype, t->N, t->M, ldo, 1, 0, dtype == GRWS_F32 ? 32 : 64, 32);
}

static int status_word(int **word) {
    static int *known[MAX_DEVICES];
    const int dev = current_device();
    if (dev < 0) return fail(GRWS_ERR_CUDA, "no current device");
    *word = __atomic_load_n(&known[dev], __ATOMIC_RELAXED);
    if (!*word) {
        void *p = nullptr;
        GRWS_CUDA_TRY(cudaGetSymbolAddress(&p, g_status));
        *word = static_cast<int *>(p);
        __atomic_store_n(&known[dev], *word, __ATOMIC_RELAXED);
    }
    return GRWS_OK;
}

static int product_params(const Problem &p, int dtype, prod::Params *r) {
    int *status = nullptr;
    if (int rc = status_word(&status)) return rc;
    *r = prod::Params{};
    r->tasks = 1;
    r->bf16 = dtype != GRWS_F16;
    r->labels = p.labels; r->label_bytes = p.label_bytes; r->ignore_index = p.ignore_index; r->V = p.V;
    r->reduction = p.reduction; r->grad = p.grad; r->count = p.count; r->norm = p.norm;
    r->state = p.state;
    r->scale = 1.0f;
    r->status = status;
    r->wait_limit = __atomic_load_n(&g_wait_limit, __ATOMIC_RELAXED);
#ifdef GRWS_TC5_PROFILING
    const char *withhold = getenv("GRWS_CE_WITHHOLD");
    r->withhold = withhold ? atoi(withhold) : 0;
#endif
    return GRWS_OK;
}

template <int MODE> static int launch_product(int cg, int kind, const prod::Maps &maps, const prod::Params &r, cudaStream_t st) {
    if (kind == prod::PLANES3) return cg == 2 ? prod::launch_product<2, MODE, prod::PLANES3>(maps, r, st) : prod::launch_product<1, MODE, prod::PLANES3>(maps, r, st);
    if constexpr (MODE != prod::SUM) {
        if (kind == prod::CHAINS) return cg == 2 ? prod::launch_product<2, MODE, prod::CHAINS>(maps, r, st) : prod::launch_product<1, MODE, prod::CHAINS>(maps, r, st);
    }
    return cg == 2 ? prod::launch_product<2, MODE, prod::WHOLE>(maps, r, st) : prod::launch_product<1, MODE, prod::WHOLE>(maps, r, st);
}

template <typename T> static int tensor_forward(const Problem &p, const Plan &q, float2 *part, float *label_score, int *done, char *scratch, cudaStream_t st) {
    Operands o;
    if (int rc = pack_operands<T>(p, q, scratch, &o, st)) return rc;
    prod::Params r;
    if (int rc = product_params(p, o.dtype, &r)) return rc;
    prod::Maps maps;
    const int cg = cta_group(p.n);
    if (int rc = set_task(&r.task[0], &maps.a[0], &maps.b[0], cg, q.score_kind, o.dtype, o.x, 0, o.w, !p.class_major, p.n, p.V, p.d)) return rc;
    r.task[0].run = (int)q.run;
    r.task[0].runs = (int)q.parts;
    r.part = part;
    r.label_score = label_score;
    r.done = done;
    return launch_product<prod::STATS>(cg, q.score_kind, maps, r, st);
}

// G in fp16 is held as 2^12 G: |G| <= 1, and a probability of 2^-26 is still a normal number
static float stored_scale(const Operands &o) { return o.dtype == GRWS_F16 ? 4096.0f : 1.0f; }

template <typename T> static int tensor_backward(const Problem &p, const Plan &q, void *dx, void *dw, char *scratch, cudaStream_t st) {
    Operands o;
    if (int rc = pack_operands<T>(p, q, scratch, &o, st)) return rc;
    float *dx_sum = reinterpret_cast<float *>(scratch + q.dx_sum), *dw_sum = reinterpret_cast<float *>(scratch + q.dw_sum);
    for (int64_t v0 = 0; v0 < p.V; v0 += q.piece) {
        const int64_t cols = p.V - v0 < q.piece ? p.V - v0 : q.piece;
        const View G = {scratch + q.G, p.n, cols, q.ldg, p.n * q.ldg, q.planes};
        prod::Params r;
        if (int rc = product_params(p, o.dtype, &r)) return rc;
        prod::Maps maps;
        const int cg = cta_group(p.n);
        if (int rc = set_task(&r.task[0], &maps.a[0], &maps.b[0], cg, q.score_kind, o.dtype, o.x, 0, o.w, !p.class_major, p.n, cols, p.d)) return rc;
        if (int rc = prod::encode_map(&maps.c[0], G.p, o.dtype, cols, p.n, q.ldg, q.planes, G.plane, q.planes == 3 ? 32 : 64, 32)) return rc;
        int64_t run, runs;
        cut_runs(p.n, r.task[0].m_tiles, r.task[0].n_tiles, r.task[0].k_blocks * step_cost(q.score_kind), sm_count() / cg, false, &run, &runs);
        r.task[0].run = (int)run;
        r.task[0].runs = (int)runs;
        r.task[0].b_row0 = (int)v0;
        r.v0 = v0;
        r.scale = stored_scale(o);
        if (int rc = launch_product<prod::GRAD>(cg, q.score_kind, maps, r, st)) return rc;

        if (int rc = product_params(p, o.dtype, &r)) return rc;
        r.scale = 1.0f / stored_scale(o);
        r.tasks = 0;
        const int pg = cta_group(p.n > p.d ? p.n : p.d);
        const int64_t M = p.class_major ? cols : p.d, N = p.class_major ? p.d : cols, ldo = p.class_major ? p.d : p.V;
        T *dw_out = static_cast<T *>(dw) + (p.class_major ? v0 * p.d : v0);
        // the longer units first
        for (int k = 0; k < 2; ++k) {
            const bool is_dw = (q.dw_len >= q.dx_len) == (k == 0);
            if (!(is_dw ? dw : dx)) continue;
            const int i = r.tasks++;
            prod::Task *t = &r.task[i];
            int rc;
            if (is_dw) {
                // [d, V]: x^T G, or the transpose of G^T x; [V, d]: G^T x
                rc = p.class_major || q.turn_dw ? set_task(t, &maps.a[i], &maps.b[i], pg, q.kind, o.dtype, G, 1, o.x, 1, cols, p.d, p.n)
                                                : set_task(t, &maps.a[i], &maps.b[i], pg, q.kind, o.dtype, o.x, 1, G, 1, M, N, p.n);
                if (rc != GRWS_OK) return rc;
                t->k_len = (int)q.dw_len;
                if (q.turn_dw) {
                    t->rounded = 1;
                    t->turned = true;
                    t->out = dw_out;
                    t->ldo = ldo;
                } else {
                    rc = q.sum_dw ? set_sums(t, &maps.c[i], q.dw_parts, dw_sum, q.ld_dw, false) : set_rounded(t, &maps.c[i], p.dtype, dw_out, ldo);
                }
            } else {
                rc = set_task(t, &maps.a[i], &maps.b[i], pg, q.kind, o.dtype, G, 0, o.w, p.class_major, p.n, p.d, cols);
                if (rc != GRWS_OK) return rc;
                t->b_k0 = (int)v0;
                t->k_len = (int)q.dx_len;
                rc = q.sum_dx ? set_sums(t, &maps.c[i], ceil_div((int64_t)t->k_blocks, q.dx_len), dx_sum, q.ld_dx, v0 > 0)      // (a last, shorter piece: fewer)
                            : set_rounded(t, &maps.c[i], p.dtype, dx, p.d);
            }
            if (rc != GRWS_OK) return rc;
        }
        const int64_t ctas = sm_count() / pg, units = r.task[0].units() + (r.tasks > 1 ? r.task[1].units() : 0);
        // few units per CTA: dealt out by length (many: in order, so that those at work at a time share operands in L2)
        if (r.tasks > 1 && units <= 12 * ctas) {
            r.deal = 1;
            deal_units(r.task[0].units(), unit_time(r.task[0].k_len * step_cost(q.kind)), r.task[1].units(), unit_time(r.task[1].k_len * step_cost(q.kind)), units < ctas ? units : ctas, &r.deal_less, &r.deal_more);
        }
        if (int rc = launch_product<prod::SUM>(pg, q.kind, maps, r, st)) return rc;
        if (dw && q.sum_dw) if (int rc = launch_round<T>(p, dw_sum, q.dw_parts, M, N, q.ld_dw, r.scale, dw_out, ldo, 1, st)) return rc;
    }
    return dx && q.sum_dx ? launch_round<T>(p, dx_sum, q.dx_parts, p.n, p.d, q.ld_dx, 1.0f / stored_scale(o), dx, p.d, 1, st) : GRWS_OK;
}

template <typename T> static int forward(const Problem &p, const Plan &q, float *loss, float2 *state, float *count, char *scratch, cudaStream_t st) {
    float2 *part = reinterpret_cast<float2 *>(scratch + q.stats), *partial = reinterpret_cast<float2 *>(scratch + q.partial);
    float *label_score = reinterpret_cast<float *>(scratch + q.label_score);
    int *done = reinterpret_cast<int *>(scratch + q.done);
    if (int rc = q.tensor ? tensor_forward<T>(p, q, part, label_score, done, scratch, st)
                          : launch_next(plain_stats_kernel, dim3((unsigned)ceil_div(p.n, (int64_t)TM), (unsigned)q.parts), 256, 0, st, 1, p, part, label_score, done))
        return rc;
    const int rows = rows_per_block(q.parts);
    return launch_next(rows == 32 ? rows_kernel<8> : rows_kernel<1>, dim3((unsigned)ceil_div(p.n, (int64_t)rows)), 256, 0, st, 1, p, part,
                       (int)(q.tensor ? 2 * q.parts : q.parts), label_score, state, loss, count, partial, done);
}

static int plain_backward(const Problem &p, const Plan &q, float *dx, float *dw, char *scratch, cudaStream_t st) {
    float *G = reinterpret_cast<float *>(scratch + q.G), *dx_sum = reinterpret_cast<float *>(scratch + q.dx_sum), *dw_sum = reinterpret_cast<float *>(scratch + q.dw_sum);
    const unsigned row_tiles = (unsigned)ceil_div(p.n, (int64_t)TM);
    const float *x = static_cast<const float *>(p.x), *w = static_cast<const float *>(p.w);
    const bool sum_dx = q.dx_parts > 1 || q.piece < p.V, sum_dw = q.dw_parts > 1;
    const int64_t ok = p.class_major ? 1 : p.V, ov = p.class_major ? p.d : 1;
    for (int64_t v0 = 0; v0 < p.V; v0 += q.piece) {
        const int64_t cols = p.V - v0 < q.piece ? p.V - v0 : q.piece;
        if (int rc = launch_next(plain_grad_kernel, dim3(row_tiles, (unsigned)ceil_div(cols, (int64_t)TN)), 256, 0, st, 1, p, v0, cols, G, q.piece)) return rc;
        PlainTask tx = {}, tw = {};
        if (dx) {
            tx = PlainTask{G, w + v0 * p.w_v(), q.piece, 1, p.w_v(), p.w_k(), p.n, p.d, cols, q.dx_len, (int)row_tiles, (int)ceil_div(p.d, (int64_t)TN),
                           (int)ceil_div(cols, q.dx_len), v0 > 0, dx_sum, sum_dx ? nullptr : dx, p.d, 1};
        }
        float *dw_out = dw + v0 * ov;
        if (dw) {
            tw = PlainTask{x, G, 1, p.ldx, q.piece, 1, p.d, cols, p.n, q.dw_len, (int)ceil_div(p.d, (int64_t)TM), (int)ceil_div(cols, (int64_t)TN),
                           (int)q.dw_parts, 0, dw_sum, sum_dw ? nullptr : dw_out, ok, ov};
        }
        if (int rc = launch_next(plain_products_kernel, dim3((unsigned)(tx.blocks() + tw.blocks())), 256, 0, st, 1, p, tx, tw)) return rc;
        if (dw && sum_dw) if (int rc = launch_round<float>(p, dw_sum, q.dw_parts, p.d, cols, cols, 1.0f, dw_out, ok, ov, st)) return rc;
    }
    return dx && sum_dx ? launch_round<float>(p, dx_sum, q.dx_parts, p.n, p.d, p.d, 1.0f, dx, p.d, 1, st) : GRWS_OK;
}

template <typename T> static int backward(Problem p, const Plan &q, void *dx, void *dw, char *scratch, cudaStream_t st) {
    if (p.reduction == RED_NONE) {
        float *norm = reinterpret_cast<float *>(scratch + q.norm);
        if (int rc = launch_next(grad_norm_kernel, dim3(1), 1024, 0, st, 1, p, norm)) return rc;
        p.norm = norm;
    }
    return q.tensor ? tensor_backward<T>(p, q, dx, dw, scratch, st) : plain_backward(p, q, static_cast<float *>(dx), static_cast<float *>(dw), scratch, st);
}

static int check(const Problem &p) {
    GRWS_REQUIRE(p.n >= 0 && p.d > 0 && p.V > 0, "bad size (rows = %lld, width = %lld, classes = %lld)", (long long)p.n, (long long)p.d, (long long)p.V);
    GRWS_REQUIRE(p.n <= INT32_MAX && p.d <= INT32_MAX && p.V <= INT32_MAX, "rows, width and classes must fit 31 bits");
    GRWS_REQUIRE((double)p.n * (double)p.V < 3.0e13, "rows x classes must stay below 3e13");      // tiles are numbered in 31 bits
    GRWS_REQUIRE(p.ldx >= p.d && p.ldw >= (p.class_major ? p.d : p.V), "leading dimension smaller than the row");
    GRWS_REQUIRE(p.class_major == 0 || p.class_major == 1, "bad weight order %d", p.class_major);
    if (p.dtype < GRWS_F32 || p.dtype > GRWS_BF16) return fail(GRWS_ERR_UNSUPPORTED, "bad dtype %d", p.dtype);
    GRWS_REQUIRE(p.label_bytes == 4 || p.label_bytes == 8, "labels are 4- or 8-byte integers");
    GRWS_REQUIRE(p.reduction >= RED_NONE && p.reduction <= RED_SUM, "bad reduction %d", p.reduction);
    return GRWS_OK;
}

static Problem problem(const void *x, int64_t ldx, const void *w, int64_t ldw, int class_major, const void *labels, int label_bytes, int64_t ignore_index,
                       int64_t n, int64_t d, int64_t V, int dtype, int reduction) {
    Problem p = {};
    p.x = x; p.ldx = ldx; p.w = w; p.ldw = ldw; p.class_major = class_major; p.labels = labels; p.label_bytes = label_bytes;
    p.ignore_index = ignore_index; p.n = n; p.d = d; p.V = V; p.dtype = dtype; p.reduction = reduction;
    return p;
}

}  // namespace lce
}  // namespace grws

using namespace grws;

extern "C" {

__attribute__((visibility("default")))
size_t grws_linear_ce_scratch_bytes(const void *x, int64_t ldx, const void *w, int64_t ldw, int class_major, int64_t rows, int64_t width,
                                    int64_t classes, int dtype, int backward) {
    if (rows <= 0 || width <= 0 || classes <= 0) return 0;
    const auto bytes = [&](int reduction) {
        return lce::make_plan(lce::problem(x, ldx, w, ldw, class_major, nullptr, 8, 0, rows, width, classes, dtype, reduction), backward != 0).bytes;
    };
    const size_t reduced = bytes(cls::RED_MEAN);
    if (backward != 1 || dtype != GRWS_F16) return reduced;
    const size_t rowwise = bytes(cls::RED_NONE);
    return rowwise > reduced ? rowwise : reduced;
}

__attribute__((visibility("default")))
int grws_linear_ce_fwd(const void *x, int64_t ldx, const void *w, int64_t ldw, int class_major, const void *labels, int label_bytes,
                       int64_t ignore_index, int64_t rows, int64_t width, int64_t classes, int dtype, int reduction, float *loss,
                       float *state, float *count, void *scratch, size_t scratch_bytes, void *stream) {
    const lce::Problem p = lce::problem(x, ldx, w, ldw, class_major, labels, label_bytes, ignore_index, rows, width, classes, dtype, reduction);
    const int rc = lce::check(p);
    if (rc != GRWS_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GRWS_REQUIRE(reduction == cls::RED_NONE || (loss && count), "null pointer");
    if (rows == 0) {
        if (reduction == cls::RED_NONE) return GRWS_OK;
        cls::loss_sum_kernel<<<1, 32, 0, st>>>(nullptr, 0, reduction, loss, count);
        GRWS_CUDA_TRY(cudaGetLastError());
        return GRWS_OK;
    }
    GRWS_REQUIRE(x && w && labels && loss && state && scratch, "null pointer");
    GRWS_REQUIRE(aligned16(state) && aligned16(scratch), "state and scratch must be 16-byte aligned");
    const lce::Plan q = lce::make_plan(p, false);
    if (scratch_bytes < q.bytes) return fail(GRWS_ERR_SCRATCH, "linear cross entropy scratch too small");
    char *s = static_cast<char *>(scratch);
    float2 *state2 = reinterpret_cast<float2 *>(state);
    switch (dtype) {
        case GRWS_F32: return lce::forward<float>(p, q, loss, state2, count, s, st);
        case GRWS_F16: return lce::forward<__half>(p, q, loss, state2, count, s, st);
        default: return lce::forward<__nv_bfloat16>(p, q, loss, state2, count, s, st);
    }
}

__attribute__((visibility("default")))
int grws_linear_ce_bwd(const void *x, int64_t ldx, const void *w, int64_t ldw, int class_major, const void *labels, int label_bytes,
                       int64_t ignore_index, int64_t rows, int64_t width, int64_t classes, int dtype, int reduction,
                       const float *grad_loss, const float *state, const float *count, void *dx, void *dw, void *scratch,
                       size_t scratch_bytes, void *stream) {
    lce::Problem p = lce::problem(x, ldx, w, ldw, class_major, labels, label_bytes, ignore_index, rows, width, classes, dtype, reduction);
    const int rc = lce::check(p);
    if (rc != GRWS_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (dw) GRWS_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)width * classes * dtype_bytes(dtype), st));
        return GRWS_OK;
    }
    if (!dx && !dw) return GRWS_OK;
    GRWS_REQUIRE(x && w && labels && grad_loss && state && scratch, "null pointer");
    GRWS_REQUIRE(reduction != cls::RED_MEAN || count, "null pointer");
    GRWS_REQUIRE(aligned16(state) && aligned16(scratch), "state and scratch must be 16-byte aligned");
    const lce::Plan q = lce::make_plan(p, true);
    if (scratch_bytes < q.bytes) return fail(GRWS_ERR_SCRATCH, "linear cross entropy scratch too small");
    p.state = reinterpret_cast<const float2 *>(state);
    p.grad = grad_loss;
    p.count = count;
    char *s = static_cast<char *>(scratch);
    switch (dtype) {
        case GRWS_F32: return lce::backward<float>(p, q, dx, dw, s, st);
        case GRWS_F16: return lce::backward<__half>(p, q, dx, dw, s, st);
        default: return lce::backward<__nv_bfloat16>(p, q, dx, dw, s, st);
    }
}

__attribute__((visibility("default")))
int grws_linear_ce_check(void *stream) {
    int *word = nullptr, status = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (int rc = lce::status_word(&word)) return rc;
    GRWS_CUDA_TRY(cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, s));
    GRWS_CUDA_TRY(cudaStreamSynchronize(s));
    if (status == 0) return GRWS_OK;
    GRWS_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), s));
    static const char *const what[] = {"", "operand tiles never arrived", "a stage was never released", "an accumulator was never released",
                                       "a tile was never finished"};
    return fail(GRWS_ERR_DEVICE, "a linear cross entropy launch on this device gave up waiting: %s (code %d); its output is incomplete",
                status >= 1 && status <= 4 ? what[status] : "unknown wait", status);
}

__attribute__((visibility("default")))
int grws_linear_ce_set_wait_limit(long long sm_clocks) {
    GRWS_REQUIRE(sm_clocks >= 0, "negative limit");
    __atomic_store_n(&lce::g_wait_limit, sm_clocks > 0 ? sm_clocks : prod::WAIT_LIMIT_CYCLES, __ATOMIC_RELAXED);
    return GRWS_OK;
}

}  // extern "C"
