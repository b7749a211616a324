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
    const float *label_score;            // [n], behind them
    const float *grad, *count;           // backward: gradient of the loss, number of counted rows
    const float *norm;                   // backward without a reduction: largest |gradient| of a row
    __host__ __device__ int64_t w_k() const { return class_major ? 1 : ldw; }
    __host__ __device__ int64_t w_v() const { return class_major ? ldw : 1; }
};

// largest finite |gradient| of a row: with it a row's factor is at most 1, whatever the scale of the loss
__global__ void __launch_bounds__(1024) grad_norm_kernel(const float *__restrict__ grad, int64_t n, float *__restrict__ norm) {
    __shared__ float red[32];
    float m = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const float g = fabsf(grad[i]);
        if (g < INFINITY) m = fmaxf(m, g);
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

// Joins the parts of the rows' statistics in order and takes the rows' losses; a thread per row.
__global__ void __launch_bounds__(256) rows_kernel(const Problem p, const float2 *__restrict__ part, int parts, const float *__restrict__ label_score,
                                                   float2 *__restrict__ state, float *__restrict__ loss, float *__restrict__ count,
                                                   float2 *__restrict__ partial) {
    __shared__ float red[64];
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    float l = 0.0f, counted = 0.0f;
    if (row < p.n) {
        float m = NEG_INF, s = 0.0f;
        for (int i = 0; i < parts; ++i) {
            const float2 q = part[(int64_t)i * p.n + row];
            join_stats(m, s, q.x, q.y, LOG2E);
        }
        state[row] = make_float2(m, s);
        const int64_t label = load_index(p.labels, p.label_bytes, row);
        if (label != p.ignore_index) {
            l = label >= 0 && label < p.V ? logf(s) - (label_score[row] - m) : NAN;
            counted = 1.0f;
        }
        if (p.reduction == RED_NONE) loss[row] = l;
    }
    if (p.reduction == RED_NONE) return;
    block_sum2(l, counted, red);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) finish_loss(l, counted, p.reduction, loss, count);
        else partial[blockIdx.x] = make_float2(l, counted);
    }
}

// ---------------------------------------------------------------------------------------------
// fp32 arithmetic on the general cores: any stride, any size.  64 x 64 tiles, 16 deep, 4 x 4 a thread.
// ---------------------------------------------------------------------------------------------
constexpr int TM = 64, TN = 64, TK = 16, PAD = 4;

struct Tiles { float a[TK][TM + PAD], b[TK][TN + PAD]; };

template <typename TA, typename TB>
__device__ __forceinline__ void tile_product(const TA *A, int64_t am, int64_t ak, const TB *B, int64_t bk, int64_t bn, int64_t M, int64_t N,
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
            t.a[ak_i][am_i] = ma < M && ka < k1 ? to_float(A[ma * am + ka * ak]) : 0.0f;
            t.b[bk_i][bn_i] = nb < N && kb < k1 ? to_float(B[kb * bk + nb * bn]) : 0.0f;
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
template <typename T> __global__ void __launch_bounds__(256) plain_stats_kernel(const Problem p, float2 *__restrict__ part, float *__restrict__ label_score) {
    __shared__ __align__(16) Tiles t;
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
        tile_product(static_cast<const T *>(p.x), p.ldx, (int64_t)1, static_cast<const T *>(p.w), p.w_k(), p.w_v(), p.n, p.V, m0, n0, 0, p.d, t, acc);
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
template <typename T> __global__ void __launch_bounds__(256) plain_grad_kernel(const Problem p, int64_t v0, int64_t cols, float *__restrict__ G, int64_t ldg) {
    __shared__ __align__(16) Tiles t;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int64_t m0 = (int64_t)blockIdx.x * TM, n0 = (int64_t)blockIdx.y * TN;
    float acc[4][4];
    tile_product(static_cast<const T *>(p.x), p.ldx, (int64_t)1, static_cast<const T *>(p.w) + v0 * p.w_v(), p.w_k(), p.w_v(), p.n, cols, m0, n0, 0, p.d, t, acc);
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

// part blockIdx.z of the product A [M, K] B [K, N] into (or onto) its own plane of fp32 partial sums [parts][M][N]
template <typename TA, typename TB>
__global__ void __launch_bounds__(256) plain_product_kernel(const TA *A, int64_t am, int64_t ak, const TB *B, int64_t bk, int64_t bn, int64_t M, int64_t N,
                                                            int64_t K, int64_t k_part, float *__restrict__ out, int add) {
    __shared__ __align__(16) Tiles t;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int64_t m0 = (int64_t)blockIdx.x * TM, n0 = (int64_t)blockIdx.y * TN, k0 = (int64_t)blockIdx.z * k_part;
    float acc[4][4];
    tile_product(A, am, ak, B, bk, bn, M, N, m0, n0, k0, min(K, k0 + k_part), t, acc);
    out += (int64_t)blockIdx.z * M * N;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= M || n >= N) continue;
            float *o = out + m * N + n;
            *o = add ? *o + acc[i][j] : acc[i][j];
        }
}

// out(m, n) = alpha * sum of the partial planes in order, rounded once to the output's type; out(m, n) at m * om + n * on
template <typename T> __global__ void __launch_bounds__(256) round_kernel(const Problem p, const float *__restrict__ part, int parts, int64_t M, int64_t N,
                                                                          float scale, T *__restrict__ out, int64_t om, int64_t on) {
    const float alpha = prod::grad_alpha(p) * scale;
    const int64_t total = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int k = 0; k < parts; ++k) s += part[k * total + i];
        const int64_t m = i / N, n = i - m * N;
        out[m * om + n * on] = from_float<T>(s * alpha);
    }
}

// Operand for the tensor cores from one whose rows no TMA copy can start at (or of fp32: three bf16 planes): rows of `ldp`
// elements, a multiple of 8.  A thread per 8 elements.
template <typename T> __global__ void __launch_bounds__(256) pack_kernel(const T *__restrict__ src, int64_t ld, int64_t rows, int64_t cols,
                                                                         uint16_t *__restrict__ dst, int64_t ldp, int64_t plane) {
    const int64_t per_row = ldp / 8, total = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, c = (i - row * per_row) * 8;
        const T *s = src + row * ld + c;
        uint16_t *d = dst + row * ldp + c;
        if constexpr (sizeof(T) == 2) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t lo = c + 2 * j < cols ? reinterpret_cast<const uint16_t *>(s)[2 * j] : 0;
                const uint32_t hi = c + 2 * j + 1 < cols ? reinterpret_cast<const uint16_t *>(s)[2 * j + 1] : 0;
                q[j] = lo | hi << 16;
            }
            *reinterpret_cast<uint4 *>(d) = make_uint4(q[0], q[1], q[2], q[3]);
        } else {
            uint32_t q[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float a[2], b[2], e[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) prod::split3(c + 2 * j + h < cols ? to_float(s[2 * j + h]) : 0.0f, a[h], b[h], e[h]);
                q[0][j] = prod::pack2(a[0], a[1], 1);
                q[1][j] = prod::pack2(b[0], b[1], 1);
                q[2][j] = prod::pack2(e[0], e[1], 1);
            }
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4 *>(d + k * plane) = make_uint4(q[k][0], q[k][1], q[k][2], q[k][3]);
        }
    }
}

// Worst status of a tensor-core launch on this device since it was last read
static __device__ int g_status;

// ---------------------------------------------------------------------------------------------
// plan: how a call is cut up, and where its workspace lies
// ---------------------------------------------------------------------------------------------
constexpr size_t PIECE_BYTES = 256ull << 20;       // workspace for G
constexpr double TENSOR_PRODUCTS = 1 << 22;        // n d V from which the tensor cores take the call

struct Plan {
    bool tensor;
    int planes;                                    // of an operand: 1, or 3 of bf16 for fp32
    bool pack_x, pack_w;
    int64_t ldx, ldw, ldg;                         // rows of the operands as the tensor cores read them
    int64_t run, parts;                            // forward: class tiles per unit, parts of the class axis
    int64_t piece;                                 // backward: classes per piece
    int64_t dx_parts, dx_len, dw_parts, dw_len;    // parts of the two products' inner axes (classes of a piece, rows)
    size_t x, w;                                   // packed operands
    size_t stats, partial;                         // forward scratch
    size_t norm, G, dx_sum, dw_sum;                // backward scratch
    size_t bytes;
};

static size_t place(size_t &at, size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
}
// parts of an inner axis of K so that `tiles` output tiles give every SM two blocks; none shorter than `least`
static void cut(int64_t tiles, int64_t K, int64_t least, int64_t unit, int64_t *parts, int64_t *len) {
    int64_t s = ceil_div((int64_t)sm_count() * 2, tiles > 0 ? tiles : 1);
    if (s > K / least) s = K / least;
    if (s < 1) s = 1;
    *len = ceil_div(ceil_div(K > 0 ? K : 1, s), unit) * unit;
    *parts = ceil_div(K > 0 ? K : 1, *len);
}

static int columns_per_tile(int64_t N, int cg) {
    const int64_t tiles = ceil_div(N, (int64_t)prod::BN);
    return (int)(ceil_div(ceil_div(N, tiles), (int64_t)(32 * cg)) * 32 * cg);
}
// CTAs that share a tile: pairs where there are more rows than one CTA's
static int cta_group(int64_t M) { return M > prod::BM ? 2 : 1; }

static bool needs_packing(const void *p, int64_t ld, int dtype) { return dtype == GRWS_F32 || !aligned16(p) || ld % 8 != 0; }

// Class tiles that one unit of the forward pass takes: as many as leave the SMs equally busy to a few per cent
static void cut_runs(int64_t m_tiles, int64_t n_tiles, int64_t ctas, int64_t *run, int64_t *runs) {
    int64_t best = 1;
    double best_cost = 1e300;
    for (int64_t r = 1; r <= n_tiles && r <= 64; ++r) {
        const int64_t k = ceil_div(n_tiles, r);
        const double cost = (double)ceil_div(m_tiles * k, ctas) * (double)r + 0.05 * (double)k;      // a part costs a write and a read per row
        if (cost <= best_cost) { best_cost = cost; best = r; }
    }
    *run = best;
    *runs = ceil_div(n_tiles, best);
}

// Parts of the inner axes of dx (classes of a piece) and dw (rows), which run in one launch: a unit should be short against the
// launch, since units are dealt out round robin, but every part is one more plane of fp32 sums through memory.  In units of one
// 64-element step of one tile: about 0.4 us of a pair of SMs.
static void cut_products(int64_t tiles0, int64_t k0, double sums0, int64_t tiles1, int64_t k1, double sums1, int64_t ctas, int64_t *parts0, int64_t *parts1) {
    static const int64_t tries[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128};
    double best = 1e300;
    for (int64_t a : tries) {
        if (a > 1 && k0 / a < 8) break;
        for (int64_t b : tries) {
            if (b > 1 && k1 / b < 8) break;
            const int64_t l0 = ceil_div(k0, a), l1 = ceil_div(k1, b), units = tiles0 * a + tiles1 * b;
            const double all = (double)(tiles0 * k0 + tiles1 * k1) / (double)ctas;
            const double longest = (double)(l0 > l1 ? l0 : l1);
            const double rounds = (double)ceil_div(units, ctas) * ((double)(tiles0 * k0 + tiles1 * k1) / (double)units);
            double cost = rounds > all ? rounds : all;
            if (cost < longest) cost = longest;
            cost += ((a > 1 ? (double)a * sums0 : 0.0) + (b > 1 ? (double)b * sums1 : 0.0)) * 8.0 / 6.0e12 / 0.4e-6;
            if (cost < best) { best = cost; *parts0 = a; *parts1 = b; }
        }
    }
}

static Plan make_plan(const Problem &p, bool backward) {
    Plan q = {};
    const int64_t n = p.n, d = p.d, V = p.V;
    q.tensor = (double)n * (double)d * (double)V >= TENSOR_PRODUCTS;
    size_t at = 0;
    if (!q.tensor) {
        const int64_t row_tiles = ceil_div(n, (int64_t)TM), class_tiles = ceil_div(V, (int64_t)TN), width_tiles = ceil_div(d, (int64_t)TN);
        if (!backward) {
            q.parts = ceil_div((int64_t)sm_count() * 2, row_tiles > 0 ? row_tiles : 1);
            if (q.parts > class_tiles) q.parts = class_tiles;
            q.stats = place(at, (size_t)q.parts * n * sizeof(float2));
            q.partial = place(at, (size_t)ceil_div(n, (int64_t)256) * sizeof(float2));
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
    q.planes = p.dtype == GRWS_F32 ? 3 : 1;
    const int64_t w_rows = p.class_major ? V : d, w_cols = p.class_major ? d : V;
    q.pack_x = needs_packing(p.x, p.ldx, p.dtype);
    q.pack_w = needs_packing(p.w, p.ldw, p.dtype);
    q.ldx = q.pack_x ? ceil_div(d, (int64_t)8) * 8 : p.ldx;
    q.ldw = q.pack_w ? ceil_div(w_cols, (int64_t)8) * 8 : p.ldw;
    if (q.pack_x) q.x = place(at, (size_t)q.planes * n * q.ldx * 2);
    if (q.pack_w) q.w = place(at, (size_t)q.planes * w_rows * q.ldw * 2);
    const int cg = cta_group(n);
    if (!backward) {
        const int64_t bn = columns_per_tile(V, cg);
        cut_runs(ceil_div(n, (int64_t)(prod::BM * cg)), ceil_div(V, bn), sm_count() / cg, &q.run, &q.parts);
        q.stats = place(at, (size_t)q.parts * 2 * n * sizeof(float2));
        q.partial = place(at, (size_t)ceil_div(n, (int64_t)256) * sizeof(float2));
    } else {
        q.piece = (int64_t)(PIECE_BYTES / (2 * q.planes)) / n / prod::BN * prod::BN;
        if (q.piece < prod::BN) q.piece = prod::BN;
        if (q.piece > V) q.piece = V;
        q.ldg = ceil_div(q.piece, (int64_t)8) * 8;
        const int pg = cta_group(n > d ? n : d);
        const int64_t rows0 = n, cols0 = d, rows1 = p.class_major ? q.piece : d, cols1 = p.class_major ? d : q.piece;
        const int64_t tiles0 = ceil_div(rows0, (int64_t)(prod::BM * pg)) * ceil_div(cols0, (int64_t)columns_per_tile(cols0, pg));
        const int64_t tiles1 = ceil_div(rows1, (int64_t)(prod::BM * pg)) * ceil_div(cols1, (int64_t)columns_per_tile(cols1, pg));
        const int64_t k0 = ceil_div(q.piece, (int64_t)prod::BK), k1 = ceil_div(n, (int64_t)prod::BK);
        cut_products(tiles0, k0, (double)rows0 * cols0, tiles1, k1, (double)rows1 * cols1, sm_count() / pg, &q.dx_parts, &q.dw_parts);
        q.dx_len = ceil_div(k0, q.dx_parts);
        q.dx_parts = ceil_div(k0, q.dx_len);
        q.dw_len = ceil_div(k1, q.dw_parts);
        q.dw_parts = ceil_div(k1, q.dw_len);
        q.norm = place(at, sizeof(float));
        q.G = place(at, (size_t)q.planes * n * q.ldg * 2);
        if (q.dx_parts > 1 || q.piece < V) q.dx_sum = place(at, (size_t)q.dx_parts * n * d * sizeof(float));
        if (q.dw_parts > 1) q.dw_sum = place(at, (size_t)q.dw_parts * d * q.piece * sizeof(float));
    }
    q.bytes = at;
    return q;
}

template <typename T> static int launch_round(const Problem &p, const float *part, int64_t parts, int64_t M, int64_t N, float scale, void *out, int64_t om,
                                              int64_t on, cudaStream_t st) {
    int64_t g = ceil_div(M * N, (int64_t)256);
    const int64_t most = (int64_t)sm_count() * 8;
    if (g > most) g = most;
    round_kernel<T><<<(unsigned)g, 256, 0, st>>>(p, part, (int)parts, M, N, scale, static_cast<T *>(out), om, on);
    GRWS_CUDA_TRY(cudaGetLastError());
    return GRWS_OK;
}

// ---- the tensor cores' way ----
struct Operands { const void *x, *w; int64_t ldx, ldw, x_plane, w_plane, w_rows, w_cols; };

template <typename T> static int launch_pack(const void *src, int64_t ld, int64_t rows, int64_t cols, void *dst, int64_t ldp, cudaStream_t st) {
    int64_t g = ceil_div(rows * (ldp / 8), (int64_t)256);
    const int64_t most = (int64_t)sm_count() * 8;
    if (g > most) g = most;
    pack_kernel<T><<<(unsigned)g, 256, 0, st>>>(static_cast<const T *>(src), ld, rows, cols, static_cast<uint16_t *>(dst), ldp, rows * ldp);
    GRWS_CUDA_TRY(cudaGetLastError());
    return GRWS_OK;
}

template <typename T> static int pack_operands(const Problem &p, const Plan &q, char *scratch, Operands *o, cudaStream_t st) {
    o->w_rows = p.class_major ? p.V : p.d;
    o->w_cols = p.class_major ? p.d : p.V;
    o->x = q.pack_x ? scratch + q.x : p.x;
    o->w = q.pack_w ? scratch + q.w : p.w;
    o->ldx = q.ldx; o->ldw = q.ldw;
    o->x_plane = p.n * q.ldx;
    o->w_plane = o->w_rows * q.ldw;
    if (q.pack_x) if (int rc = launch_pack<T>(p.x, p.ldx, p.n, p.d, scratch + q.x, q.ldx, st)) return rc;
    if (q.pack_w) if (int rc = launch_pack<T>(p.w, p.ldw, o->w_rows, o->w_cols, scratch + q.w, q.ldw, st)) return rc;
    return GRWS_OK;
}

// sets a product up: its tile counts, and the maps of its operands ([rows][cols] in memory, cols contiguous)
static int set_task(prod::Task *t, CUtensorMap *ma, CUtensorMap *mb, int cg, int bf16, int planes, const void *a, int64_t a_rows, int64_t a_cols, int64_t lda,
                    int64_t a_plane, int a_outer, const void *b, int64_t b_rows, int64_t b_cols, int64_t ldb, int64_t b_plane, int b_outer, int64_t M, int64_t N,
                    int64_t K) {
    t->M = M; t->N = N;
    t->bn = columns_per_tile(N, cg);
    t->m_tiles = (int)ceil_div(M, (int64_t)(prod::BM * cg));
    t->n_tiles = (int)ceil_div(N, (int64_t)t->bn);
    t->run = 1; t->runs = t->n_tiles; t->splits = 1;
    t->k_blocks = t->k_len = (int)ceil_div(K, (int64_t)prod::BK);
    t->group = t->m_tiles < 16 ? t->m_tiles : 16;
    t->a_outer = a_outer; t->b_outer = b_outer;
    if (int rc = prod::encode_map(ma, a, bf16, a_cols, a_rows, lda, planes, a_plane, a_outer ? prod::BK : prod::BM)) return rc;
    return prod::encode_map(mb, b, bf16, b_cols, b_rows, ldb, planes, b_plane, b_outer ? prod::BK : prod::BN / cg);
}

static int product_params(const Problem &p, const Plan &q, prod::Params *r) {
    void *status = nullptr;
    GRWS_CUDA_TRY(cudaGetSymbolAddress(&status, g_status));
    *r = prod::Params{};
    r->tasks = 1;
    r->pairs = q.planes == 3 ? 6 : 1;
    r->bf16 = p.dtype != GRWS_F16;
    r->labels = p.labels; r->label_bytes = p.label_bytes; r->ignore_index = p.ignore_index; r->V = p.V;
    r->reduction = p.reduction; r->grad = p.grad; r->count = p.count; r->norm = p.norm;
    r->state = p.state;
    r->scale = 1.0f;
    r->status = static_cast<int *>(status);
    r->wait_limit = prod::WAIT_LIMIT_CYCLES;
    return GRWS_OK;
}

template <int MODE> static int launch_grouped(int cg, const prod::Maps &maps, const prod::Params &r, cudaStream_t st) {
    return cg == 2 ? prod::launch_product<2, MODE>(maps, r, st) : prod::launch_product<1, MODE>(maps, r, st);
}

template <typename T> static int tensor_forward(const Problem &p, const Plan &q, float2 *part, float *label_score, char *scratch, cudaStream_t st) {
    Operands o;
    if (int rc = pack_operands<T>(p, q, scratch, &o, st)) return rc;
    prod::Params r;
    if (int rc = product_params(p, q, &r)) return rc;
    prod::Maps maps;
    const int cg = cta_group(p.n);
    if (int rc = set_task(&r.task[0], &maps.a[0], &maps.b[0], cg, r.bf16, q.planes, o.x, p.n, p.d, o.ldx, o.x_plane, 0, o.w, o.w_rows, o.w_cols, o.ldw, o.w_plane,
                          !p.class_major, p.n, p.V, p.d)) return rc;
    r.task[0].run = (int)q.run;
    r.task[0].runs = (int)q.parts;
    r.part = part;
    r.label_score = label_score;
    return launch_grouped<prod::STATS>(cg, maps, r, st);
}

// G in fp16 is held as 2^12 G: |G| <= 1, and a probability of 2^-26 is still a normal number
static float stored_scale(const Problem &p) { return p.dtype == GRWS_F16 ? 4096.0f : 1.0f; }

template <typename T> static int tensor_backward(const Problem &p, const Plan &q, void *dx, void *dw, char *scratch, cudaStream_t st) {
    Operands o;
    if (int rc = pack_operands<T>(p, q, scratch, &o, st)) return rc;
    void *G = scratch + q.G;
    float *dx_sum = reinterpret_cast<float *>(scratch + q.dx_sum), *dw_sum = reinterpret_cast<float *>(scratch + q.dw_sum);
    const int64_t g_plane = p.n * q.ldg;
    const bool sum_dx = q.dx_parts > 1 || q.piece < p.V;
    for (int64_t v0 = 0; v0 < p.V; v0 += q.piece) {
        const int64_t cols = p.V - v0 < q.piece ? p.V - v0 : q.piece;
        prod::Params r;
        if (int rc = product_params(p, q, &r)) return rc;
        prod::Maps maps;
        const int cg = cta_group(p.n);
        if (int rc = set_task(&r.task[0], &maps.a[0], &maps.b[0], cg, r.bf16, q.planes, o.x, p.n, p.d, o.ldx, o.x_plane, 0, o.w, o.w_rows, o.w_cols, o.ldw,
                              o.w_plane, !p.class_major, p.n, cols, p.d)) return rc;
        r.task[0].b_row0 = (int)v0;
        r.v0 = v0;
        r.label_score = const_cast<float *>(p.label_score);
        r.scale = stored_scale(p);
        r.G = G; r.ldg = q.ldg; r.plane = g_plane;
        if (int rc = launch_grouped<prod::GRAD>(cg, maps, r, st)) return rc;

        if (int rc = product_params(p, q, &r)) return rc;
        r.scale = 1.0f / stored_scale(p);
        r.tasks = 0;
        const int pg = cta_group(p.n > p.d ? p.n : p.d);
        int64_t dw_parts = 1;
        if (dw) {
            prod::Task *t = &r.task[r.tasks];
            // [d, V]: x^T G; [V, d]: G^T x
            const int64_t M = p.class_major ? cols : p.d, N = p.class_major ? p.d : cols;
            int rc;
            if (p.class_major)
                rc = set_task(t, &maps.a[r.tasks], &maps.b[r.tasks], pg, r.bf16, q.planes, G, p.n, cols, q.ldg, g_plane, 1, o.x, p.n, p.d, o.ldx, o.x_plane, 1, M, N, p.n);
            else
                rc = set_task(t, &maps.a[r.tasks], &maps.b[r.tasks], pg, r.bf16, q.planes, o.x, p.n, p.d, o.ldx, o.x_plane, 1, G, p.n, cols, q.ldg, g_plane, 1, M, N, p.n);
            if (rc != GRWS_OK) return rc;
            t->k_len = (int)q.dw_len;
            t->splits = (int)(dw_parts = q.dw_parts);
            t->sum = dw_sum;
            t->out_dtype = p.dtype;
            t->ldo = p.class_major ? p.d : p.V;
            if (dw_parts == 1) t->out = static_cast<T *>(dw) + (p.class_major ? v0 * p.d : v0);
            ++r.tasks;
        }
        if (dx) {
            prod::Task *t = &r.task[r.tasks];
            if (int rc = set_task(t, &maps.a[r.tasks], &maps.b[r.tasks], pg, r.bf16, q.planes, G, p.n, cols, q.ldg, g_plane, 0, o.w, o.w_rows, o.w_cols, o.ldw,
                                  o.w_plane, p.class_major, p.n, p.d, cols)) return rc;
            t->b_k0 = (int)v0;
            t->k_len = (int)q.dx_len;
            t->splits = (int)ceil_div((int64_t)t->k_blocks, q.dx_len);      // (a last, shorter piece has fewer)
            t->sum = dx_sum;
            t->add = v0 > 0;
            t->out_dtype = p.dtype;
            t->ldo = p.d;
            if (!sum_dx) t->out = dx;
            ++r.tasks;
        }
        if (int rc = launch_grouped<prod::SUM>(pg, maps, r, st)) return rc;
        if (dw && dw_parts > 1) {
            const int64_t M = p.class_major ? cols : p.d, N = p.class_major ? p.d : cols, ld = p.class_major ? p.d : p.V;
            if (int rc = launch_round<T>(p, dw_sum, dw_parts, M, N, r.scale, static_cast<T *>(dw) + (p.class_major ? v0 * p.d : v0), ld, 1, st)) return rc;
        }
    }
    return dx && sum_dx ? launch_round<T>(p, dx_sum, q.dx_parts, p.n, p.d, 1.0f / stored_scale(p), dx, p.d, 1, st) : GRWS_OK;
}

template <typename T> static int forward(const Problem &p, const Plan &q, float *loss, float2 *state, float *label_score, float *count, char *scratch,
                                         cudaStream_t st) {
    float2 *part = reinterpret_cast<float2 *>(scratch + q.stats), *partial = reinterpret_cast<float2 *>(scratch + q.partial);
    if (q.tensor) {
        if (int rc = tensor_forward<T>(p, q, part, label_score, scratch, st)) return rc;
    } else {
        plain_stats_kernel<T><<<dim3((unsigned)ceil_div(p.n, (int64_t)TM), (unsigned)q.parts), 256, 0, st>>>(p, part, label_score);
        GRWS_CUDA_TRY(cudaGetLastError());
    }
    const int64_t blocks = ceil_div(p.n, (int64_t)256);
    rows_kernel<<<(unsigned)blocks, 256, 0, st>>>(p, part, (int)(q.tensor ? 2 * q.parts : q.parts), label_score, state, loss, count, partial);
    GRWS_CUDA_TRY(cudaGetLastError());
    if (p.reduction != RED_NONE && blocks > 1) {
        loss_sum_kernel<<<1, 512, 0, st>>>(partial, (int)blocks, p.reduction, loss, count);
        GRWS_CUDA_TRY(cudaGetLastError());
    }
    return GRWS_OK;
}

template <typename T> static int backward(Problem p, const Plan &q, void *dx, void *dw, char *scratch, cudaStream_t st) {
    float *G = reinterpret_cast<float *>(scratch + q.G), *dx_sum = reinterpret_cast<float *>(scratch + q.dx_sum);
    float *dw_sum = reinterpret_cast<float *>(scratch + q.dw_sum), *norm = reinterpret_cast<float *>(scratch + q.norm);
    if (p.reduction == RED_NONE) {
        grad_norm_kernel<<<1, 1024, 0, st>>>(p.grad, p.n, norm);
        GRWS_CUDA_TRY(cudaGetLastError());
        p.norm = norm;
    }
    if (q.tensor) return tensor_backward<T>(p, q, dx, dw, scratch, st);
    const unsigned row_tiles = (unsigned)ceil_div(p.n, (int64_t)TM), width_tiles = (unsigned)ceil_div(p.d, (int64_t)TN);
    const T *x = static_cast<const T *>(p.x), *w = static_cast<const T *>(p.w);
    for (int64_t v0 = 0; v0 < p.V; v0 += q.piece) {
        const int64_t cols = p.V - v0 < q.piece ? p.V - v0 : q.piece;
        const unsigned class_tiles = (unsigned)ceil_div(cols, (int64_t)TN);
        plain_grad_kernel<T><<<dim3(row_tiles, class_tiles), 256, 0, st>>>(p, v0, cols, G, q.piece);
        GRWS_CUDA_TRY(cudaGetLastError());
        if (dx) {
            plain_product_kernel<float, T><<<dim3(row_tiles, width_tiles, (unsigned)q.dx_parts), 256, 0, st>>>(
                G, q.piece, (int64_t)1, w + v0 * p.w_v(), p.w_v(), p.w_k(), p.n, p.d, cols, q.dx_len, dx_sum, v0 > 0);
            GRWS_CUDA_TRY(cudaGetLastError());
        }
        if (dw) {
            plain_product_kernel<T, float><<<dim3(width_tiles, class_tiles, (unsigned)q.dw_parts), 256, 0, st>>>(
                x, (int64_t)1, p.ldx, G, q.piece, (int64_t)1, p.d, cols, p.n, q.dw_len, dw_sum, 0);
            GRWS_CUDA_TRY(cudaGetLastError());
            const int64_t ok = p.class_major ? 1 : p.V, ov = p.class_major ? p.d : 1;
            const int rc = launch_round<T>(p, dw_sum, q.dw_parts, p.d, cols, 1.0f, static_cast<T *>(dw) + v0 * ov, ok, ov, st);
            if (rc != GRWS_OK) return rc;
        }
    }
    return dx ? launch_round<T>(p, dx_sum, q.dx_parts, p.n, p.d, 1.0f, dx, p.d, 1, st) : GRWS_OK;
}

static int check(const Problem &p) {
    GRWS_REQUIRE(p.n >= 0 && p.d > 0 && p.V > 0, "bad size (rows = %lld, width = %lld, classes = %lld)", (long long)p.n, (long long)p.d, (long long)p.V);
    GRWS_REQUIRE(p.n <= INT32_MAX && p.d <= INT32_MAX && p.V <= INT32_MAX, "rows, width and classes must fit 31 bits");
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
    return lce::make_plan(lce::problem(x, ldx, w, ldw, class_major, nullptr, 8, 0, rows, width, classes, dtype, 0), backward != 0).bytes;
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
    float *label_score = state + 2 * rows;
    switch (dtype) {
        case GRWS_F32: return lce::forward<float>(p, q, loss, state2, label_score, count, s, st);
        case GRWS_F16: return lce::forward<__half>(p, q, loss, state2, label_score, count, s, st);
        default: return lce::forward<__nv_bfloat16>(p, q, loss, state2, label_score, count, s, st);
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
    p.label_score = state + 2 * rows;
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
    void *word = nullptr;
    int status = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    GRWS_CUDA_TRY(cudaGetSymbolAddress(&word, lce::g_status));
    GRWS_CUDA_TRY(cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, s));
    GRWS_CUDA_TRY(cudaStreamSynchronize(s));
    if (status == 0) return GRWS_OK;
    GRWS_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), s));
    static const char *const what[] = {"", "operand tiles never arrived", "a stage was never released", "an accumulator was never released",
                                       "a tile was never finished"};
    return fail(GRWS_ERR_DEVICE, "a linear cross entropy launch on this device gave up waiting: %s (code %d); its output is incomplete",
                status >= 1 && status <= 4 ? what[status] : "unknown wait", status);
}

}  // extern "C"
