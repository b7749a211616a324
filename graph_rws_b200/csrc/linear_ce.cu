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
#include "class_loss.cuh"

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
    const float *norm;                   // backward without a reduction: largest |gradient| of a row
    __host__ __device__ int64_t w_k() const { return class_major ? 1 : ldw; }
    __host__ __device__ int64_t w_v() const { return class_major ? ldw : 1; }
};

// 0 for an ignored row, NaN for a label that is no class
__device__ __forceinline__ float row_factor(const Problem &p, int64_t row, int64_t label) {
    if (label == p.ignore_index) return 0.0f;
    if (label < 0 || label >= p.V) return NAN;
    if (p.reduction != RED_NONE) return 1.0f;
    const float norm = __ldg(p.norm);
    return norm > 0.0f ? __ldg(p.grad + row) / norm : __ldg(p.grad + row);
}
__device__ __forceinline__ float alpha_of(const Problem &p) {
    if (p.reduction != RED_NONE) return loss_factor(p.grad, p.count, p.reduction);
    const float norm = __ldg(p.norm);
    return norm > 0.0f ? norm : 1.0f;
}

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
        const float r = row_factor(p, row, label);
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
    const float alpha = alpha_of(p) * scale;
    const int64_t total = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int k = 0; k < parts; ++k) s += part[k * total + i];
        const int64_t m = i / N, n = i - m * N;
        out[m * om + n * on] = from_float<T>(s * alpha);
    }
}

// ---------------------------------------------------------------------------------------------
// plan: how a call is cut up, and where its workspace lies
// ---------------------------------------------------------------------------------------------
constexpr size_t PIECE_BYTES = 256ull << 20;       // workspace for G

struct Plan {
    int64_t parts;                                 // forward: parts of the class axis
    int64_t piece;                                 // backward: classes per piece
    int64_t dx_parts, dx_len, dw_parts, dw_len;    // parts of the two products' inner axes (classes of a piece, rows)
    size_t stats, label_score, partial;            // forward scratch
    size_t norm, G, dx_sum, dw_sum;                // backward scratch
    size_t fwd_bytes, bwd_bytes;
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

static Plan make_plan(int64_t n, int64_t d, int64_t V) {
    Plan q = {};
    const int64_t row_tiles = ceil_div(n, (int64_t)TM), class_tiles = ceil_div(V, (int64_t)TN), width_tiles = ceil_div(d, (int64_t)TN);
    q.parts = ceil_div((int64_t)sm_count() * 2, row_tiles > 0 ? row_tiles : 1);
    if (q.parts > class_tiles) q.parts = class_tiles;
    size_t at = 0;
    q.stats = place(at, (size_t)q.parts * n * sizeof(float2));
    q.label_score = place(at, (size_t)n * sizeof(float));
    q.partial = place(at, (size_t)ceil_div(n, (int64_t)256) * sizeof(float2));
    q.fwd_bytes = at;
    q.piece = (int64_t)(PIECE_BYTES / sizeof(float)) / (n > 0 ? n : 1) / TN * TN;
    if (q.piece < TN) q.piece = TN;
    if (q.piece > 32768) q.piece = 32768;           // (a grid has at most 65,535 tiles in y)
    if (q.piece > V) q.piece = V;
    cut(row_tiles * width_tiles, q.piece, 128, TK, &q.dx_parts, &q.dx_len);
    cut(width_tiles * ceil_div(q.piece, (int64_t)TN), n, 128, TK, &q.dw_parts, &q.dw_len);
    at = 0;
    q.norm = place(at, sizeof(float));
    q.G = place(at, (size_t)n * q.piece * sizeof(float));
    q.dx_sum = place(at, (size_t)q.dx_parts * n * d * sizeof(float));
    q.dw_sum = place(at, (size_t)q.dw_parts * d * q.piece * sizeof(float));
    q.bwd_bytes = at;
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

template <typename T> static int forward(const Problem &p, const Plan &q, float *loss, float2 *state, float *count, char *scratch, cudaStream_t st) {
    float2 *part = reinterpret_cast<float2 *>(scratch + q.stats), *partial = reinterpret_cast<float2 *>(scratch + q.partial);
    float *label_score = reinterpret_cast<float *>(scratch + q.label_score);
    plain_stats_kernel<T><<<dim3((unsigned)ceil_div(p.n, (int64_t)TM), (unsigned)q.parts), 256, 0, st>>>(p, part, label_score);
    GRWS_CUDA_TRY(cudaGetLastError());
    const int64_t blocks = ceil_div(p.n, (int64_t)256);
    rows_kernel<<<(unsigned)blocks, 256, 0, st>>>(p, part, (int)q.parts, label_score, state, loss, count, partial);
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
    (void)x; (void)ldx; (void)w; (void)ldw; (void)class_major; (void)dtype;
    if (rows <= 0 || width <= 0 || classes <= 0) return 0;
    const lce::Plan q = lce::make_plan(rows, width, classes);
    return backward ? q.bwd_bytes : q.fwd_bytes;
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
    const lce::Plan q = lce::make_plan(rows, width, classes);
    if (scratch_bytes < q.fwd_bytes) return fail(GRWS_ERR_SCRATCH, "linear cross entropy scratch too small");
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
    const lce::Plan q = lce::make_plan(rows, width, classes);
    if (scratch_bytes < q.bwd_bytes) return fail(GRWS_ERR_SCRATCH, "linear cross entropy scratch too small");
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

}  // extern "C"
