// Distillation from a teacher's best scores.  A row of student scores z [V] is compared with K kept teacher scores t and their
// class ids at temperature T:
//
//     p_j = softmax_j(t_j / T) over the row's entries (id >= 0),   log q_v = z_v / T - log sum_v exp(z_v / T)
//     loss = T^2 sum_j p_j (log p_j - log q_id(j)),                dz_v = g T (q_v - sum of p_j with id(j) = v)
//
// Forward is one pass over z with a running maximum and sum, backward one pass that reads z and writes dz: both are bound by
// memory.  A row's state (maximum and sum of z, of t) goes from one to the other as four floats.  The maximum is kept apart
// from the sum because z - max is exact where q is large, z / T - log sum would round at the size of z.
//
// Rows are walked in 16-byte pieces from the first aligned address on; what is before and behind them is read and written
// element by element, so that rows of any length, stride and offset work and nothing outside of a row is touched.
#include "class_loss.cuh"

namespace grws {
namespace distill {

using namespace cls;

constexpr int MAX_KEPT = 1024;
constexpr int THREADS = 256;
constexpr int CTAS_PER_SM = 8;
constexpr int SHORT_ROW_BYTES = 32768;   // rows up to which a group of lanes may take one
constexpr int SHORT_KEPT = 64;           // entries that such a group holds in shared memory
constexpr int LONG_HELD = 2;             // entries per lane of the warp that takes a long row's loss, loaded ahead
constexpr int SPLIT_MIN = 4096;          // classes below which a row is not cut any further

struct Args {
    const void *z; int ldz;              // 32-bit sizes and strides: a 64-bit product of two of them is one instruction
    const void *t; int ldt, t_dtype;
    const void *ids; int ldi, id_bytes;
    int n, V, K;
    float c;                             // log2(e) / T
    float T;
    int reduction;
    float *loss;                         // forward: [n] (no reduction)
    float4 *state;                       // [n]: max z, sum exp((z - max) / T), max t, sum exp((t - max) / T); sum of t 0: no entry
    float2 *partial;                     // [grid] sums of (loss, counted rows)
    float2 *stats;                       // [splits][n] of rows cut into parts
    int splits, part;                    // parts of a row and their length
    const float *grad, *count;           // backward
    void *dz; int ldo;
};

__device__ __forceinline__ float teacher_at(const Args &a, int row, int j) {
    const int64_t i = (int64_t)row * a.ldt + j;
    if (a.t_dtype == GRWS_F32) return static_cast<const float *>(a.t)[i];
    if (a.t_dtype == GRWS_F16) return to_float(static_cast<const __half *>(a.t)[i]);
    return to_float(static_cast<const __nv_bfloat16 *>(a.t)[i]);
}
__device__ __forceinline__ int64_t id_at(const Args &a, int row, int j) { return load_index(a.ids, a.id_bytes, (int64_t)row * a.ldi + j); }

template <int L> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o, L));
    return v;
}
template <int L> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, L);
    return v;
}

// `len` elements at p: those before the first aligned address, whole pieces, the rest
template <typename T> struct Span {
    const T *p;
    int head, pieces, tail;
    __device__ __forceinline__ Span(const T *start, int len) : p(start) {
        constexpr int E = Piece<T>::E;
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15u) / (int)sizeof(T);
        head = min((E - off) & (E - 1), len);
        pieces = (len - head) / E;
        tail = len - head - pieces * E;
    }
    __device__ __forceinline__ const uint4 *body() const { return reinterpret_cast<const uint4 *>(p + head); }
    __device__ __forceinline__ const T *rest() const { return p + head + pieces * Piece<T>::E; }
};

// U pieces of a span per lane, -inf behind its end
template <typename T, int U> struct Batch { uint4 u[U]; };
template <typename T, int U> __device__ __forceinline__ void load_batch(Batch<T, U> &b, const uint4 *body, int k, int lanes, int pieces) {
    constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int i = 0; i < U; ++i) b.u[i] = k + i * lanes < pieces ? body[k + i * lanes] : make_uint4(none, none, none, none);
}

// What a lane needs of a row before it can do anything is asked for in one go: its first U pieces, its part of the elements
// before and behind them (EDGE of them at most), its first H entries.  Short rows are bound by their instructions (577 per
// four rows of 47 classes when all had U = 2, EDGE = 2 and H = 2), so each size has its own.
struct Entry { int64_t id; float t, z; };

template <typename T> __device__ __forceinline__ void load_entry(Entry &e, const Args &a, int row, int j) {
    e.id = j < a.K ? id_at(a, row, j) : -1;
    e.t = j < a.K ? teacher_at(a, row, j) : NEG_INF;
    if (e.id >= a.V) e.t = NAN;          // makes the row's sum NaN, and with it its loss and gradient
}
template <typename T> __device__ __forceinline__ void load_score(Entry &e, const Args &a, int row) {
    e.z = e.id >= 0 && e.id < a.V ? to_float(static_cast<const T *>(a.z)[(int64_t)row * a.ldz + e.id]) : 0.0f;
}

template <typename T> constexpr int edge_elements(int lanes, bool aligned) { return ((aligned ? 1 : 2) * (Piece<T>::E - 1) + lanes - 1) / lanes; }

template <typename T, int LANES, int U, int EDGE> struct Front {
    Batch<T, U> first;
    float edge[EDGE];
    __device__ __forceinline__ void load(const Span<T> &sp, int lane) {
        load_batch(first, sp.body(), lane, LANES, sp.pieces);
#pragma unroll
        for (int i = 0; i < EDGE; ++i) {
            const int k = lane + i * LANES;
            edge[i] = k < sp.head ? to_float(sp.p[k]) : k < sp.head + sp.tail ? to_float(sp.rest()[k - sp.head]) : NEG_INF;
        }
    }
    // running statistics of the span; the next pieces are on their way while these are added
    __device__ __forceinline__ void stats(const Span<T> &sp, int lane, float c, float &m, float &s) {
        const int pieces = sp.pieces;
        Batch<T, U> cur = first;
        for (int k = lane; k < pieces;) {
            Batch<T, U> next;
            k += U * LANES;
            if (LANES >= 32 || k < pieces) load_batch(next, sp.body(), k, LANES, pieces);
            add_pieces<T, U>(m, s, cur.u, c);
            cur = next;
        }
        add_values<EDGE>(m, s, edge, c);
    }
    // f exp((z - m) c) over the span; what the teacher's entries take off is put right behind it
    __device__ __forceinline__ void grad(const Span<T> &sp, T *out, bool vector, int lane, float c, float m, float f) {
        constexpr int E = Piece<T>::E;
        const int pieces = sp.pieces;
        T *body = out + sp.head, *rest = body + pieces * E;
        const uint64_t minus = pair2(-m, -m), cc = pair2(c, c), ff = pair2(f, f);
        Batch<T, U> cur = first;
        for (int k = lane; k < pieces; k += U * LANES) {
            Batch<T, U> next;
            if (LANES >= 32 || k + U * LANES < pieces) load_batch(next, sp.body(), k + U * LANES, LANES, pieces);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (k + i * LANES >= pieces) break;
                float v[E];
                Piece<T>::unpack(cur.u[i], v);
#pragma unroll
                for (int e = 0; e < E; e += 2) unpair2(mul2(exp2_pair(v[e], v[e + 1], minus, cc), ff), v[e], v[e + 1]);
                T *to = body + (k + i * LANES) * E;
                if (vector) {
                    *reinterpret_cast<uint4 *>(to) = Piece<T>::pack(v);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) to[e] = from_float<T>(v[e]);
                }
            }
            cur = next;
        }
#pragma unroll
        for (int i = 0; i < EDGE; ++i) {
            const int k = lane + i * LANES;
            const T v = from_float<T>(f * exp2_approx((edge[i] - m) * c));
            if (k < sp.head) out[k] = v;
            else if (k < sp.head + sp.tail) rest[k - sp.head] = v;
        }
    }
};

// The row's loss from its statistics, by L lanes that hold the same (m, s) and the row's first entries; writes the state,
// returns the loss in every lane.
template <typename T, int L, int H> __device__ __forceinline__ float row_loss(const Args &a, int row, int lane, bool active, float m, float s,
                                                                       const Entry (&held)[H], float &counted) {
    auto entry = [&](int i) {
        Entry e;
        load_entry<T>(e, a, row, lane + i * L);
        load_score<T>(e, a, row);
        return e;
    };
    const int per_lane = active ? (a.K + L - 1) / L : 0;          // (the same in all lanes of the group)
    float tm = NEG_INF;
    auto look = [&](const Entry &e) { if (e.id >= 0) tm = fmaxf(tm, e.t); };
#pragma unroll
    for (int i = 0; i < H; ++i) look(held[i]);
    for (int i = H; i < per_lane; ++i) look(entry(i));
    tm = group_max<L>(tm);
    const float safe = finite_or_zero(tm);
    float ts = 0.0f;
    auto weigh = [&](const Entry &e) { if (e.id >= 0) ts += exp2_approx((e.t - safe) * a.c); };
#pragma unroll
    for (int i = 0; i < H; ++i) weigh(held[i]);
    for (int i = H; i < per_lane; ++i) weigh(entry(i));
    ts = group_sum<L>(ts);
    const float log_s = log2f(s), log_ts = log2f(ts);
    float l = 0.0f;
    auto take = [&](const Entry &e) {
        if (e.id < 0) return;
        const float lp = (e.t - safe) * a.c - log_ts, p = exp2_approx(lp);
        if (p != 0.0f) l += p * (lp - ((e.z - m) * a.c - log_s));
    };
    if (ts != 0.0f) {
#pragma unroll
        for (int i = 0; i < H; ++i) take(held[i]);
        for (int i = H; i < per_lane; ++i) take(entry(i));
    }
    l = group_sum<L>(l) * (a.T * a.T * LN2);
    counted = ts != 0.0f ? 1.0f : 0.0f;          // no entry, or none of any weight: the sum is 0
    if (active && lane == 0) {
        a.state[row] = make_float4(m, s, safe, ts);
        if (a.reduction == RED_NONE) a.loss[row] = l;
    }
    return l;
}

// ---- short rows: L lanes a row, the losses of a block's rows summed ----
template <typename T, int L, int U, int EDGE, int H> __global__ void __launch_bounds__(THREADS) short_fwd_kernel(const Args a) {
    wait_for_previous();
    let_next_start();
    __shared__ float red[64];
    const int lane = threadIdx.x % L;
    constexpr int ROWS = THREADS / L;
    float sum = 0.0f, count = 0.0f;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.n; r0 += (int64_t)gridDim.x * ROWS) {
        const bool active = r0 + threadIdx.x / L < a.n;
        const int row = (int)r0 + threadIdx.x / L;
        float m = NEG_INF, s = 0.0f;
        Entry held[H];
#pragma unroll
        for (int i = 0; i < H; ++i) held[i] = {-1, NEG_INF, 0.0f};
        if (active) {
            const Span<T> sp(static_cast<const T *>(a.z) + (int64_t)row * a.ldz, a.V);
            Front<T, L, U, EDGE> front;
#pragma unroll
            for (int i = 0; i < H; ++i) load_entry<T>(held[i], a, row, lane + i * L);
            front.load(sp, lane);
#pragma unroll
            for (int i = 0; i < H; ++i) load_score<T>(held[i], a, row);
            front.stats(sp, lane, a.c, m, s);
        }
        const float top = group_max<L>(m);
        s = group_sum<L>(s * exp2_approx((m - finite_or_zero(top)) * a.c));
        float counted;
        const float l = row_loss<T, L, H>(a, row, lane, active, top, s, held, counted);
        if (lane == 0 && active) { sum += l; count += counted; }
    }
    if (a.reduction == RED_NONE) return;
    block_sum2(sum, count, red);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = make_float2(sum, count);
}

__device__ __forceinline__ float row_factor(const Args &a, int row, const float4 &st) {
    if (st.w == 0.0f) return 0.0f;
    const float g = a.reduction == RED_NONE ? a.grad[row] : loss_factor(a.grad, a.count, a.reduction);
    return g * a.T;
}

// A row's entries in shared memory, ids below 0 absent, each with its probability
__device__ __forceinline__ void stage_entry(const Args &a, const Entry &e, int j, const float4 &st, float inv, int *ids, float *p) {
    if (j >= a.K) return;
    ids[j] = e.id < 0 || e.id >= a.V ? -1 : (int)e.id;
    p[j] = e.id < 0 ? 0.0f : exp2_approx((e.t - st.z) * a.c) * inv;
}

// Class of an entry within [lo, hi): q minus the sum of all the row's entries of that class, so that an id that occurs several
// times gets the same value from each
template <typename T> __device__ __forceinline__ void fix_entry(const Args &a, const Entry &e, T *dz, const int *ids, const float *p, int lo, int hi,
                                                                float m, float inv_s, float f) {
    if (e.id < lo || e.id >= hi) return;          // (an absent one is below every lo)
    float taken = 0.0f;
    for (int i = 0; i < a.K; ++i) if (ids[i] == (int)e.id) taken += p[i];
    dz[e.id] = from_float<T>(f * (exp2_approx((e.z - m) * a.c) * inv_s - taken));
}

// The gradient of the part [lo, hi) of a row by LANES threads; `sync` joins them.
template <typename T, int LANES, int U, int EDGE, int H, typename Sync> __device__ __forceinline__ void row_grad(const Args &a, int row, int lo, int hi, int lane,
                                                                                                 bool active, int *ids, float *p, Sync sync) {
    const T *z = static_cast<const T *>(a.z) + (active ? (int64_t)row * a.ldz : 0);
    T *dz = static_cast<T *>(a.dz) + (active ? (int64_t)row * a.ldo : 0);
    float4 st = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
    Entry held[H];
#pragma unroll
    for (int i = 0; i < H; ++i) held[i] = {-1, NEG_INF, 0.0f};
    float f = 0.0f, inv_s = 0.0f;
    bool has = false;
    const int per_lane = (a.K + LANES - 1) / LANES;
    auto later = [&](int i) {
        Entry e;
        load_entry<T>(e, a, row, lane + i * LANES);
        load_score<T>(e, a, row);
        return e;
    };
    if (active) {
        const Span<T> sp(z + lo, hi - lo);
        Front<T, LANES, U, EDGE> front;
        st = a.state[row];
#pragma unroll
        for (int i = 0; i < H; ++i) load_entry<T>(held[i], a, row, lane + i * LANES);
        front.load(sp, lane);
#pragma unroll
        for (int i = 0; i < H; ++i) load_score<T>(held[i], a, row);
        if (st.w != 0.0f) {
            f = st.w != st.w ? NAN : row_factor(a, row, st);
            inv_s = 1.0f / st.y;
            has = st.w > 0.0f;
            const float inv = 1.0f / st.w;
#pragma unroll
            for (int i = 0; i < H; ++i) stage_entry(a, held[i], lane + i * LANES, st, inv, ids, p);
            for (int i = H; i < per_lane; ++i) stage_entry(a, later(i), lane + i * LANES, st, inv, ids, p);
            front.grad(sp, dz + lo, ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u) == 0, lane, a.c, st.x, f * inv_s);
        } else {
            for (int i = lo + lane; i < hi; i += LANES) dz[i] = from_float<T>(0.0f);
        }
    }
    sync();                                          // the stores and staged entries of all before the corrections
    if (has) {
#pragma unroll
        for (int i = 0; i < H; ++i) fix_entry<T>(a, held[i], dz, ids, p, lo, hi, st.x, inv_s, f);
        for (int i = H; i < per_lane; ++i) fix_entry<T>(a, later(i), dz, ids, p, lo, hi, st.x, inv_s, f);
    }
    sync();
}

template <typename T, int L, int U, int EDGE, int H> __global__ void __launch_bounds__(THREADS) short_bwd_kernel(const Args a) {
    wait_for_previous();
    let_next_start();
    constexpr int ROWS = THREADS / L;
    __shared__ int s_ids[ROWS][SHORT_KEPT];
    __shared__ float s_p[ROWS][SHORT_KEPT];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.n; r0 += (int64_t)gridDim.x * ROWS) {
        const bool active = r0 + group < a.n;
        const int row = (int)r0 + group;
        row_grad<T, L, U, EDGE, H>(a, row, 0, a.V, lane, active, s_ids[group], s_p[group], [] { __syncwarp(); });
    }
}

// ---- longer rows: a CTA per row, or per part of a row where there are few rows ----
// end of the part that starts at lo (lo + part may pass 31 bits)
__device__ __forceinline__ int part_end(const Args &a, int lo) { return a.V - lo > a.part ? lo + a.part : a.V; }

template <typename T> __global__ void __launch_bounds__(THREADS) long_fwd_kernel(const Args a) {
    wait_for_previous();
    let_next_start();
    __shared__ float red_m[THREADS / 32], red_s[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float sum = 0.0f, count = 0.0f;
    const int64_t items = (int64_t)a.n * a.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = (int)(item / a.splits);
        const int split = (int)(item - (int64_t)row * a.splits);
        const int lo = split * a.part, hi = part_end(a, lo);
        float m = NEG_INF, s = 0.0f;
        const T *z = static_cast<const T *>(a.z) + (int64_t)row * a.ldz;
        Entry held[LONG_HELD];
        const bool ends = warp == 0 && a.splits == 1;          // this warp takes the row's loss
        const Span<T> sp(z + lo, hi - lo);
        Front<T, THREADS, 4, 1> front;
        if (ends) {
#pragma unroll
            for (int i = 0; i < LONG_HELD; ++i) load_entry<T>(held[i], a, row, lane + i * 32);
        }
        front.load(sp, threadIdx.x);
        if (ends) {
#pragma unroll
            for (int i = 0; i < LONG_HELD; ++i) load_score<T>(held[i], a, row);
        }
        front.stats(sp, threadIdx.x, a.c, m, s);
        float top = group_max<32>(m);
        s = group_sum<32>(s * exp2_approx((m - finite_or_zero(top)) * a.c));
        if (lane == 0) { red_m[warp] = top; red_s[warp] = s; }
        __syncthreads();
        if (warp == 0) {
            m = lane < THREADS / 32 ? red_m[lane] : NEG_INF;
            s = lane < THREADS / 32 ? red_s[lane] : 0.0f;
            top = group_max<32>(m);
            s = group_sum<32>(s * exp2_approx((m - finite_or_zero(top)) * a.c));
            if (a.splits == 1) {
                float counted;
                sum += row_loss<T, 32, LONG_HELD>(a, row, lane, true, top, s, held, counted);
                count += counted;
            } else if (lane == 0) {
                a.stats[(int64_t)split * a.n + row] = make_float2(top, s);
            }
        }
        __syncthreads();
    }
    if (a.splits == 1 && a.reduction != RED_NONE && threadIdx.x == 0) a.partial[blockIdx.x] = make_float2(sum, count);
}

// joins the parts of the rows of long_fwd_kernel; a warp per row
template <typename T> __global__ void __launch_bounds__(THREADS) join_fwd_kernel(const Args a) {
    wait_for_previous();
    let_next_start();
    __shared__ float red[64];
    const int lane = threadIdx.x & 31;
    float sum = 0.0f, count = 0.0f;
    for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); r < a.n; r += (int64_t)gridDim.x * (THREADS / 32)) {
        const int row = (int)r;
        float m = NEG_INF, s = 0.0f;
        Entry held[LONG_HELD];
#pragma unroll
        for (int i = 0; i < LONG_HELD; ++i) { load_entry<T>(held[i], a, row, lane + i * 32); load_score<T>(held[i], a, row); }
        for (int i = lane; i < a.splits; i += 32) {
            const float2 p = a.stats[(int64_t)i * a.n + row];
            join_stats(m, s, p.x, p.y, a.c);
        }
        const float top = group_max<32>(m);
        s = group_sum<32>(s * exp2_approx((m - finite_or_zero(top)) * a.c));
        float counted;
        const float l = row_loss<T, 32, LONG_HELD>(a, row, lane, true, top, s, held, counted);
        if (lane == 0) { sum += l; count += counted; }
    }
    if (a.reduction == RED_NONE) return;
    block_sum2(sum, count, red);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = make_float2(sum, count);
}

template <typename T> __global__ void __launch_bounds__(THREADS) long_bwd_kernel(const Args a) {
    wait_for_previous();
    let_next_start();
    __shared__ int s_ids[MAX_KEPT];
    __shared__ float s_p[MAX_KEPT];
    const int64_t items = (int64_t)a.n * a.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = (int)(item / a.splits);
        const int lo = (int)(item - (int64_t)row * a.splits) * a.part;
        row_grad<T, THREADS, 4, 1, 1>(a, row, lo, part_end(a, lo), threadIdx.x, true, s_ids, s_p, [] { __syncthreads(); });
    }
}

static int64_t grid_limit() { return (int64_t)sm_count() * CTAS_PER_SM; }

// A warp (or less) per row, which has no barrier and no idle warps at a row's end, while there are rows enough to fill the SMs
// with warps; else a CTA per row or part of a row.  Warp against CTA, us forward and backward, bf16: 100,000 x 1,000 191 / 1,008;
// 1,000 x 2,000 10.7 / 16.7; 500 x 8,000 16.7 / 12.6, 2,000 x 8,000 23 / 27; 1,000 x 16,000 25.5 / 22, 5,000 x 16,000 96 / 106;
// 20,000 x 32,000 677 / 652.  fp32: 2,000 x 8,000 41 / 41, 20,000 x 8,000 323 / 364; 5,000 x 16,000 194 / 173.
static bool short_rows(int64_t n, int64_t V, int K, size_t es) {
    const int64_t bytes = V * (int64_t)es, full = (int64_t)sm_count() * 4;
    return K <= SHORT_KEPT && (V <= 1024 || (bytes <= SHORT_ROW_BYTES && n >= full && n >= bytes / 16));
}
// Parts of a long row: as many as give every SM work, none shorter than SPLIT_MIN classes; part lengths are whole pieces.
static void split_rows(int64_t n, int64_t V, int *splits, int *part) {
    int64_t s = ceil_div(grid_limit() / 2, n > 0 ? n : 1);
    const int64_t most = V / SPLIT_MIN;
    if (s > most) s = most;
    if (s < 1) s = 1;
    const int64_t p = ceil_div(ceil_div(V, s), (int64_t)64) * 64;
    *part = (int)(p < V ? p : V);
    *splits = (int)ceil_div(V, p);
}

struct Layout { size_t partial, stats, bytes; };
static Layout layout(int64_t n, int64_t V) {
    int splits, part;
    split_rows(n, V, &splits, &part);
    Layout l;
    l.partial = 0;
    l.stats = (size_t)grid_limit() * sizeof(float2);
    l.bytes = l.stats + (splits > 1 ? (size_t)splits * (size_t)n * sizeof(float2) : 0);
    return l;
}

template <typename T, int L, int U, int EDGE> static int launch_short(const Args &a, bool fwd, int64_t *grid, cudaStream_t st) {
    int64_t g = ceil_div((int64_t)a.n, (int64_t)(THREADS / L));
    if (g > grid_limit()) g = grid_limit();
    *grid = g;
    void (*kernel)(const Args) = a.K <= L ? (fwd ? short_fwd_kernel<T, L, U, EDGE, 1> : short_bwd_kernel<T, L, U, EDGE, 1>)
                                          : (fwd ? short_fwd_kernel<T, L, U, EDGE, 2> : short_bwd_kernel<T, L, U, EDGE, 2>);
    return launch_next(kernel, dim3((unsigned)g), THREADS, 0, st, 1, a);
}

// lanes of a short row: one or two 16-byte pieces each, four at a time for a warp
template <typename T> static int launch_short_rows(const Args &a, bool fwd, int64_t *grid, cudaStream_t st) {
    const int64_t pieces = ceil_div(a.V * (int64_t)sizeof(T), (int64_t)16);
    const bool aligned = aligned16(a.z) && a.ldz * (int64_t)sizeof(T) % 16 == 0;
    if (pieces <= 8) return aligned ? launch_short<T, 8, 1, edge_elements<T>(8, true)>(a, fwd, grid, st) : launch_short<T, 8, 1, edge_elements<T>(8, false)>(a, fwd, grid, st);
    if (pieces <= 16) return aligned ? launch_short<T, 8, 2, edge_elements<T>(8, true)>(a, fwd, grid, st) : launch_short<T, 8, 2, edge_elements<T>(8, false)>(a, fwd, grid, st);
    if (pieces <= 32) return launch_short<T, 16, 2, 1>(a, fwd, grid, st);
    return launch_short<T, 32, 4, 1>(a, fwd, grid, st);
}

template <typename T> static int launch(Args a, bool fwd, float *loss, float *count, cudaStream_t st) {
    int64_t grid = 0;
    if (short_rows(a.n, a.V, a.K, sizeof(T))) {
        if (int rc = launch_short_rows<T>(a, fwd, &grid, st)) return rc;
    } else {
        split_rows(a.n, a.V, &a.splits, &a.part);
        grid = (int64_t)a.n * a.splits < grid_limit() ? (int64_t)a.n * a.splits : grid_limit();
        if (int rc = launch_next(fwd ? long_fwd_kernel<T> : long_bwd_kernel<T>, dim3((unsigned)grid), THREADS, 0, st, 1, a)) return rc;
        if (fwd && a.splits > 1) {
            grid = ceil_div((int64_t)a.n, (int64_t)(THREADS / 32));
            if (grid > grid_limit()) grid = grid_limit();
            if (int rc = launch_next(join_fwd_kernel<T>, dim3((unsigned)grid), THREADS, 0, st, 1, a)) return rc;
        }
    }
    if (fwd && a.reduction != RED_NONE) {
        if (int rc = launch_next(loss_sum_kernel, dim3(1), 512, 0, st, 1, a.partial, (int)grid, a.reduction, loss, count)) return rc;
    }
    return GRWS_OK;
}

static int check(int64_t n, int64_t V, int64_t K, int64_t ldz, int64_t ldt, int64_t ldi, int dtype, int t_dtype, int id_bytes, float T, int reduction) {
    GRWS_REQUIRE(n >= 0 && V > 0 && K > 0, "bad size (rows = %lld, classes = %lld, kept = %lld)", (long long)n, (long long)V, (long long)K);
    GRWS_REQUIRE(V <= INT32_MAX && n <= INT32_MAX && ldz <= INT32_MAX && ldt <= INT32_MAX && ldi <= INT32_MAX, "rows, classes and strides must fit 31 bits");
    if (K > MAX_KEPT) return fail(GRWS_ERR_UNSUPPORTED, "at most %d teacher entries per row (kept = %lld)", MAX_KEPT, (long long)K);
    GRWS_REQUIRE(ldz >= V && ldt >= K && ldi >= K, "leading dimension smaller than the row");
    if (dtype < GRWS_F32 || dtype > GRWS_BF16) return fail(GRWS_ERR_UNSUPPORTED, "bad dtype %d", dtype);
    if (t_dtype < GRWS_F32 || t_dtype > GRWS_BF16) return fail(GRWS_ERR_UNSUPPORTED, "bad teacher dtype %d", t_dtype);
    GRWS_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are 4- or 8-byte integers");
    GRWS_REQUIRE(T >= 0.99e-6f && T <= 1.01e6f, "the temperature must lie between 1e-6 and 1e6");
    GRWS_REQUIRE(reduction >= RED_NONE && reduction <= RED_SUM, "bad reduction %d", reduction);
    return GRWS_OK;
}

}  // namespace distill
}  // namespace grws

using namespace grws;

extern "C" {

__attribute__((visibility("default")))
size_t grws_distill_scratch_bytes(int64_t rows, int64_t classes) {
    if (rows < 0 || classes <= 0) return 0;
    return distill::layout(rows, classes).bytes;
}

__attribute__((visibility("default")))
int grws_distill_fwd(const void *logits, int64_t ldz, int dtype, const void *teacher, int64_t ldt, int teacher_dtype, const void *ids,
                     int64_t ldi, int id_bytes, int64_t rows, int64_t classes, int64_t kept, float temperature, int reduction,
                     float *loss, float *state, float *count, void *scratch, size_t scratch_bytes, void *stream) {
    int rc = distill::check(rows, classes, kept, ldz, ldt, ldi, dtype, teacher_dtype, id_bytes, temperature, reduction);
    if (rc != GRWS_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GRWS_REQUIRE(reduction == cls::RED_NONE || (loss && count), "null pointer");
    if (rows == 0) {
        if (reduction == cls::RED_NONE) return GRWS_OK;
        cls::loss_sum_kernel<<<1, 32, 0, st>>>(nullptr, 0, reduction, loss, count);
        GRWS_CUDA_TRY(cudaGetLastError());
        return GRWS_OK;
    }
    GRWS_REQUIRE(logits && teacher && ids && loss && state && scratch, "null pointer");
    GRWS_REQUIRE(aligned16(state) && aligned16(scratch), "state and scratch must be 16-byte aligned");
    const distill::Layout l = distill::layout(rows, classes);
    if (scratch_bytes < l.bytes) return fail(GRWS_ERR_SCRATCH, "distillation scratch too small");
    distill::Args a = {};
    a.z = logits; a.ldz = (int)ldz; a.t = teacher; a.ldt = (int)ldt; a.t_dtype = teacher_dtype; a.ids = ids; a.ldi = (int)ldi; a.id_bytes = id_bytes;
    a.n = (int)rows; a.V = (int)classes; a.K = (int)kept; a.T = temperature; a.c = cls::LOG2E / temperature; a.reduction = reduction;
    a.loss = loss; a.state = reinterpret_cast<float4 *>(state); a.splits = 1; a.part = (int)classes;
    a.partial = reinterpret_cast<float2 *>(static_cast<char *>(scratch) + l.partial);
    a.stats = reinterpret_cast<float2 *>(static_cast<char *>(scratch) + l.stats);
    switch (dtype) {
        case GRWS_F32: return distill::launch<float>(a, true, loss, count, st);
        case GRWS_F16: return distill::launch<__half>(a, true, loss, count, st);
        default: return distill::launch<__nv_bfloat16>(a, true, loss, count, st);
    }
}

__attribute__((visibility("default")))
int grws_distill_bwd(const void *logits, int64_t ldz, int dtype, const void *teacher, int64_t ldt, int teacher_dtype, const void *ids,
                     int64_t ldi, int id_bytes, int64_t rows, int64_t classes, int64_t kept, float temperature, int reduction,
                     const float *grad_loss, const float *state, const float *count, void *dlogits, int64_t ldo, void *stream) {
    int rc = distill::check(rows, classes, kept, ldz, ldt, ldi, dtype, teacher_dtype, id_bytes, temperature, reduction);
    if (rc != GRWS_OK) return rc;
    GRWS_REQUIRE(ldo >= classes && ldo <= INT32_MAX, "leading dimension smaller than the row");
    if (rows == 0) return GRWS_OK;
    GRWS_REQUIRE(logits && teacher && ids && grad_loss && state && dlogits, "null pointer");
    GRWS_REQUIRE(reduction != cls::RED_MEAN || count, "null pointer");
    GRWS_REQUIRE(aligned16(state), "state must be 16-byte aligned");
    distill::Args a = {};
    a.z = logits; a.ldz = (int)ldz; a.t = teacher; a.ldt = (int)ldt; a.t_dtype = teacher_dtype; a.ids = ids; a.ldi = (int)ldi; a.id_bytes = id_bytes;
    a.n = (int)rows; a.V = (int)classes; a.K = (int)kept; a.T = temperature; a.c = cls::LOG2E / temperature; a.reduction = reduction;
    a.state = reinterpret_cast<float4 *>(const_cast<float *>(state)); a.splits = 1; a.part = (int)classes;
    a.grad = grad_loss; a.count = count; a.dz = dlogits; a.ldo = (int)ldo;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case GRWS_F32: return distill::launch<float>(a, false, nullptr, nullptr, st);
        case GRWS_F16: return distill::launch<__half>(a, false, nullptr, nullptr, st);
        default: return distill::launch<__nv_bfloat16>(a, false, nullptr, nullptr, st);
    }
}

}  // extern "C"
