// Group norm with an activation over node features X [rows, C] (channels last), forward and backward.
//
// A batch holds `samples` graphs end to end; the statistics of graph s and group g (D = C / groups channels) run
// over M = len(s) * D values:
//     mean = sum x / M,  r = 1 / sqrt(sum (x - mean)^2 / M + eps),  xh = (x - mean) r,  u = xh w + b,  y = act(u)
// and with d = dy act'(u), e = d w, S1 = sum e, S2 = sum e xh over the same M values:
//     dx = r (e - (S1 + xh S2) / M),   dw_c = sum d xh,   db_c = sum d   over all rows.
//
// A statistic needs all of its graph before the first output, so memory traffic bounds both directions.  Two forms:
//   one launch   a workgroup owns a graph (and, where there are few graphs, only some groups of it).  Up to kHeld rows
//                per thread stay in registers between the statistics and the outputs; longer graphs are read again
//                while they are in the workgroup's L2;
//   pieces       graphs too long for that are cut into pieces of rows: partial statistics per piece and CHANNEL,
//                one small launch that joins them per graph and group, and a second pass over the pieces, last
//                piece first, for the outputs (what was read last is still in the last-level cache).
// A thread keeps the same V channels for all of its rows, so weights, statistics and channel sums live in registers.
// V is 16 bytes' worth at any width: the last vector of a row begins where it still fits and overlaps the one
// before, whose channels it computes again and writes with the same bits.  Nothing is added with atomics: the same
// call gives the same bits.
//
// Measured (one MI355X, kernel times):
//   one graph of 232 965 nodes, 128 channels, fp32, SiLU, in pieces: forward 33 + 7 + 39 us, backward 44 + 7 + 55 us; the
//   passes move 3.6, 6.1, 5.4 and 6.5 TB/s against 5.1 of a 2 GiB copy (what the last-level cache holds comes on top)
//   2 000 graphs, 100 000 nodes, 256 channels, bf16, SiLU, in one launch: forward 38 to 41, backward 59 to 62 + 6 us; half of it is
//   arithmetic (28 and 53 vector instructions a value), the rest latency of a graph at a time
//   the same in fp32: forward 69 us; backward, whose held rows its longest graphs outgrow, in pieces: 43 + 41 + 6 + 59 us
//   512 nodes, 64 channels, fp32, ReLU: forward 6.6 us
//
// Statistics are means and centred sums of squares throughout -- batches of rows centred on their own mean, then
// joined by  M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb)  or centred on the joint mean -- so a mean far from zero
// costs no digits; pieces are joined in 64 bits, where plain sums and sums of squares do.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "dense_types.h"

namespace {

using namespace cbm_dense;

constexpr int kMaxThreads = 1024;
constexpr int kMaxLanes = 4096;            // channels times slots of a workgroup: 32 KiB of LDS for two floats each
constexpr int kHeld = 8;                   // rows per thread that stay in registers
constexpr int kBatch = 8;                  // rows a thread has in flight in the statistics passes
constexpr int kApplyBatch = 4;             // ... and where it reads two arrays or writes one

constexpr int most_threads(int V) { return V * kMaxThreads > kMaxLanes ? kMaxLanes / V : kMaxThreads; }

// Which rows: piece p of the launch is rows [row0, row0 + rows) of sample s.
struct Rows {
    const int4* pieces;                    // ragged batch: {sample, row0, rows, 0} per piece; NULL: equal lengths
    const int* piece_ptr;                  // ragged batch: first piece of every sample (samples + 1)
    int samples, len, per_sample, piece_rows;   // equal lengths: pieces of a sample, rows of a piece
};

struct Piece { int s, row0, rows; };

__device__ __forceinline__ Piece piece_of(const Rows& R, int p) {
    if (R.pieces) {
        const int4 t = R.pieces[p];
        return {t.x, t.y, t.z};
    }
    const int s = p / R.per_sample, i = p - s * R.per_sample;
    return {s, s * R.len + i * R.piece_rows, min(R.piece_rows, R.len - i * R.piece_rows)};
}

// Pieces [p0, p0 + n) of sample s, and the rows of its i-th.
struct Span { int p0, n; };
__device__ __forceinline__ Span pieces_of(const Rows& R, int s) {
    if (R.piece_ptr) return {R.piece_ptr[s], R.piece_ptr[s + 1] - R.piece_ptr[s]};
    return {s * R.per_sample, R.per_sample};
}
__device__ __forceinline__ int rows_of_piece(const Rows& R, const Span& P, int i) {
    return R.pieces ? R.pieces[P.p0 + i].z : min(R.piece_rows, R.len - i * R.piece_rows);
}

struct Shape {
    int C, D, groups, act;
    int width;                             // channels of a workgroup (the last one's may be fewer)
    int cols, slots, log_slots;            // vectors across `width`; rows at a time, a power of two
    unsigned col_magic, d_magic;           // t / cols = t col_magic >> 20 for t < 1024;  c / D = c d_magic >> 32 for c <= 65536 (D = 1: 0)
    int ng;                                // one launch: groups of a workgroup
    int log_seg, log_unit;                 // one launch: lanes that sum a group, of which lanes across its units
    int64_t ldx, ldy, ldg;
    float eps;
};

// Which columns: the thread's channels are c .. c + V - 1; threads are slot-major.  live = false for the threads that
// round the workgroup up to whole wavefronts.
struct Lane { int slot, col, c; bool live; };

template <int V>
__device__ __forceinline__ Lane lane_of(const Shape& S, int c0) {
    const int slot = threadIdx.x * S.col_magic >> 20, col = threadIdx.x - slot * S.cols, end = min(c0 + S.width, S.C);
    return {slot, col, min(c0 + col * V, end - V), slot < S.slots && c0 + col * V < end};
}

// exp and reciprocal of the hardware: the first is off by (2 + |u|) 2^-24 of its value (its argument's product with log2 e is
// rounded), the second by 2^-23, and a sigmoid below 2^-126 counts as 0.  Where u is far below zero and |u| counts, u s itself
// is small.  A division to half a unit in the last place costs ten more instructions, and a graph batch in bf16 is bound by
// them, not by its bytes.
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __expf(-u)); }

template <int ACT>
__device__ __forceinline__ float activate(float u) {
    if constexpr (ACT == CBM_ACT_RELU) return u < 0.f ? 0.f : u;      // NaN stays NaN
    if constexpr (ACT == CBM_ACT_SILU) return u * sigmoid(u);
    return u;
}

// act'(u) dy; the ReLU's derivative at zero is zero
template <int ACT>
__device__ __forceinline__ float activate_grad(float u, float dy) {
    if constexpr (ACT == CBM_ACT_RELU) return u > 0.f ? dy : (u != u ? u : 0.f);
    if constexpr (ACT == CBM_ACT_SILU) {
        const float s = sigmoid(u);
        return dy * (s * (1.f + u * (1.f - s)));
    }
    return dy;
}

// fn with the activation as a constant: the choice is made once per loop over rows, not once per value
template <typename Fn>
__device__ __forceinline__ void by_activation(int act, Fn fn) {
    if (act == CBM_ACT_SILU) fn(std::integral_constant<int, CBM_ACT_SILU>());
    else if (act == CBM_ACT_RELU) fn(std::integral_constant<int, CBM_ACT_RELU>());
    else fn(std::integral_constant<int, CBM_ACT_NONE>());
}

// One row's arithmetic at a time: rows interleaved for their exponentials' sake need registers that are not there.
__device__ __forceinline__ void row_done() { __builtin_amdgcn_sched_barrier(0); }

// Rows slot, slot + slots, ... < rows.
__device__ __forceinline__ int rows_of_slot(int rows, int slot, int log_slots) {
    return rows > slot ? (rows - slot + (1 << log_slots) - 1) >> log_slots : 0;
}

// Joins a batch of `have` <= N rows to the channel statistics of n rows.  any: rows that any thread of the workgroup has
// (the same for all of them, so rows beyond it cost nothing).
template <typename T, int V, int N>
__device__ __forceinline__ void join_batch(const Raw<T, V> (&raw)[N], int have, int any, float n, float (&mean)[V], float (&m2)[V]) {
    const float cnt = static_cast<float>(have), inv = 1.f / cnt, w = cnt / (n + cnt);
    float m[V], q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = q[i] = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (k >= any) break;
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] += k < have ? raw[k][i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] *= inv;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (k >= any) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = k < have ? raw[k][i] - m[i] : 0.f;
            q[i] = __builtin_fmaf(d, d, q[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float d = m[i] - mean[i];
        mean[i] += d * w;
        m2[i] += q[i] + d * d * (n * w);
    }
}

// Rows first, first + slots, ... of x, the first N of them that there are.
template <typename T, int V, int N>
__device__ __forceinline__ void load_batch(const T* __restrict__ x, int64_t ld, int rows, int first, int slots, Raw<T, V> (&raw)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (first + k * slots < rows) raw[k] = load_raw<T, V>(x + static_cast<int64_t>(first + k * slots) * ld);
}

// Mean and centred sum of squares per channel of the rows slot, slot + slots, ... < rows.
template <typename T, int V>
__device__ __forceinline__ void thread_stats(const T* __restrict__ x, int64_t ld, int rows, int slot, int log_slots,
                                             float (&mean)[V], float (&m2)[V]) {
    const int slots = 1 << log_slots;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    float n = 0.f;
    for (int r = slot; r < rows; r += kBatch * slots) {
        Raw<T, V> raw[kBatch];
        load_batch<T, V, kBatch>(x, ld, rows, r, slots, raw);
        const int have = min(kBatch, rows_of_slot(rows, r, log_slots));
        join_batch<T, V, kBatch>(raw, have, rows_of_slot(rows, r - slot, log_slots), n, mean, m2);
        n += static_cast<float>(have);
    }
}

// Reduces two values per channel over the slots in LDS, slot by slot in halves: afterwards slot 0's a[..], b[..] hold
// the result.  STATS: mean and m2 with their rows; else plain sums.
template <int V, bool STATS>
__device__ __forceinline__ void join_slots(float (&p)[V], float (&q)[V], float* a, float* b, const Shape& S, const Lane& L, int rows) {
    const int width = S.cols * V, at = L.slot * width + L.col * V, base = rows >> S.log_slots, rest = rows & (S.slots - 1);
    auto count = [&](int s) { return s < S.slots ? base + (s < rest ? 1 : 0) : 0; };
    if (L.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a[at + i] = p[i]; b[at + i] = q[i]; }
    }
    __syncthreads();
    int n = STATS && L.live ? count(L.slot) : 0;
    for (int half = S.slots >> 1; half > 0; half >>= 1) {
        if (L.live && L.slot < half) {
            int nb = 0;                                     // rows already joined into slot + half
            if constexpr (STATS)
                for (int s = L.slot + half; s < S.slots; s += 2 * half) nb += count(s);
            const float w = nb ? static_cast<float>(nb) / static_cast<float>(n + nb) : 0.f, nw = static_cast<float>(n) * w;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float pb = a[at + half * width + i], qb = b[at + half * width + i];
                if constexpr (STATS) {
                    const float d = pb - p[i];
                    p[i] += d * w;
                    q[i] += qb + d * d * nw;
                } else {
                    p[i] += pb;
                    q[i] += qb;
                }
                a[at + i] = p[i];
                b[at + i] = q[i];
            }
            n += nb;
        }
        __syncthreads();
    }
}

// Sum over the lanes of a segment of 2^log_seg <= 64 lanes, in every one of them.
__device__ __forceinline__ float segment_sum(float v, int log_seg) {
    for (int o = (1 << log_seg) >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// What the one-launch kernels share: the units of a group in LDS.  A unit is a thread's whole vector where vectors do
// not straddle groups (WHOLE), a channel otherwise; a[slot * across + unit].
template <int V, bool WHOLE>
struct Units {
    int across, per_group;
    float weight;                          // channels of a unit
    __device__ __forceinline__ explicit Units(const Shape& S)
        : across(WHOLE ? S.cols : S.width), per_group(WHOLE ? S.D / V : S.D), weight(WHOLE ? V : 1) {}
};

template <typename T, int V, int ACT>
__device__ __forceinline__ void write_rows(const T* __restrict__ x, T* __restrict__ y, int64_t ldx, int64_t ldy, int rows,
                                           int slot, int slots, const float (&mean)[V], const float (&scale)[V],
                                           const float (&shift)[V]) {
    for (int r = slot; r < rows; r += kApplyBatch * slots) {
        Raw<T, V> raw[kApplyBatch];
        load_batch<T, V, kApplyBatch>(x, ldx, rows, r, slots, raw);
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            if (r + k * slots >= rows) break;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = activate<ACT>(__builtin_fmaf(raw[k][i] - mean[i], scale[i], shift[i]));
            store_from_f32<T, V>(y + static_cast<int64_t>(r + k * slots) * ldy, v);
        }
    }
}

// Adds d and d xh of one row to the channel sums.
template <typename T, int V, int ACT>
__device__ __forceinline__ void add_grads(const Raw<T, V>& x, const Raw<T, V>& dy, const float (&mean)[V], const float (&rstd)[V],
                                          const float (&w)[V], const float (&b)[V], float (&p1)[V], float (&p2)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float xh = (x[i] - mean[i]) * rstd[i];
        const float d = activate_grad<ACT>(__builtin_fmaf(xh, w[i], b[i]), dy[i]);
        p1[i] += d;
        p2[i] += d * xh;
    }
}

// dx = r (d w - c1 - xh c2) with c1 = S1 / M, c2 = S2 / M
template <typename T, int V, int ACT>
__device__ __forceinline__ void write_grad(const Raw<T, V>& x, const Raw<T, V>& dy, T* __restrict__ dx, const float (&mean)[V],
                                           const float (&rstd)[V], const float (&w)[V], const float (&b)[V], const float (&c1)[V],
                                           const float (&c2)[V]) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float xh = (x[i] - mean[i]) * rstd[i];
        const float d = activate_grad<ACT>(__builtin_fmaf(xh, w[i], b[i]), dy[i]);
        v[i] = rstd[i] * (__builtin_fmaf(d, w[i], -c1[i]) - xh * c2[i]);
    }
    store_from_f32<T, V>(dx, v);
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void thread_grad_sums(const T* __restrict__ x, const T* __restrict__ dy, int64_t ldx, int64_t ldg,
                                                 int rows, int slot, int slots, const float (&mean)[V], const float (&rstd)[V],
                                                 const float (&w)[V], const float (&b)[V], float (&p1)[V], float (&p2)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) p1[i] = p2[i] = 0.f;
    for (int r = slot; r < rows; r += kApplyBatch * slots) {
        Raw<T, V> xr[kApplyBatch], gr[kApplyBatch];
        load_batch<T, V, kApplyBatch>(x, ldx, rows, r, slots, xr);
        load_batch<T, V, kApplyBatch>(dy, ldg, rows, r, slots, gr);
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            if (r + k * slots >= rows) break;
            add_grads<T, V, ACT>(xr[k], gr[k], mean, rstd, w, b, p1, p2);
            row_done();
        }
    }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void write_grad_rows(const T* __restrict__ x, const T* __restrict__ dy, T* __restrict__ dx, int64_t ldx,
                                                int64_t ldg, int64_t ldd, int rows, int slot, int slots, const float (&mean)[V],
                                                const float (&rstd)[V], const float (&w)[V], const float (&b)[V],
                                                const float (&c1)[V], const float (&c2)[V]) {
    for (int r = slot; r < rows; r += kApplyBatch * slots) {
        Raw<T, V> xr[kApplyBatch], gr[kApplyBatch];
        load_batch<T, V, kApplyBatch>(x, ldx, rows, r, slots, xr);
        load_batch<T, V, kApplyBatch>(dy, ldg, rows, r, slots, gr);
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            if (r + k * slots >= rows) break;
            write_grad<T, V, ACT>(xr[k], gr[k], dx + static_cast<int64_t>(r + k * slots) * ldd, mean, rstd, w, b, c1, c2);
            row_done();
        }
    }
}

template <int V>
__device__ __forceinline__ void channel_params(const float* __restrict__ p, float otherwise, int c, bool live, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (p && live) ? p[c + i] : otherwise;
}

__device__ __forceinline__ int group_of(int c, unsigned d_magic) { return d_magic ? __umulhi(c, d_magic) : c; }

// A per-group value for each of a thread's channels first .. first + V - 1.
template <int V, bool WHOLE>
__device__ __forceinline__ void group_values(const float* __restrict__ p, int first, unsigned d_magic, float (&out)[V]) {
    if constexpr (WHOLE) {
        const float v = p[group_of(first, d_magic)];
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = v;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = p[group_of(first + i, d_magic)];
    }
}

// ---------------------------------------------------------------------------------------------
// one launch: workgroup (sample, block of whole groups)
// ---------------------------------------------------------------------------------------------
template <typename T, int V, bool WHOLE, int ACT>
__global__ __launch_bounds__(most_threads(V)) __attribute__((amdgpu_waves_per_eu(4))) void norm_forward_one(const T* __restrict__ X, T* __restrict__ Y,
                                                                    const float* __restrict__ weight, const float* __restrict__ bias,
                                                                    const int* __restrict__ ptr, const int* __restrict__ order, int len,
                                                                    float* __restrict__ mean_out,
                                                                    float* __restrict__ rstd_out, Shape S) {
    extern __shared__ float lds[];
    const int s = order ? order[blockIdx.x] : blockIdx.x, g0 = blockIdx.y * S.ng, c0 = g0 * S.D;
    const int row0 = ptr ? ptr[s] : s * len, rows = ptr ? ptr[s + 1] - row0 : len;
    if (rows == 0) {                                        // the same for the whole workgroup
        for (int g = threadIdx.x; mean_out && g < S.ng; g += blockDim.x) {
            mean_out[static_cast<int64_t>(s) * S.groups + g0 + g] = 0.f;
            rstd_out[static_cast<int64_t>(s) * S.groups + g0 + g] = 1.f / sqrtf(S.eps);
        }
        return;
    }
    const Lane L = lane_of<V>(S, c0);
    const Units<V, WHOLE> U(S);
    float* a = lds;
    float* b = a + S.slots * U.across;
    float* gm = b + S.slots * U.across;                    // mean and 1/std of the workgroup's groups
    float* gr = gm + S.ng;
    const T* x = X + static_cast<int64_t>(row0) * S.ldx + L.c;
    const int chunk = kHeld * S.slots;
    Raw<T, V> raw[kHeld];
    float mean[V], m2[V], scale[V], shift[V];
    channel_params<V>(weight, 1.f, L.c, L.live, scale);
    channel_params<V>(bias, 0.f, L.c, L.live, shift);
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    const int mine = L.live ? rows_of_slot(rows, L.slot, S.log_slots) : 0;
    for (int k = 0, r = L.slot; k < mine; k += kHeld, r += chunk) {
        load_batch<T, V, kHeld>(x, S.ldx, rows, r, S.slots, raw);
        join_batch<T, V, kHeld>(raw, min(kHeld, mine - k), rows_of_slot(rows - k * S.slots, 0, S.log_slots), static_cast<float>(k), mean, m2);
    }
    if (L.live) {
        if constexpr (WHOLE) {
            float m = 0.f, q = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) m += mean[i];
            m *= 1.f / V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = mean[i] - m;
                q += m2[i] + d * d * static_cast<float>(mine);
            }
            a[L.slot * U.across + L.col] = m;
            b[L.slot * U.across + L.col] = q;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[L.slot * U.across + L.c - c0 + i] = mean[i];
                b[L.slot * U.across + L.c - c0 + i] = m2[i];
            }
        }
    }
    __syncthreads();
    {
        const int seg = threadIdx.x >> S.log_seg, segs = blockDim.x >> S.log_seg, sub = threadIdx.x & ((1 << S.log_seg) - 1);
        const int u0 = sub & ((1 << S.log_unit) - 1), s0 = sub >> S.log_unit, ds = 1 << (S.log_seg - S.log_unit), du = 1 << S.log_unit;
        const int base = rows >> S.log_slots, rest = rows & (S.slots - 1);
        const float count = static_cast<float>(rows) * static_cast<float>(S.D);
        for (int g = seg; g < S.ng; g += segs) {
            float sum = 0.f, sq = 0.f;
            for (int t = s0; t < S.slots; t += ds) {
                const float n = U.weight * static_cast<float>(base + (t < rest ? 1 : 0));
                for (int u = u0; u < U.per_group; u += du) sum += n * a[t * U.across + g * U.per_group + u];
            }
            const float m = segment_sum(sum, S.log_seg) / count;
            for (int t = s0; t < S.slots; t += ds) {
                const float n = U.weight * static_cast<float>(base + (t < rest ? 1 : 0));
                for (int u = u0; u < U.per_group; u += du) {
                    const float d = a[t * U.across + g * U.per_group + u] - m;
                    sq += b[t * U.across + g * U.per_group + u] + d * d * n;
                }
            }
            const float r = 1.f / sqrtf(segment_sum(sq, S.log_seg) / count + S.eps);
            if (sub == 0) {
                gm[g] = m;
                gr[g] = r;
                if (mean_out) {
                    mean_out[static_cast<int64_t>(s) * S.groups + g0 + g] = m;
                    rstd_out[static_cast<int64_t>(s) * S.groups + g0 + g] = r;
                }
            }
        }
    }
    __syncthreads();
    if (!mine) return;
    forget(raw);
    group_values<V, WHOLE>(gm, L.c - c0, S.d_magic, mean);
    group_values<V, WHOLE>(gr, L.c - c0, S.d_magic, m2);
#pragma unroll
    for (int i = 0; i < V; ++i) scale[i] *= m2[i];
    T* y = Y + static_cast<int64_t>(row0) * S.ldy + L.c;
    for (int r = L.slot; r < rows; r += chunk) {
        if (rows > chunk) load_batch<T, V, kHeld>(x, S.ldx, rows, r, S.slots, raw);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            if (r + k * S.slots >= rows) break;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = activate<ACT>(__builtin_fmaf(raw[k][i] - mean[i], scale[i], shift[i]));
            store_from_f32<T, V>(y + static_cast<int64_t>(r + k * S.slots) * S.ldy, v);
            row_done();
        }
    }
}

// rows per thread of x and of dy that stay in registers: 32 registers of 4 channels each
constexpr int held_grad(int element) { return element == 2 ? 8 : 4; }

// Workgroup (i, block of groups) takes the samples i, i + gridDim.x, ...; its sums for dw and db over all of them
// go to part[(2 i + which) C + c].
template <typename T, int V, bool WHOLE, int ACT>
__global__ __launch_bounds__(most_threads(V)) __attribute__((amdgpu_waves_per_eu(4))) void norm_backward_one(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ DX,
                                                                     const float* __restrict__ weight, const float* __restrict__ bias,
                                                                     const int* __restrict__ ptr, const int* __restrict__ order, int len, int samples,
                                                                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                     float* __restrict__ part, int64_t ldd, Shape S) {
    extern __shared__ float lds[];
    constexpr int HELD = held_grad(sizeof(T));
    const int g0 = blockIdx.y * S.ng, c0 = g0 * S.D;
    const Lane L = lane_of<V>(S, c0);
    const Units<V, WHOLE> U(S);
    const int across = S.cols * V > U.across ? S.cols * V : U.across;
    float* a = lds;
    float* b = a + S.slots * across;
    float* gs1 = b + S.slots * across;
    float* gs2 = gs1 + S.ng;
    const int seg = threadIdx.x >> S.log_seg, segs = blockDim.x >> S.log_seg, sub = threadIdx.x & ((1 << S.log_seg) - 1);
    const int u0 = sub & ((1 << S.log_unit) - 1), s0 = sub >> S.log_unit, ds = 1 << (S.log_seg - S.log_unit), du = 1 << S.log_unit;
    float w[V], bi[V], dw[V], db[V];
    channel_params<V>(weight, 1.f, L.c, L.live, w);
    channel_params<V>(bias, 0.f, L.c, L.live, bi);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
    for (int k = blockIdx.x; k < samples; k += gridDim.x) {
        const int s = order ? order[k] : k;
        int slot = L.slot;                                  // its row offsets are the same for all samples: not to be kept
        forget(slot);
        const int row0 = ptr ? ptr[s] : s * len, rows = ptr ? ptr[s + 1] - row0 : len;
        if (rows == 0) continue;                            // the same for the whole workgroup
        const int mine = L.live ? rows_of_slot(rows, slot, S.log_slots) : 0;
        const int chunk = HELD * S.slots;
        const T* x = X + static_cast<int64_t>(row0) * S.ldx + L.c;
        const T* dy = DY + static_cast<int64_t>(row0) * S.ldg + L.c;
        float mean[V], rstd[V];
        if (L.live) {
            group_values<V, WHOLE>(mean_in + static_cast<int64_t>(s) * S.groups, L.c, S.d_magic, mean);
            group_values<V, WHOLE>(rstd_in + static_cast<int64_t>(s) * S.groups, L.c, S.d_magic, rstd);
        }
        // sums of e = d w and e xh: over the thread's vector where that lies in one group, else per channel
        constexpr int E = WHOLE ? 1 : V;
        float s1[E], s2[E];
#pragma unroll
        for (int i = 0; i < E; ++i) s1[i] = s2[i] = 0.f;
        Raw<T, V> xr[HELD], gr[HELD];
        for (int k = 0, r = slot; k < mine; k += HELD, r += chunk) {
            load_batch<T, V, HELD>(x, S.ldx, rows, r, S.slots, xr);
            load_batch<T, V, HELD>(dy, S.ldg, rows, r, S.slots, gr);
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                if (k + j >= mine) break;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = (xr[j][i] - mean[i]) * rstd[i];
                    const float d = activate_grad<ACT>(__builtin_fmaf(xh, w[i], bi[i]), gr[j][i]), e = d * w[i];
                    db[i] += d;
                    dw[i] = __builtin_fmaf(d, xh, dw[i]);
                    s1[WHOLE ? 0 : i] += e;
                    s2[WHOLE ? 0 : i] = __builtin_fmaf(e, xh, s2[WHOLE ? 0 : i]);
                }
                row_done();
            }
        }
        if (!DX) continue;                                  // the same for the whole workgroup
        if (L.live) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int at = slot * U.across + (WHOLE ? L.col : L.c - c0 + i);
                a[at] = s1[i];
                b[at] = s2[i];
            }
        }
        __syncthreads();
        const float inv = 1.f / (static_cast<float>(rows) * static_cast<float>(S.D));
        for (int g = seg; g < S.ng; g += segs) {
            float e1 = 0.f, e2 = 0.f;
            for (int t = s0; t < S.slots; t += ds)
                for (int u = u0; u < U.per_group; u += du) {
                    e1 += a[t * U.across + g * U.per_group + u];
                    e2 += b[t * U.across + g * U.per_group + u];
                }
            e1 = segment_sum(e1, S.log_seg);
            e2 = segment_sum(e2, S.log_seg);
            if (sub == 0) { gs1[g] = e1 * inv; gs2[g] = e2 * inv; }
        }
        __syncthreads();                                    // a and b are free again; gs1, gs2 until the next but one
        // xh and d of the held rows would take more registers than the 128 that let 4 wavefronts share a SIMD
        forget(xr);
        forget(gr);
        if (mine) {
            float c1[V], c2[V];
            group_values<V, WHOLE>(gs1, L.c - c0, S.d_magic, c1);
            group_values<V, WHOLE>(gs2, L.c - c0, S.d_magic, c2);
            T* dx = DX + static_cast<int64_t>(row0) * ldd + L.c;
            for (int r = slot; r < rows; r += chunk) {
                if (rows > chunk) {
                    load_batch<T, V, HELD>(x, S.ldx, rows, r, S.slots, xr);
                    load_batch<T, V, HELD>(dy, S.ldg, rows, r, S.slots, gr);
                }
#pragma unroll
                for (int j = 0; j < HELD; ++j) {
                    if (r + j * S.slots >= rows) break;
                    write_grad<T, V, ACT>(xr[j], gr[j], dx + static_cast<int64_t>(r + j * S.slots) * ldd, mean, rstd, w, bi, c1, c2);
                    row_done();
                }
            }
        }
    }
    if (!part) return;
    __syncthreads();
    join_slots<V, false>(db, dw, a, b, S, L, 0);
    if (L.live && L.slot == 0) {
        float* o = part + static_cast<int64_t>(blockIdx.x) * 2 * S.C + L.c;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = db[i]; o[S.C + i] = dw[i]; }
    }
}

// ---------------------------------------------------------------------------------------------
// pieces: workgroup (piece, block of columns)
// ---------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_stats_pieces(const T* __restrict__ X, float* __restrict__ part, Rows R, Shape S) {
    extern __shared__ float lds[];
    const Piece P = piece_of(R, blockIdx.x);
    const Lane L = lane_of<V>(S, blockIdx.y * S.width);
    float mean[V], m2[V];
    thread_stats<T, V>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, S.ldx, L.live ? P.rows : 0, L.slot, S.log_slots, mean, m2);
    join_slots<V, true>(mean, m2, lds, lds + S.slots * S.cols * V, S, L, P.rows);
    if (L.live && L.slot == 0) {
        float* o = part + static_cast<int64_t>(blockIdx.x) * 2 * S.C + L.c;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = mean[i]; o[S.C + i] = m2[i]; }
    }
}

// Three sums over the workgroup, in thread 0.  lds: 3 kMaxThreads / kWave values.
__device__ __forceinline__ void block_sums(double (&v)[3], double* lds) {
    const int waves = blockDim.x / kWave;
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 3; ++i) v[i] += __shfl_xor(v[i], o);
    if (threadIdx.x % kWave == 0)
#pragma unroll
        for (int i = 0; i < 3; ++i) lds[3 * (threadIdx.x / kWave) + i] = v[i];
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < waves; ++w)
#pragma unroll
            for (int i = 0; i < 3; ++i) v[i] += lds[3 * w + i];
}

// fn(value, second value, rows of the piece, channel of the group) for every piece and channel of a group, the loads of
// kAhead pieces at a time ahead of their use (one after the other, 1024 pieces took 12 us, most of it waiting)
constexpr int kAhead = 8;
template <typename Fn>
__device__ __forceinline__ void for_partials(const float* __restrict__ part, const Rows& R, const Shape& S, int s, int g, Fn fn) {
    const Span P = pieces_of(R, s);
    const int lanes = min(1 << S.log_unit, static_cast<int>(blockDim.x)), c0 = threadIdx.x & (lanes - 1), dp = blockDim.x / lanes;
    for (int c = c0; c < S.D; c += lanes) {
        const float* at = part + static_cast<int64_t>(P.p0) * 2 * S.C + g * S.D + c;
        for (int i = threadIdx.x / lanes; i < P.n; i += kAhead * dp) {
            float v1[kAhead], v2[kAhead];
            int n[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int j = i + k * dp, in = min(j, P.n - 1);
                v1[k] = at[static_cast<int64_t>(in) * 2 * S.C];
                v2[k] = at[static_cast<int64_t>(in) * 2 * S.C + S.C];
                n[k] = rows_of_piece(R, P, in);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i + k * dp < P.n) fn(v1[k], v2[k], n[k], c);
        }
    }
}

// Joins the pieces' channel statistics: one workgroup per (sample, group).  In 64 bits a sum of squares loses nothing
// that fp32 statistics hold, so one pass does.
__global__ __launch_bounds__(kMaxThreads) void norm_join_stats(const float* __restrict__ part, float* __restrict__ mean_out,
                                                               float* __restrict__ rstd_out, Rows R, Shape S) {
    __shared__ double red[3 * kMaxThreads / kWave];
    const int s = blockIdx.x / S.groups, g = blockIdx.x - s * S.groups;
    double v[3] = {0.0, 0.0, 0.0};                          // values, their sum, sum of squares
    for_partials(part, R, S, s, g, [&](float v1, float v2, int rows, int) {
        const double n = rows, m = v1;
        v[0] += n;
        v[1] += n * m;
        v[2] += v2 + n * m * m;
    });
    block_sums(v, red);
    if (threadIdx.x == 0) {
        const double mean = v[0] > 0.0 ? v[1] / v[0] : 0.0, var = v[0] > 0.0 ? v[2] / v[0] - mean * mean : 0.0;
        mean_out[blockIdx.x] = static_cast<float>(mean);
        rstd_out[blockIdx.x] = static_cast<float>(1.0 / sqrt((var < 0.0 ? 0.0 : var) + static_cast<double>(S.eps)));
    }
}

template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_apply_pieces(const T* __restrict__ X, T* __restrict__ Y, const float* __restrict__ weight,
                                                                     const float* __restrict__ bias, const float* __restrict__ mean_in,
                                                                     const float* __restrict__ rstd_in, Rows R, Shape S) {
    const Piece P = piece_of(R, gridDim.x - 1 - blockIdx.x);
    const Lane L = lane_of<V>(S, blockIdx.y * S.width);
    if (!L.live) return;
    float mean[V], rstd[V], scale[V], shift[V];
    channel_params<V>(weight, 1.f, L.c, true, scale);
    channel_params<V>(bias, 0.f, L.c, true, shift);
    group_values<V, false>(mean_in + static_cast<int64_t>(P.s) * S.groups, L.c, S.d_magic, mean);
    group_values<V, false>(rstd_in + static_cast<int64_t>(P.s) * S.groups, L.c, S.d_magic, rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) scale[i] *= rstd[i];
    by_activation(S.act, [&](auto act) {
        write_rows<T, V, decltype(act)::value>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, Y + static_cast<int64_t>(P.row0) * S.ldy + L.c,
                                               S.ldx, S.ldy, P.rows, L.slot, S.slots, mean, scale, shift);
    });
}

template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_grad_pieces(const T* __restrict__ X, const T* __restrict__ DY,
                                                                    const float* __restrict__ weight, const float* __restrict__ bias,
                                                                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                    float* __restrict__ part, Rows R, Shape S) {
    extern __shared__ float lds[];
    const Piece P = piece_of(R, blockIdx.x);
    const Lane L = lane_of<V>(S, blockIdx.y * S.width);
    float mean[V], rstd[V], w[V], b[V], p1[V], p2[V];
    channel_params<V>(weight, 1.f, L.c, L.live, w);
    channel_params<V>(bias, 0.f, L.c, L.live, b);
    if (L.live) {
        group_values<V, false>(mean_in + static_cast<int64_t>(P.s) * S.groups, L.c, S.d_magic, mean);
        group_values<V, false>(rstd_in + static_cast<int64_t>(P.s) * S.groups, L.c, S.d_magic, rstd);
    }
    by_activation(S.act, [&](auto act) {
        thread_grad_sums<T, V, decltype(act)::value>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c,
                                                     DY + static_cast<int64_t>(P.row0) * S.ldg + L.c, S.ldx, S.ldg, L.live ? P.rows : 0,
                                                     L.slot, S.slots, mean, rstd, w, b, p1, p2);
    });
    join_slots<V, false>(p1, p2, lds, lds + S.slots * S.cols * V, S, L, 0);
    if (L.live && L.slot == 0) {
        float* o = part + static_cast<int64_t>(blockIdx.x) * 2 * S.C + L.c;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = p1[i]; o[S.C + i] = p2[i]; }
    }
}

constexpr int kSumChannels = 8;            // channels of a workgroup that sums dw and db over the parts

// Workgroups [0, pairs): S1 / M and S2 / M of a (sample, group), any number of threads.  The rest: dw and db of
// kSumChannels channels each, the partial sums of all `parts` rows of part, kMaxThreads threads.
__global__ __launch_bounds__(kMaxThreads) void norm_join_grads(const float* __restrict__ part, const float* __restrict__ weight,
                                                               float* __restrict__ c1_out, float* __restrict__ c2_out,
                                                               float* __restrict__ dw, float* __restrict__ db, int pairs, int parts,
                                                               Rows R, Shape S) {
    __shared__ float red[2][kMaxThreads];
    __shared__ double redd[3 * kMaxThreads / kWave];
    if (static_cast<int>(blockIdx.x) < pairs) {
        const int s = blockIdx.x / S.groups, g = blockIdx.x - s * S.groups;
        double v[3] = {0.0, 0.0, 0.0};
        for_partials(part, R, S, s, g, [&](float v1, float v2, int rows, int c) {
            const double w = weight ? weight[g * S.D + c] : 1.f;
            v[0] += rows;
            v[1] += w * v1;
            v[2] += w * v2;
        });
        block_sums(v, redd);
        if (threadIdx.x == 0) {
            c1_out[blockIdx.x] = v[0] > 0.0 ? static_cast<float>(v[1] / v[0]) : 0.f;
            c2_out[blockIdx.x] = v[0] > 0.0 ? static_cast<float>(v[2] / v[0]) : 0.f;
        }
        return;
    }
    const int c = (blockIdx.x - pairs) * kSumChannels + threadIdx.x % kSumChannels, k = threadIdx.x / kSumChannels;
    float v1 = 0.f, v2 = 0.f;
    if (c < S.C)
#pragma unroll 8
        for (int p = k; p < parts; p += kMaxThreads / kSumChannels) {
            v1 += part[static_cast<int64_t>(p) * 2 * S.C + c];
            v2 += part[static_cast<int64_t>(p) * 2 * S.C + S.C + c];
        }
    red[0][threadIdx.x] = v1;
    red[1][threadIdx.x] = v2;
    __syncthreads();
    for (int half = kMaxThreads / kSumChannels / 2; half > 0; half >>= 1) {
        if (k < half) {
            red[0][threadIdx.x] += red[0][threadIdx.x + kSumChannels * half];
            red[1][threadIdx.x] += red[1][threadIdx.x + kSumChannels * half];
        }
        __syncthreads();
    }
    if (k == 0 && c < S.C) {
        if (db) db[c] = red[0][threadIdx.x];
        if (dw) dw[c] = red[1][threadIdx.x];
    }
}

template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_grad_apply_pieces(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ DX,
                                                                          const float* __restrict__ weight, const float* __restrict__ bias,
                                                                          const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                          const float* __restrict__ c1_in, const float* __restrict__ c2_in,
                                                                          int64_t ldd, Rows R, Shape S) {
    const Piece P = piece_of(R, gridDim.x - 1 - blockIdx.x);
    const Lane L = lane_of<V>(S, blockIdx.y * S.width);
    if (!L.live) return;
    float mean[V], rstd[V], w[V], b[V], c1[V], c2[V];
    channel_params<V>(weight, 1.f, L.c, true, w);
    channel_params<V>(bias, 0.f, L.c, true, b);
    const int64_t at = static_cast<int64_t>(P.s) * S.groups;
    group_values<V, false>(mean_in + at, L.c, S.d_magic, mean);
    group_values<V, false>(rstd_in + at, L.c, S.d_magic, rstd);
    group_values<V, false>(c1_in + at, L.c, S.d_magic, c1);
    group_values<V, false>(c2_in + at, L.c, S.d_magic, c2);
    by_activation(S.act, [&](auto act) {
        write_grad_rows<T, V, decltype(act)::value>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c,
                                                    DY + static_cast<int64_t>(P.row0) * S.ldg + L.c,
                                                    DX + static_cast<int64_t>(P.row0) * ldd + L.c, S.ldx, S.ldg, ldd, P.rows, L.slot, S.slots,
                                                    mean, rstd, w, b, c1, c2);
    });
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int kBackwardGroups = 1024;      // most workgroups that walk the samples of a one-launch backward
constexpr int kFewGraphs = 64;             // fewer graphs than this leave most CUs idle unless their groups are split
// One launch or pieces?  A workgroup that cannot hold its graph walks it twice, a chunk of held rows in 2 to 3 us, while
// pieces cost two launches more and are spread over all CUs.  37 graphs of up to 2 500 nodes, 602 channels, fp16 (5
// chunks): 66 + 83 us in one launch each way, 33 + 41 us in pieces.  2 000 graphs of up to 400 nodes (50 on average), 256
// channels, bf16 (up to 6 chunks, longest graphs first): 38 + 60 us in one launch, 44 + 66 us and the joins in pieces.
constexpr int kPieceThreads = 512;         // 2 workgroups per CU (the caller cuts 512 pieces): 256 and 1024 within 2 %
constexpr int kChunksFew = 3, kChunksMany = 8;

struct Plan {
    bool one, whole;
    int V, threads, blocks_y;
    Shape S;
};

// Channels of a thread: 16 bytes' worth; the one-launch backward keeps too much per channel for 8 of them.
int vector_of(int dtype, int width, bool one_backward) {
    const int v = one_backward ? 4 : 16 / element_bytes(dtype);
    return v > width ? 1 : v;
}

int log2_up(int v) {
    int l = 0;
    while ((1 << l) < v) ++l;
    return l;
}

int log2_down(int v) {
    int l = 0;
    while ((2 << l) <= v) ++l;
    return l;
}

Plan plan_of(const cbm_norm_batch* B, int C, int groups, int dtype, bool backward) {
    Plan P{};
    Shape& S = P.S;
    const int D = C / groups, e = element_bytes(dtype);
    S.C = C;
    S.D = D;
    S.groups = groups;
    auto cols_of = [](int width, int V) { return (width + V - 1) / V; };
    auto fits = [&](int width) {
        const int V = vector_of(dtype, width, backward);
        return cols_of(width, V) <= most_threads(V);
    };
    // one launch: all groups of a graph in a workgroup; fewer where there are few graphs (at least 64 bytes of a row)
    // or where a row is too wide for one
    int ng = fits(C) ? groups : 0;
    if (ng == 0 || B->samples < kFewGraphs)
        for (int g = 1; g <= groups; ++g)
            if (groups % g == 0 && g * D * e >= 64 && fits(g * D)) {
                ng = g;
                break;
            }
    const bool few = B->samples < kFewGraphs;
    auto slots = [&](int64_t want) { return log2_down(static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, B->max_len)))); };
    if (ng > 0 && ng <= 4096) {
        S.ng = ng;
        S.width = ng * D;
        P.V = vector_of(dtype, S.width, backward);
        S.cols = cols_of(S.width, P.V);
        P.blocks_y = groups / ng;
        P.whole = D % P.V == 0;
        // as many rows at a time as hold the longest of few graphs in the largest workgroup, or four average ones of many
        // in 512 threads (2 000 graphs as above, forward: 64 us with 128 threads, 42 with 256, 38 with 512)
        const int held = backward ? held_grad(e) : kHeld;
        const int64_t rows = few ? B->max_len : 4LL * B->rows / B->samples;
        S.log_slots = slots(std::min<int64_t>((rows + held - 1) / held, (few ? most_threads(P.V) : 512) / S.cols));
        P.one = B->max_len <= (static_cast<int64_t>(few ? kChunksFew : kChunksMany) * held << S.log_slots);
    }
    if (!P.one) {
        P.V = vector_of(dtype, C, false);
        const int total = cols_of(C, P.V), most = most_threads(P.V);
        P.blocks_y = (total + most - 1) / most;
        S.cols = (total + P.blocks_y - 1) / P.blocks_y;
        P.blocks_y = (total + S.cols - 1) / S.cols;
        S.width = S.cols * P.V;
        S.log_slots = slots(kPieceThreads / S.cols);
    }
    S.slots = 1 << S.log_slots;
    S.col_magic = ((1u << 20) + S.cols - 1) / S.cols;
    S.d_magic = D == 1 ? 0 : static_cast<unsigned>(((1ull << 32) + D - 1) / D);
    P.threads = (S.cols * S.slots + kWave - 1) / kWave * kWave;
    // lanes that sum a group: an equal share of the workgroup, a power of two of at most a wavefront
    const int units = P.one ? (P.whole ? D / P.V : D) : D;
    S.log_unit = log2_up(units);
    if (P.one) {
        S.log_seg = std::min(6, log2_up(std::max(1, P.threads / S.ng)));
        if ((P.threads >> S.log_seg) < 1) S.log_seg = 0;
        S.log_unit = std::min(S.log_unit, S.log_seg);
    }
    return P;
}

static_assert(sizeof(cbm_norm_batch) == 56, "the layout that bindings mirror");

Rows rows_of(const cbm_norm_batch* B) {
    Rows R{};
    R.pieces = reinterpret_cast<const int4*>(B->pieces);
    R.piece_ptr = B->piece_ptr;
    R.samples = B->samples;
    R.len = B->max_len;
    R.piece_rows = B->piece_rows;
    R.per_sample = B->piece_rows > 0 ? (B->max_len + B->piece_rows - 1) / B->piece_rows : 0;
    return R;
}

int pieces_total(const cbm_norm_batch* B, const Rows& R) { return B->pieces ? B->n_pieces : B->samples * R.per_sample; }

int check_batch(const cbm_norm_batch* B, int C, int groups, int dtype, int act) {
    if (!B) return CBM_ERR_NULL;
    if (dtype < CBM_DTYPE_F32 || dtype > CBM_DTYPE_F16 || act < CBM_ACT_NONE || act > CBM_ACT_SILU) return CBM_ERR_SHAPE;
    if (C < 1 || C > (1 << 16) || groups < 1 || C % groups) return CBM_ERR_SHAPE;
    if (B->samples < 0 || B->rows < 0 || B->max_len < 0 || B->max_len > B->rows) return CBM_ERR_SHAPE;
    if (B->samples > CBM_NORM_MAX_GRAPHS || static_cast<int64_t>(B->samples) * groups > CBM_NORM_MAX_PAIRS) return CBM_ERR_SHAPE;
    if (!B->ptr && static_cast<int64_t>(B->samples) * B->max_len != B->rows) return CBM_ERR_SHAPE;
    if (B->ptr && B->rows > 0 && (!B->pieces || !B->piece_ptr || B->n_pieces < 1)) return CBM_ERR_NULL;
    if (B->rows > 0 && B->piece_rows < 1) return CBM_ERR_SHAPE;
    return CBM_OK;
}

// Threads that join the pieces of a (sample, group), by its number of partial results; a grid holds fewer than 2^32 threads
// along one dimension (the limits on graphs and pairs keep the others below that).
int join_threads(int pieces, int D, int samples, int groups) {
    const int64_t items = static_cast<int64_t>(pieces) * D / samples;
    if (static_cast<int64_t>(samples) * groups > (1 << 21)) return kWave;
    return items >= 2048 ? kMaxThreads : items >= 256 ? 256 : kWave;
}

// Two floats per slot and channel, and two per group.
size_t lds_of(const Plan& P) {
    const int across = std::max(P.S.cols * P.V, P.S.width);
    return sizeof(float) * (2u * P.S.slots * across + 2u * (P.one ? P.S.ng : 0));
}

#define CBM_NORM_BY_VECTOR(T, VMAX, CALL)                 \
    if (P.V == 1) { constexpr int V = 1; CALL(T, V); }    \
    else { constexpr int V = VMAX; CALL(T, V); }
#define CBM_NORM_BY_TYPE(VHALF, CALL)                                             \
    if (dtype == CBM_DTYPE_F32) { CBM_NORM_BY_VECTOR(float, 4, CALL) }            \
    else if (dtype == CBM_DTYPE_BF16) { CBM_NORM_BY_VECTOR(__bf16, VHALF, CALL) } \
    else { CBM_NORM_BY_VECTOR(_Float16, VHALF, CALL) }
#define CBM_NORM_ONE_ACT(KERNEL, T, V, W, ...)                                                                \
    if (act == CBM_ACT_SILU) hipLaunchKernelGGL((KERNEL<T, V, W, CBM_ACT_SILU>), __VA_ARGS__);                \
    else if (act == CBM_ACT_RELU) hipLaunchKernelGGL((KERNEL<T, V, W, CBM_ACT_RELU>), __VA_ARGS__);           \
    else hipLaunchKernelGGL((KERNEL<T, V, W, CBM_ACT_NONE>), __VA_ARGS__)
#define CBM_NORM_ONE(KERNEL, T, V, ...)                                                                       \
    if (P.whole) { CBM_NORM_ONE_ACT(KERNEL, T, V, true, __VA_ARGS__); }                                       \
    else { CBM_NORM_ONE_ACT(KERNEL, T, V, (V == 1), __VA_ARGS__); }

}  // namespace

extern "C" {

int64_t cbm_group_norm_workspace_floats(const cbm_norm_batch* B, int32_t C, int32_t groups, int32_t dtype, int32_t backward) {
    if (check_batch(B, C, groups, dtype, CBM_ACT_NONE) != CBM_OK || B->rows == 0) return 0;
    const Plan P = plan_of(B, C, groups, dtype, backward != 0);
    const Rows R = rows_of(B);
    const int64_t pairs = static_cast<int64_t>(B->samples) * groups;
    if (P.one) return backward ? 2LL * C * std::min<int64_t>(B->samples, kBackwardGroups) : 0;
    return 2LL * C * pieces_total(B, R) + 2 * pairs;
}

int cbm_group_norm_forward(const cbm_norm_batch* B, const void* X, void* Y, const float* weight, const float* bias, float* mean,
                           float* rstd, float* workspace, int32_t C, int32_t groups, int64_t ldx, int64_t ldy, float eps, int32_t act,
                           int32_t dtype, void* stream) {
    if (int rc = check_batch(B, C, groups, dtype, act)) return rc;
    if ((mean == nullptr) != (rstd == nullptr)) return CBM_ERR_NULL;
    if (B->rows == 0) return CBM_OK;
    if (!X || !Y) return CBM_ERR_NULL;
    if (ldx < C || ldy < C || !(eps >= 0.f)) return CBM_ERR_SHAPE;
    // Both directions read their inputs again after others have begun to write, and two threads share the channels where a
    // row's last vector overlaps the one before.
    if (overlap(X, ldx, Y, ldy, B->rows, C, element_bytes(dtype))) return CBM_ERR_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    Plan P = plan_of(B, C, groups, dtype, false);
    Shape& S = P.S;
    S.act = act;
    S.ldx = ldx;
    S.ldy = ldy;
    S.eps = eps;
    const Rows R = rows_of(B);
    if (P.one) {
#define ONE(T, V)                                                                                                                    \
    CBM_NORM_ONE(norm_forward_one, T, V, dim3(B->samples, P.blocks_y), dim3(P.threads), lds_of(P), st, static_cast<const T*>(X),   \
                   static_cast<T*>(Y), weight, bias, B->ptr, B->order, B->max_len, mean, rstd, S)
        CBM_NORM_BY_TYPE(8, ONE)
#undef ONE
        return check_launch();
    }
    if (!workspace) return CBM_ERR_NULL;
    const int np = pieces_total(B, R);
    const int64_t pairs = static_cast<int64_t>(B->samples) * groups;
    float* part = workspace;
    float* m = mean ? mean : workspace + 2LL * C * np;
    float* r = rstd ? rstd : m + pairs;
#define STATS(T, V)                                                                                                                \
    hipLaunchKernelGGL((norm_stats_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), lds_of(P), st, static_cast<const T*>(X), \
                       part, R, S)
#define APPLY(T, V)                                                                                                          \
    hipLaunchKernelGGL((norm_apply_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), 0, st, static_cast<const T*>(X),    \
                       static_cast<T*>(Y), weight, bias, m, r, R, S)
    CBM_NORM_BY_TYPE(8, STATS)
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(norm_join_stats, dim3(static_cast<unsigned>(pairs)), dim3(join_threads(np, S.D, B->samples, groups)), 0, st,
                       part, m, r, R, S);
    if (int rc = check_launch()) return rc;
    CBM_NORM_BY_TYPE(8, APPLY)
#undef STATS
#undef APPLY
    return check_launch();
}

int cbm_group_norm_backward(const cbm_norm_batch* B, const void* X, const void* DY, void* DX, const float* weight, const float* bias,
                            const float* mean, const float* rstd, float* dweight, float* dbias, float* workspace, int32_t C,
                            int32_t groups, int64_t ldx, int64_t ldg, int64_t ldd, int32_t act, int32_t dtype, void* stream) {
    if (int rc = check_batch(B, C, groups, dtype, act)) return rc;
    if (B->rows > 0 && (!X || !DY || !mean || !rstd)) return CBM_ERR_NULL;
    if (ldx < C || ldg < C || (DX && ldd < C)) return CBM_ERR_SHAPE;
    if (overlap(X, ldx, DX, ldd, B->rows, C, element_bytes(dtype)) || overlap(DY, ldg, DX, ldd, B->rows, C, element_bytes(dtype)))
        return CBM_ERR_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool params = dweight || dbias;
    if (!params && (!DX || B->rows == 0)) return CBM_OK;
    if (B->rows > 0 && !workspace) return CBM_ERR_NULL;
    const unsigned channel_blocks = static_cast<unsigned>((C + kSumChannels - 1) / kSumChannels);
    Plan P = plan_of(B, C, groups, dtype, true);
    Shape& S = P.S;
    S.act = act;
    S.ldx = ldx;
    S.ldg = ldg;
    const Rows R = rows_of(B);
    if (B->rows == 0) {                                    // no rows: the parameters' gradients are zero
        hipLaunchKernelGGL(norm_join_grads, dim3(channel_blocks), dim3(kMaxThreads), 0, st, nullptr, weight, nullptr, nullptr, dweight,
                           dbias, 0, 0, R, S);
        return check_launch();
    }
    if (P.one) {
        const int walkers = std::min(B->samples, kBackwardGroups);
#define ONE(T, V)                                                                                                                    \
    CBM_NORM_ONE(norm_backward_one, T, V, dim3(walkers, P.blocks_y), dim3(P.threads), lds_of(P), st, static_cast<const T*>(X),     \
                   static_cast<const T*>(DY), static_cast<T*>(DX), weight, bias, B->ptr, B->order, B->max_len, B->samples, mean, rstd,         \
                   params ? workspace : nullptr, ldd, S)
        CBM_NORM_BY_TYPE(4, ONE)
#undef ONE
        if (int rc = check_launch()) return rc;
        if (!params) return CBM_OK;
        hipLaunchKernelGGL(norm_join_grads, dim3(channel_blocks), dim3(kMaxThreads), 0, st, workspace, weight, nullptr, nullptr, dweight,
                           dbias, 0, walkers, R, S);
        return check_launch();
    }
    const int np = pieces_total(B, R);
    const int pairs = B->samples * groups;
    float* part = workspace;
    float* c1 = workspace + 2LL * C * np;
    float* c2 = c1 + pairs;
#define SUMS(T, V)                                                                                                                 \
    hipLaunchKernelGGL((norm_grad_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), lds_of(P), st, static_cast<const T*>(X),  \
                       static_cast<const T*>(DY), weight, bias, mean, rstd, part, R, S)
#define APPLY(T, V)                                                                                                                \
    hipLaunchKernelGGL((norm_grad_apply_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), 0, st, static_cast<const T*>(X),    \
                       static_cast<const T*>(DY), static_cast<T*>(DX), weight, bias, mean, rstd, c1, c2, ldd, R, S)
    CBM_NORM_BY_TYPE(8, SUMS)
    if (int rc = check_launch()) return rc;
    // both joins in one launch, unless the pairs are many and small
    const int threads = join_threads(np, S.D, B->samples, groups);
    const bool apart = params && threads < kMaxThreads;
    hipLaunchKernelGGL(norm_join_grads, dim3(pairs + (params && !apart ? channel_blocks : 0)), dim3(threads), 0, st, part, weight, c1, c2,
                       dweight, dbias, pairs, np, R, S);
    if (int rc = check_launch()) return rc;
    if (apart) {
        hipLaunchKernelGGL(norm_join_grads, dim3(channel_blocks), dim3(kMaxThreads), 0, st, part, weight, nullptr, nullptr, dweight, dbias,
                           0, np, R, S);
        if (int rc = check_launch()) return rc;
    }
    if (!DX) return CBM_OK;
    CBM_NORM_BY_TYPE(8, APPLY)
#undef SUMS
#undef APPLY
    return check_launch();
}

}  // extern "C"
