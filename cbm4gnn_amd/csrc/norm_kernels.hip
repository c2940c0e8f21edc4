// Group norm with an activation over node features X [rows, C] (channels last), forward and backward.
//
// A batch holds `samples` graphs end to end; the statistics of graph s and group g (D = C / groups channels) run
// over M = len(s) * D values:
//     mean = sum x / M,  r = 1 / sqrt(sum (x - mean)^2 / M + eps),  xh = (x - mean) r,  u = xh w + b,  y = act(u)
// and with d = dy act'(u), e = d w, S1 = sum e, S2 = sum e xh over the same M values:
//     dx = r (e - (S1 + xh S2) / M),   dw_c = sum d xh,   db_c = sum d   over all rows.
//
// Both directions read everything twice (a statistic needs all of its graph before the first output), so memory
// traffic bounds them; a graph whose share of a workgroup stays in the cache is read from memory once.  Two forms:
//   one launch   a workgroup owns a graph (and, where there are few graphs, only some groups of it): statistics,
//                then outputs, from the same rows while they are in its L2;
//   pieces       graphs too long for that are cut into pieces of rows: partial statistics per piece and CHANNEL
//                (so that a group may start anywhere in a vector), one small launch that joins them per graph and
//                group, and a second pass over the pieces for the outputs.
// A thread keeps the same V channels (one 16-byte vector where rows divide into them) for all of its rows, so
// weights, statistics and channel sums live in registers.  Nothing is added with atomics: the same call gives the
// same bits.
//
// Statistics are means and centred sums of squares throughout -- batches of rows centred on their own mean, then
// joined pairwise by  M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb)  -- so a mean far from zero costs no digits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense_types.h"

namespace {

using namespace cbm_dense;

constexpr int kMaxThreads = 1024;
constexpr int kMaxLanes = 4096;            // channels times slots of a workgroup: 32 KiB of LDS for two floats each
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

// Which columns: a workgroup covers `cols` vectors of V channels from channel c0, `slots` rows at a time; its
// threads are slot-major.  live = false for the threads that round the workgroup up to whole wavefronts.
struct Lane { int slot, col, c; bool live; };

__device__ __forceinline__ Lane lane_of(int c0, int cols, int slots, int total_cols, int V) {
    const int slot = threadIdx.x / cols, col = threadIdx.x - slot * cols;
    return {slot, col, c0 + col * V, slot < slots && c0 / V + col < total_cols};
}

__device__ __forceinline__ float sigmoid(float u) { return 1.f / (1.f + __expf(-u)); }

__device__ __forceinline__ float activate(float u, int act) {
    if (act == CBM_ACT_RELU) return u < 0.f ? 0.f : u;      // NaN stays NaN
    if (act == CBM_ACT_SILU) return u * sigmoid(u);
    return u;
}

// act'(u) dy; the ReLU's derivative at zero is zero
__device__ __forceinline__ float activate_grad(float u, float dy, int act) {
    if (act == CBM_ACT_RELU) return u > 0.f ? dy : (u != u ? u : 0.f);
    if (act == CBM_ACT_SILU) {
        const float s = sigmoid(u);
        return dy * (s * (1.f + u * (1.f - s)));
    }
    return dy;
}

// (n, mean, m2) of both halves of a set -> of the whole
__device__ __forceinline__ void join(float& n, float& mean, float& m2, float nb, float mb, float m2b) {
    const float t = n + nb;
    if (nb == 0.f) return;
    const float w = nb / t, d = mb - mean;
    mean += d * w;
    m2 += m2b + d * d * (n * w);
    n = t;
}

// Mean and centred sum of squares per channel of the rows slot, slot + slots, ... < rows.
template <typename T, int V>
__device__ __forceinline__ void thread_stats(const T* __restrict__ x, int64_t ld, int rows, int slot, int slots,
                                             float (&mean)[V], float (&m2)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    float n = 0.f;
    for (int r = slot; r < rows; r += kBatch * slots) {
        float v[kBatch][V];
        const int have = min(kBatch, (rows - r + slots - 1) / slots);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)                    // rows past the end: the last row again, not counted
            load_as_f32<T, V>(x + static_cast<int64_t>(min(r + k * slots, rows - 1)) * ld, v[k]);
        const float cnt = static_cast<float>(have), inv = 1.f / cnt, t = n + cnt, w = cnt / t;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = 0.f, q = 0.f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) s += k < have ? v[k][i] : 0.f;
            const float m = s * inv;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const float d = k < have ? v[k][i] - m : 0.f;
                q = __builtin_fmaf(d, d, q);
            }
            const float d = m - mean[i];
            mean[i] += d * w;
            m2[i] += q + d * d * (n * w);
        }
        n = t;
    }
}

__device__ __forceinline__ float rows_of_slot(int rows, int slot, int slots) {
    return static_cast<float>(rows > slot ? (rows - slot + slots - 1) / slots : 0);
}

// Joins the slots' channel statistics in LDS: afterwards a[c], b[c] (c < cols * V) hold mean and m2 over all rows.
template <int V>
__device__ __forceinline__ void join_slots(float (&mean)[V], float (&m2)[V], float* a, float* b, int cols, int slots,
                                           const Lane& L, int rows) {
    const int width = cols * V, at = L.slot * width + L.col * V;
    float n = rows_of_slot(rows, L.slot, slots);
    if (L.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a[at + i] = mean[i]; b[at + i] = m2[i]; }
    }
    __syncthreads();
    int half = 1;
    while (half < slots) half <<= 1;
    // n of a joined slot is the number of rows of all slots congruent to it modulo `half`
    for (half >>= 1; half > 0; half >>= 1) {
        if (L.live && L.slot < half && L.slot + half < slots) {
            float nb = 0.f;
            for (int s = L.slot + half; s < slots; s += 2 * half) nb += rows_of_slot(rows, s, slots);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float k = n;
                join(k, mean[i], m2[i], nb, a[at + half * width + i], b[at + half * width + i]);
                a[at + i] = mean[i];
                b[at + i] = m2[i];
            }
            n += nb;
        }
        __syncthreads();
    }
}

// Sums two values per channel over the slots in LDS: afterwards a[c], b[c] hold them.
template <int V>
__device__ __forceinline__ void sum_slots(float (&p1)[V], float (&p2)[V], float* a, float* b, int cols, int slots, const Lane& L) {
    const int width = cols * V, at = L.slot * width + L.col * V;
    if (L.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a[at + i] = p1[i]; b[at + i] = p2[i]; }
    }
    __syncthreads();
    int half = 1;
    while (half < slots) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        if (L.live && L.slot < half && L.slot + half < slots) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p1[i] += a[at + half * width + i];
                p2[i] += b[at + half * width + i];
                a[at + i] = p1[i];
                b[at + i] = p2[i];
            }
        }
        __syncthreads();
    }
}

template <typename T, int V>
__device__ __forceinline__ void write_rows(const T* __restrict__ x, T* __restrict__ y, int64_t ldx, int64_t ldy, int rows,
                                           const Lane& L, int slots, const float (&mean)[V], const float (&scale)[V],
                                           const float (&shift)[V], int act) {
    for (int r = L.slot; r < rows; r += kApplyBatch * slots) {
        float v[kApplyBatch][V];
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k)
            load_as_f32<T, V>(x + static_cast<int64_t>(min(r + k * slots, rows - 1)) * ldx, v[k]);
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            if (r + k * slots >= rows) break;
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = activate(__builtin_fmaf(v[k][i] - mean[i], scale[i], shift[i]), act);
            store_from_f32<T, V>(y + static_cast<int64_t>(r + k * slots) * ldy, v[k]);
        }
    }
}

// Channel sums of d and d xh over the rows of a thread.
template <typename T, int V>
__device__ __forceinline__ void thread_grad_sums(const T* __restrict__ x, const T* __restrict__ dy, int64_t ldx, int64_t ldg,
                                                 int rows, int slot, int slots, const float (&mean)[V], const float (&rstd)[V],
                                                 const float (&w)[V], const float (&b)[V], int act, float (&p1)[V], float (&p2)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) p1[i] = p2[i] = 0.f;
    for (int r = slot; r < rows; r += kApplyBatch * slots) {
        float v[kApplyBatch][V], g[kApplyBatch][V];
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            const int64_t row = min(r + k * slots, rows - 1);
            load_as_f32<T, V>(x + row * ldx, v[k]);
            load_as_f32<T, V>(dy + row * ldg, g[k]);
        }
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            const bool in = r + k * slots < rows;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (v[k][i] - mean[i]) * rstd[i];
                const float d = in ? activate_grad(__builtin_fmaf(xh, w[i], b[i]), g[k][i], act) : 0.f;
                p1[i] += d;
                p2[i] += in ? d * xh : 0.f;
            }
        }
    }
}

// dx = r (d w - c1 - xh c2) with c1 = S1 / M, c2 = S2 / M
template <typename T, int V>
__device__ __forceinline__ void write_grad_rows(const T* __restrict__ x, const T* __restrict__ dy, T* __restrict__ dx, int64_t ldx,
                                                int64_t ldg, int64_t ldd, int rows, const Lane& L, int slots, const float (&mean)[V],
                                                const float (&rstd)[V], const float (&w)[V], const float (&b)[V],
                                                const float (&c1)[V], const float (&c2)[V], int act) {
    for (int r = L.slot; r < rows; r += kApplyBatch * slots) {
        float v[kApplyBatch][V], g[kApplyBatch][V];
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            const int64_t row = min(r + k * slots, rows - 1);
            load_as_f32<T, V>(x + row * ldx, v[k]);
            load_as_f32<T, V>(dy + row * ldg, g[k]);
        }
#pragma unroll
        for (int k = 0; k < kApplyBatch; ++k) {
            if (r + k * slots >= rows) break;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (v[k][i] - mean[i]) * rstd[i];
                const float d = activate_grad(__builtin_fmaf(xh, w[i], b[i]), g[k][i], act);
                v[k][i] = rstd[i] * (__builtin_fmaf(d, w[i], -c1[i]) - xh * c2[i]);
            }
            store_from_f32<T, V>(dx + static_cast<int64_t>(r + k * slots) * ldd, v[k]);
        }
    }
}

template <int V>
__device__ __forceinline__ void channel_params(const float* __restrict__ p, float otherwise, int c, bool live, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (p && live) ? p[c + i] : otherwise;
}

struct Shape {
    int C, D, groups, total_cols, cols, slots, act;
    int64_t ldx, ldy, ldg;
    float eps;
};

// ---------------------------------------------------------------------------------------------
// one launch: workgroup (sample, block of whole groups)
// ---------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_forward_one(const T* __restrict__ X, T* __restrict__ Y,
                                                                const float* __restrict__ weight, const float* __restrict__ bias,
                                                                const int* __restrict__ ptr, int len, int groups_per_block,
                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out, Shape S) {
    extern __shared__ float lds[];
    const int s = blockIdx.x, g0 = blockIdx.y * groups_per_block, ng = min(groups_per_block, S.groups - g0);
    const int row0 = ptr ? ptr[s] : s * len, rows = ptr ? ptr[s + 1] - row0 : len;
    const int c0 = g0 * S.D, width = S.cols * V;
    const Lane L = lane_of(c0, S.cols, S.slots, (c0 + ng * S.D) / V, V);
    float* a = lds;
    float* b = a + S.slots * width;
    float* gm = b + S.slots * width;                       // mean and 1/std of the workgroup's groups
    float* gr = gm + groups_per_block;
    const T* x = X + static_cast<int64_t>(row0) * S.ldx + L.c;
    float mean[V], m2[V];
    thread_stats<T, V>(x, S.ldx, L.live ? rows : 0, L.slot, S.slots, mean, m2);
    join_slots<V>(mean, m2, a, b, S.cols, S.slots, L, rows);
    // the channels of a group have the same number of rows: group mean = mean of channel means
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, waves = blockDim.x / kWave;
    for (int g = wave; g < ng; g += waves) {
        float sum = 0.f, sq = 0.f;
        for (int i = lane; i < S.D; i += kWave) sum += a[g * S.D + i];
        const float m = wave_sum(sum) / static_cast<float>(S.D);
        for (int i = lane; i < S.D; i += kWave) {
            const float d = a[g * S.D + i] - m;
            sq += b[g * S.D + i] + d * d * static_cast<float>(rows);
        }
        const float count = static_cast<float>(rows) * static_cast<float>(S.D);
        const float r = 1.f / sqrtf((rows ? wave_sum(sq) / count : 0.f) + S.eps);
        if (lane == 0) {
            gm[g] = m;
            gr[g] = r;
            if (mean_out) {
                mean_out[static_cast<int64_t>(s) * S.groups + g0 + g] = m;
                rstd_out[static_cast<int64_t>(s) * S.groups + g0 + g] = r;
            }
        }
    }
    __syncthreads();
    if (!L.live) return;
    float scale[V], shift[V];
    channel_params<V>(weight, 1.f, L.c, true, scale);
    channel_params<V>(bias, 0.f, L.c, true, shift);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = (L.c + i - c0) / S.D;
        mean[i] = gm[g];
        scale[i] *= gr[g];
    }
    write_rows<T, V>(x, Y + static_cast<int64_t>(row0) * S.ldy + L.c, S.ldx, S.ldy, rows, L, S.slots, mean, scale, shift, S.act);
}

// Workgroup (i, block of groups) takes the samples i, i + gridDim.x, ...; its sums for dw and db over all of them
// go to part[(2 i + which) C + c].
template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_backward_one(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ DX,
                                                                 const float* __restrict__ weight, const float* __restrict__ bias,
                                                                 const int* __restrict__ ptr, int len, int samples, int groups_per_block,
                                                                 const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                 float* __restrict__ part, int64_t ldd, Shape S) {
    extern __shared__ float lds[];
    const int g0 = blockIdx.y * groups_per_block, ng = min(groups_per_block, S.groups - g0);
    const int c0 = g0 * S.D, width = S.cols * V;
    const Lane L = lane_of(c0, S.cols, S.slots, (c0 + ng * S.D) / V, V);
    float* a = lds;
    float* b = a + S.slots * width;
    float* gs1 = b + S.slots * width;
    float* gs2 = gs1 + groups_per_block;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, waves = blockDim.x / kWave;
    float w[V], bi[V], dw[V], db[V];
    channel_params<V>(weight, 1.f, L.c, L.live, w);
    channel_params<V>(bias, 0.f, L.c, L.live, bi);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
    for (int s = blockIdx.x; s < samples; s += gridDim.x) {
        const int row0 = ptr ? ptr[s] : s * len, rows = ptr ? ptr[s + 1] - row0 : len;
        if (rows == 0) continue;                            // the same for the whole workgroup
        float mean[V], rstd[V], p1[V], p2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int64_t at = static_cast<int64_t>(s) * S.groups + (L.live ? (L.c + i) / S.D : 0);
            mean[i] = mean_in[at];
            rstd[i] = rstd_in[at];
        }
        const T* x = X + static_cast<int64_t>(row0) * S.ldx + L.c;
        const T* dy = DY + static_cast<int64_t>(row0) * S.ldg + L.c;
        thread_grad_sums<T, V>(x, dy, S.ldx, S.ldg, L.live ? rows : 0, L.slot, S.slots, mean, rstd, w, bi, S.act, p1, p2);
        sum_slots<V>(p1, p2, a, b, S.cols, S.slots, L);
        if (L.live && L.slot == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) { db[i] += p1[i]; dw[i] += p2[i]; }
        }
        if (DX) {
            const float inv = 1.f / (static_cast<float>(rows) * static_cast<float>(S.D));
            for (int g = wave; g < ng; g += waves) {
                float s1 = 0.f, s2 = 0.f;
                for (int i = lane; i < S.D; i += kWave) {
                    const float wc = weight ? weight[c0 + g * S.D + i] : 1.f;
                    s1 += wc * a[g * S.D + i];
                    s2 += wc * b[g * S.D + i];
                }
                s1 = wave_sum(s1);
                s2 = wave_sum(s2);
                if (lane == 0) { gs1[g] = s1 * inv; gs2[g] = s2 * inv; }
            }
            __syncthreads();
            if (L.live) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int g = (L.c + i - c0) / S.D;
                    p1[i] = gs1[g];
                    p2[i] = gs2[g];
                }
                write_grad_rows<T, V>(x, dy, DX + static_cast<int64_t>(row0) * ldd + L.c, S.ldx, S.ldg, ldd, rows, L, S.slots, mean, rstd,
                                      w, bi, p1, p2, S.act);
            }
        }
        __syncthreads();                                    // a, b, gs1, gs2 are free again
    }
    if (part && L.live && L.slot == 0) {
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
    const Lane L = lane_of(blockIdx.y * S.cols * V, S.cols, S.slots, S.total_cols, V);
    float mean[V], m2[V];
    thread_stats<T, V>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, S.ldx, L.live ? P.rows : 0, L.slot, S.slots, mean, m2);
    join_slots<V>(mean, m2, lds, lds + S.slots * S.cols * V, S.cols, S.slots, L, P.rows);
    if (L.live && L.slot == 0) {
        float* o = part + static_cast<int64_t>(blockIdx.x) * 2 * S.C + L.c;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = mean[i]; o[S.C + i] = m2[i]; }
    }
}

__device__ __forceinline__ void pieces_of(const Rows& R, int s, int& p0, int& np) {
    p0 = R.piece_ptr ? R.piece_ptr[s] : s * R.per_sample;
    np = R.piece_ptr ? R.piece_ptr[s + 1] - p0 : R.per_sample;
}

// Joins the pieces' channel statistics: one workgroup per (sample, group).
__global__ __launch_bounds__(kMaxThreads) void norm_join_stats(const float* __restrict__ part, float* __restrict__ mean_out,
                                                               float* __restrict__ rstd_out, Rows R, Shape S) {
    __shared__ float red[kMaxThreads / kWave];
    const int s = blockIdx.x / S.groups, g = blockIdx.x - s * S.groups;
    int p0, np;
    pieces_of(R, s, p0, np);
    const int items = np * S.D;
    float sum = 0.f, rows = 0.f;
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int p = i / S.D, c = i - p * S.D;
        const float n = static_cast<float>(piece_of(R, p0 + p).rows);
        sum += n * part[static_cast<int64_t>(p0 + p) * 2 * S.C + g * S.D + c];
        rows += c == 0 ? n : 0.f;
    }
    rows = block_sum(rows, red);
    const float count = rows * static_cast<float>(S.D);
    const float mean = count > 0.f ? block_sum(sum, red) / count : 0.f;
    float sq = 0.f;
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int p = i / S.D, c = i - p * S.D;
        const float n = static_cast<float>(piece_of(R, p0 + p).rows);
        const float* at = part + static_cast<int64_t>(p0 + p) * 2 * S.C + g * S.D + c;
        const float d = at[0] - mean;
        sq += at[S.C] + n * d * d;
    }
    const float var = count > 0.f ? block_sum(sq, red) / count : 0.f;
    if (threadIdx.x == 0) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = 1.f / sqrtf(var + S.eps);
    }
}

template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_apply_pieces(const T* __restrict__ X, T* __restrict__ Y, const float* __restrict__ weight,
                                                                 const float* __restrict__ bias, const float* __restrict__ mean_in,
                                                                 const float* __restrict__ rstd_in, Rows R, Shape S) {
    const Piece P = piece_of(R, blockIdx.x);
    const Lane L = lane_of(blockIdx.y * S.cols * V, S.cols, S.slots, S.total_cols, V);
    if (!L.live) return;
    float mean[V], scale[V], shift[V];
    channel_params<V>(weight, 1.f, L.c, true, scale);
    channel_params<V>(bias, 0.f, L.c, true, shift);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int64_t at = static_cast<int64_t>(P.s) * S.groups + (L.c + i) / S.D;
        mean[i] = mean_in[at];
        scale[i] *= rstd_in[at];
    }
    write_rows<T, V>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, Y + static_cast<int64_t>(P.row0) * S.ldy + L.c, S.ldx, S.ldy, P.rows,
                     L, S.slots, mean, scale, shift, S.act);
}

template <typename T, int V>
__global__ __launch_bounds__(most_threads(V)) void norm_grad_pieces(const T* __restrict__ X, const T* __restrict__ DY,
                                                                const float* __restrict__ weight, const float* __restrict__ bias,
                                                                const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                float* __restrict__ part, Rows R, Shape S) {
    extern __shared__ float lds[];
    const Piece P = piece_of(R, blockIdx.x);
    const Lane L = lane_of(blockIdx.y * S.cols * V, S.cols, S.slots, S.total_cols, V);
    float mean[V], rstd[V], w[V], b[V], p1[V], p2[V];
    channel_params<V>(weight, 1.f, L.c, L.live, w);
    channel_params<V>(bias, 0.f, L.c, L.live, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int64_t at = static_cast<int64_t>(P.s) * S.groups + (L.live ? (L.c + i) / S.D : 0);
        mean[i] = mean_in[at];
        rstd[i] = rstd_in[at];
    }
    thread_grad_sums<T, V>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, DY + static_cast<int64_t>(P.row0) * S.ldg + L.c, S.ldx, S.ldg,
                           L.live ? P.rows : 0, L.slot, S.slots, mean, rstd, w, b, S.act, p1, p2);
    sum_slots<V>(p1, p2, lds, lds + S.slots * S.cols * V, S.cols, S.slots, L);
    if (L.live && L.slot == 0) {
        float* o = part + static_cast<int64_t>(blockIdx.x) * 2 * S.C + L.c;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = p1[i]; o[S.C + i] = p2[i]; }
    }
}

// Workgroups [0, pairs): S1 / M and S2 / M of a (sample, group).  The rest: dw and db of 32 channels each, the
// partial sums of all `parts` rows of part.  1024 threads.
__global__ __launch_bounds__(kMaxThreads) void norm_join_grads(const float* __restrict__ part, const float* __restrict__ weight,
                                                               float* __restrict__ c1_out, float* __restrict__ c2_out,
                                                               float* __restrict__ dw, float* __restrict__ db, int pairs, int parts,
                                                               Rows R, Shape S) {
    __shared__ float red[2][kMaxThreads];
    if (static_cast<int>(blockIdx.x) < pairs) {
        const int s = blockIdx.x / S.groups, g = blockIdx.x - s * S.groups;
        int p0, np;
        pieces_of(R, s, p0, np);
        const int items = np * S.D;
        float s1 = 0.f, s2 = 0.f, rows = 0.f;
        for (int i = threadIdx.x; i < items; i += blockDim.x) {
            const int p = i / S.D, c = i - p * S.D;
            const float* at = part + static_cast<int64_t>(p0 + p) * 2 * S.C + g * S.D + c;
            const float w = weight ? weight[g * S.D + c] : 1.f;
            s1 += w * at[0];
            s2 += w * at[S.C];
            rows += c == 0 ? static_cast<float>(piece_of(R, p0 + p).rows) : 0.f;
        }
        rows = block_sum(rows, red[0]);
        s1 = block_sum(s1, red[0]);
        s2 = block_sum(s2, red[0]);
        if (threadIdx.x == 0) {
            const float inv = rows > 0.f ? 1.f / (rows * static_cast<float>(S.D)) : 0.f;
            c1_out[blockIdx.x] = s1 * inv;
            c2_out[blockIdx.x] = s2 * inv;
        }
        return;
    }
    const int c = (blockIdx.x - pairs) * 32 + threadIdx.x % 32, k = threadIdx.x / 32;
    float v1 = 0.f, v2 = 0.f;
    if (c < S.C)
        for (int p = k; p < parts; p += kMaxThreads / 32) {
            v1 += part[static_cast<int64_t>(p) * 2 * S.C + c];
            v2 += part[static_cast<int64_t>(p) * 2 * S.C + S.C + c];
        }
    red[0][threadIdx.x] = v1;
    red[1][threadIdx.x] = v2;
    __syncthreads();
    for (int half = kMaxThreads / 64; half > 0; half >>= 1) {
        if (k < half) {
            red[0][threadIdx.x] += red[0][threadIdx.x + 32 * half];
            red[1][threadIdx.x] += red[1][threadIdx.x + 32 * half];
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
    const Piece P = piece_of(R, blockIdx.x);
    const Lane L = lane_of(blockIdx.y * S.cols * V, S.cols, S.slots, S.total_cols, V);
    if (!L.live) return;
    float mean[V], rstd[V], w[V], b[V], c1[V], c2[V];
    channel_params<V>(weight, 1.f, L.c, true, w);
    channel_params<V>(bias, 0.f, L.c, true, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int64_t at = static_cast<int64_t>(P.s) * S.groups + (L.c + i) / S.D;
        mean[i] = mean_in[at];
        rstd[i] = rstd_in[at];
        c1[i] = c1_in[at];
        c2[i] = c2_in[at];
    }
    write_grad_rows<T, V>(X + static_cast<int64_t>(P.row0) * S.ldx + L.c, DY + static_cast<int64_t>(P.row0) * S.ldg + L.c,
                          DX + static_cast<int64_t>(P.row0) * ldd + L.c, S.ldx, S.ldg, ldd, P.rows, L, S.slots, mean, rstd, w, b, c1, c2, S.act);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Elements of one vector: 16 bytes where the rows of every array divide into them, else the largest power of two
// that divides the width.  (Vectors need no alignment beyond an element's.)
int vector_of(int dtype, int C) {
    int v = 16 / element_bytes(dtype);
    while (C % v) v >>= 1;
    return v;
}

// One launch or pieces: pieces cost two more launches (~5 us each), one launch leaves a graph to one workgroup,
// which streams about 50 bytes per ns.
constexpr int64_t kOneLaunchBytes = 256 << 10;
constexpr int kBackwardGroups = 1024;      // most workgroups that walk the samples of a one-launch backward

struct Plan {
    bool one;
    int V, cols, slots, threads, blocks_y, groups_per_block;
};

int slots_of(int cols, int want_threads) { return std::max(1, want_threads / cols); }

Plan plan_of(const cbm_norm_batch* B, int C, int groups, int dtype) {
    Plan P{};
    const int D = C / groups;
    P.V = vector_of(dtype, C);
    const int total = C / P.V, most = most_threads(P.V);
    P.groups_per_block = groups;
    // few graphs: split the groups of a graph over workgroups, in shares of whole vectors and at least 32 bytes a row
    auto splits = [&](int gpb) {
        const int64_t c = static_cast<int64_t>(gpb) * D;
        return c % P.V == 0 && c * element_bytes(dtype) >= 32 && c / P.V <= most;
    };
    if (total > most || B->samples < 64) {
        int best = 0;
        for (int gpb = 1; gpb <= groups; ++gpb)
            if (groups % gpb == 0 && splits(gpb)) { best = gpb; break; }
        P.groups_per_block = best ? best : (total <= most ? groups : 0);
    }
    P.one = P.groups_per_block > 0 && P.groups_per_block <= 4096 &&
            static_cast<int64_t>(B->max_len) * P.groups_per_block * D * element_bytes(dtype) <= kOneLaunchBytes;
    if (P.one) {
        P.cols = P.groups_per_block * D / P.V;
        P.blocks_y = groups / P.groups_per_block;
    } else {
        P.blocks_y = (total + most - 1) / most;
        P.cols = (total + P.blocks_y - 1) / P.blocks_y;
    }
    // no more slots than rows; a graph alone gets the largest workgroup
    const int want = P.one && B->samples < 64 ? most : 256;
    P.slots = std::min(slots_of(P.cols, want), std::max(1, static_cast<int>(B->max_len)));
    P.threads = (P.cols * P.slots + kWave - 1) / kWave * kWave;
    return P;
}

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
    if (static_cast<int64_t>(B->samples) * groups > (1 << 30)) return CBM_ERR_SHAPE;
    if (!B->ptr && static_cast<int64_t>(B->samples) * B->max_len != B->rows) return CBM_ERR_SHAPE;
    if (B->ptr && B->rows > 0 && (!B->pieces || !B->piece_ptr || B->n_pieces < 1)) return CBM_ERR_NULL;
    if (B->rows > 0 && B->piece_rows < 1) return CBM_ERR_SHAPE;
    return CBM_OK;
}

size_t lds_of(const Plan& P) {
    return sizeof(float) * (2u * P.slots * P.cols * P.V + 2u * (P.one ? P.groups_per_block : 0));
}

#define CBM_NORM_BY_VECTOR(T, VMAX, CALL)                        \
    switch (P.V) {                                               \
        case 1: { constexpr int V = 1; CALL(T, V); } break;      \
        case 2: { constexpr int V = 2; CALL(T, V); } break;      \
        case 4: { constexpr int V = 4; CALL(T, V); } break;      \
        default: { constexpr int V = VMAX; CALL(T, V); } break;  \
    }
#define CBM_NORM_BY_TYPE(CALL)                                                \
    if (dtype == CBM_DTYPE_F32) { CBM_NORM_BY_VECTOR(float, 4, CALL) }        \
    else if (dtype == CBM_DTYPE_BF16) { CBM_NORM_BY_VECTOR(__bf16, 8, CALL) } \
    else { CBM_NORM_BY_VECTOR(_Float16, 8, CALL) }

}  // namespace

extern "C" {

int64_t cbm_group_norm_workspace_floats(const cbm_norm_batch* B, int32_t C, int32_t groups, int32_t dtype, int32_t backward) {
    if (check_batch(B, C, groups, dtype, CBM_ACT_NONE) != CBM_OK || B->rows == 0) return 0;
    const Plan P = plan_of(B, C, groups, dtype);
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan P = plan_of(B, C, groups, dtype);
    const Rows R = rows_of(B);
    Shape S{C, C / groups, groups, C / P.V, P.cols, P.slots, act, ldx, ldy, 0, eps};
    if (P.one) {
#define ONE(T, V)                                                                                                                     \
    hipLaunchKernelGGL((norm_forward_one<T, V>), dim3(B->samples, P.blocks_y), dim3(P.threads), lds_of(P), st,                        \
                       static_cast<const T*>(X), static_cast<T*>(Y), weight, bias, B->ptr, B->max_len, P.groups_per_block, mean, rstd, S)
        CBM_NORM_BY_TYPE(ONE)
#undef ONE
        return check_launch();
    }
    if (!workspace) return CBM_ERR_NULL;
    const int np = pieces_total(B, R);
    const int64_t pairs = static_cast<int64_t>(B->samples) * groups;
    float* part = workspace;
    float* m = mean ? mean : workspace + 2LL * C * np;
    float* r = rstd ? rstd : m + pairs;
    const int64_t items = static_cast<int64_t>(np) * S.D / B->samples;
#define STATS(T, V)                                                                                                                \
    hipLaunchKernelGGL((norm_stats_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), lds_of(P), st, static_cast<const T*>(X), \
                       part, R, S)
#define APPLY(T, V)                                                                                                          \
    hipLaunchKernelGGL((norm_apply_pieces<T, V>), dim3(np, P.blocks_y), dim3(P.threads), 0, st, static_cast<const T*>(X),    \
                       static_cast<T*>(Y), weight, bias, m, r, R, S)
    CBM_NORM_BY_TYPE(STATS)
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(norm_join_stats, dim3(static_cast<unsigned>(pairs)), dim3(items >= 2048 ? 1024 : items >= 256 ? 256 : 64), 0, st,
                       part, m, r, R, S);
    if (int rc = check_launch()) return rc;
    CBM_NORM_BY_TYPE(APPLY)
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool params = dweight || dbias;
    if (B->rows > 0 && !workspace) return CBM_ERR_NULL;
    const unsigned channel_blocks = static_cast<unsigned>((C + 31) / 32);
    if (B->rows == 0) {                                    // no rows: the parameters' gradients are zero
        Shape S{C, C / groups, groups, C, 0, 0, act, 0, 0, 0, 0.f};
        if (!params) return CBM_OK;
        hipLaunchKernelGGL(norm_join_grads, dim3(channel_blocks), dim3(kMaxThreads), 0, st, nullptr, weight, nullptr, nullptr, dweight,
                           dbias, 0, 0, Rows{}, S);
        return check_launch();
    }
    const Plan P = plan_of(B, C, groups, dtype);
    const Rows R = rows_of(B);
    Shape S{C, C / groups, groups, C / P.V, P.cols, P.slots, act, ldx, 0, ldg, 0.f};
    if (P.one) {
        const int walkers = std::min(B->samples, kBackwardGroups);
#define ONE(T, V)                                                                                                                   \
    hipLaunchKernelGGL((norm_backward_one<T, V>), dim3(walkers, P.blocks_y), dim3(P.threads), lds_of(P), st,                        \
                       static_cast<const T*>(X), static_cast<const T*>(DY), static_cast<T*>(DX), weight, bias, B->ptr, B->max_len,  \
                       B->samples, P.groups_per_block, mean, rstd, params ? workspace : nullptr, ldd, S)
        CBM_NORM_BY_TYPE(ONE)
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
    CBM_NORM_BY_TYPE(SUMS)
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(norm_join_grads, dim3(pairs + (params ? channel_blocks : 0)), dim3(kMaxThreads), 0, st, part, weight, c1, c2,
                       dweight, dbias, pairs, np, R, S);
    if (int rc = check_launch()) return rc;
    if (!DX) return CBM_OK;
    CBM_NORM_BY_TYPE(APPLY)
#undef SUMS
#undef APPLY
    return check_launch();
}

}  // extern "C"
