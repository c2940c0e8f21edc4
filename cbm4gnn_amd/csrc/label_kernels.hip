// Scores of labels: log probability of the given class, entropy of the distribution and the likeliest classes of
// every row of logits [rows, classes], and the gradient of the logits.
//
//     m = max z,  S = sum exp(z - m),  log p_j = (z_j - m) - log S,  H = log S - sum exp(z - m) (z - m) / S
//     dz_j = gl [j = label] + sum_i gt_i [j = top_i] - p_j (gl + sum_i gt_i + gH (log p_j + H))
//
// m and log S are kept apart (not summed into one float), so logits far from zero cost no digits.
//
// A row is read once and stays in registers for its maximum, its sums and its likeliest classes.  Reading the logits
// bounds the forward, reading them and writing the gradient the backward; with some ten vector instructions a value
// (the exponential alone costs four issue slots) arithmetic is not far behind.
//   narrow   up to 1024 classes: 4 to 64 lanes hold a row in vectors of 16 bytes, up to 16 rows per wavefront;
//   wide     a workgroup per row.  Rows longer than a workgroup's registers, and long rows that are few, are split
//            over workgroups whose partial results a second launch joins.
// Exponentials are the hardware's of the argument times log2 e, off by (2 + |argument|) 2^-24 of their value: two
// instructions each, and no more than a few 1e-8 of the scores (232 965 x 41 fp32, scores and gradient together: 5.1e-8
// against 3.9e-8 with exact ones).  A probability below 2^-126 counts as 0.
// Measured (one MI355X, kernel times): 232 965 x 41 fp32: scores 8.9 us (4.4 TB/s), gradient 17.1 us (4.5 TB/s); in two-byte
// types 8.0 and 12.2 us (2.6 and 3.3 TB/s);  12 000 x 41 fp32 with entropy and 5 classes: 4.8 us;  2 049 x 32 003 bf16 with
// entropy and 8 classes: 54 us (2.4 TB/s), gradient 45 us (5.8 TB/s).  Of those 54, 32 us are its 20 vector instructions a value
// and some 5 the further passes of an exponential; the rest are phases between barriers, one after the other, and the last of
// five workgroups that share a place, which has one row.  1 x 100 000 fp32 with entropy and 10 classes: 7.8 + 5.6 us, two launches' latency.
// The last vector of a row begins where it still fits and overlaps the one before, whose values it ignores.
//
// Likeliest classes order by (value, lowest index): value and index make ONE 64-bit key, so no two are equal and the
// answer does not depend on who looks at what.  Narrow rows take `top` maxima out of registers.  Wide rows first
// find a bound that at least `top` values reach (the `top`-th largest of the maxima of 128 disjoint parts), then
// collect the few values above it into LDS and rank them by counting; a row that crowds more than the list holds
// above its bound takes `top` maxima instead.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense_types.h"

namespace {

using namespace cbm_dense;
using key_t = unsigned long long;

constexpr int kMaxTop = CBM_LABELS_MAX_TOP;
constexpr int kThreads = 256;
constexpr int kParts = 128;                // disjoint parts of a wide row whose maxima bound its likeliest classes
constexpr int kList = 2048;                // candidates a wide row keeps
constexpr float kInf = __builtin_inff();

// Order of values as unsigned numbers: -inf lowest, NaN highest, -0 and +0 equal.  0 stands for no value.
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __float_as_uint(v + 0.f);
    if (v != v) return 0xffc00000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ key_t key_of(unsigned order, unsigned index) {
    return (static_cast<key_t>(order) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned index_of(key_t k) { return 0xffffffffu - static_cast<unsigned>(k); }

template <int L>
__device__ __forceinline__ key_t lanes_max_key(key_t k) {
    reduce_lanes<L>([&](auto o) {
        constexpr int O = decltype(o)::value;
        const Halves lo = halves<O>(static_cast<uint32_t>(k)), hi = halves<O>(static_cast<uint32_t>(k >> 32));
        const key_t a = (static_cast<key_t>(hi.a) << 32) | lo.a, b = (static_cast<key_t>(hi.b) << 32) | lo.b;
        k = a > b ? a : b;
    });
    return k;
}

// Softmax sums: m the maximum, s = sum exp(z - m), t = sum exp(z - m) (z - m).
struct Sums { float m, s, t; };

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    // a part of -inf alone has s = 0 (or NaN, which stays) and moves by factor 0
    const float fa = a.m == -kInf ? 0.f : __expf(a.m - m), fb = b.m == -kInf ? 0.f : __expf(b.m - m);
    const float ta = fa == 0.f ? 0.f : (a.t + a.s * (a.m - m)) * fa, tb = fb == 0.f ? 0.f : (b.t + b.s * (b.m - m)) * fb;
    return {m, a.s * fa + b.s * fb, ta + tb};
}

template <int L>
__device__ __forceinline__ Sums lanes_join(Sums S) {
    reduce_lanes<L>([&](auto o) {
        constexpr int O = decltype(o)::value;
        const Halves m = halves<O>(__float_as_uint(S.m)), s = halves<O>(__float_as_uint(S.s)), t = halves<O>(__float_as_uint(S.t));
        S = join(Sums{__uint_as_float(m.a), __uint_as_float(s.a), __uint_as_float(t.a)},
                 Sums{__uint_as_float(m.b), __uint_as_float(s.b), __uint_as_float(t.b)});
    });
    return S;
}

// Takes one value into sums whose maximum already covers it; base = m, or 0 while m is -inf.  The exponential of
// anything under -200 is 0, so the product's other factor may stop there: exp(-inf) (-inf) counts nothing.
template <bool T>
__device__ __forceinline__ void take(Sums& S, float v, float base) {
    const float d = v - base, e = __expf(d);
    S.s += e;
    if constexpr (T) S.t = __builtin_fmaf(e, fmaxf(d, -200.f), S.t);
}

struct Outputs {
    const int64_t* labels;
    float* logp;
    float* entropy;
    float* top_logp;
    int64_t* top_index;
    float* stats;
    int64_t ignore_index;
    int classes, top;
};

// {m, log S, H} of finished sums; a row of -inf alone gets (0, +inf, 0): every log probability is then -inf
// and every probability 0.
struct Final { float m, log_s, h; };
__device__ __forceinline__ Final finish(const Sums& S) {
    if (S.s == 0.f) return {0.f, kInf, 0.f};
    const float l = logf(S.s);
    return {S.m, l, l - S.t / S.s};
}

template <typename T>
__device__ __forceinline__ void write_scores(const Outputs& O, const T* __restrict__ row, int64_t r, const Final& F) {
    if (O.stats) *reinterpret_cast<float2*>(O.stats + 2 * r) = make_float2(F.m, F.log_s);
    if (O.entropy) O.entropy[r] = F.h;
    if (O.logp) {
        const int64_t y = O.labels[r];
        float v = __builtin_nanf("");
        if (y == O.ignore_index) v = 0.f;
        else if (y >= 0 && y < O.classes) v = (static_cast<float>(row[y]) - F.m) - F.log_s;
        O.logp[r] = v;
    }
}

__device__ __forceinline__ void write_top(const Outputs& O, int64_t r, int i, key_t k, const Final& F) {
    O.top_logp[r * O.top + i] = (value_of(static_cast<unsigned>(k >> 32)) - F.m) - F.log_s;
    O.top_index[r * O.top + i] = index_of(k);
}

// Vector i of the columns [.., hi): its columns at .. at + V - 1, of which those from `first` on are its own.
struct Place { int at, first; };
template <int V>
__device__ __forceinline__ Place place_of(int first, int hi) { return {min(first, hi - V), first}; }

// ---------------------------------------------------------------------------------------------
// narrow rows: vector j of lane l covers the columns (l + L j) V ..; only the last j meets the row's end
// ---------------------------------------------------------------------------------------------
template <typename T, int V, int L, int NV>
__device__ __forceinline__ void load_narrow(const T* __restrict__ row, int lane, int classes, float otherwise, float (&v)[NV][V]) {
    Raw<T, V> raw[NV];
    const Place last = place_of<V>((lane + L * (NV - 1)) * V, classes);
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j] = load_raw<T, V>(row + (j < NV - 1 ? (lane + L * j) * V : last.at));
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = j < NV - 1 || last.at + i >= last.first ? raw[j][i] : otherwise;
}

// ALL: entropy or likeliest classes are asked for too
template <typename T, int V, int L, int NV, bool ALL>
__global__ __launch_bounds__(kThreads) void label_scores_narrow(const T* __restrict__ Z, int64_t ld, int rows, Outputs O) {
    const int lane = threadIdx.x % L;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
    const T* row = Z + min(r, static_cast<int64_t>(rows - 1)) * ld;
    float v[NV][V];
    load_narrow<T, V, L, NV>(row, lane, O.classes, -kInf, v);
    Sums S{-kInf, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) S.m = fmaxf(S.m, v[j][i]);
    S.m = lanes_max<L>(S.m);
    const float base = S.m == -kInf ? 0.f : S.m;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) take<ALL>(S, v[j][i], base);
    S.s = lanes_sum<L>(S.s);
    if constexpr (ALL) S.t = lanes_sum<L>(S.t);
    const Final F = finish(S);
    const bool mine = r < rows && lane == 0;
    if (mine) write_scores<T>(O, row, r, F);
    if constexpr (ALL) {
        const Place last = place_of<V>((lane + L * (NV - 1)) * V, O.classes);
        unsigned taken = 0;
        for (int i = 0; i < O.top; ++i) {
            unsigned best = 0, at = 0, bit = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const unsigned b = 1u << (j * V + e), c = (j < NV - 1 ? (lane + L * j) * V : last.at) + e;
                    const bool own = j < NV - 1 || last.at + e >= last.first;
                    const unsigned o = own && !(taken & b) ? order_of(v[j][e]) : 0u;
                    if (o > best) { best = o; at = c; bit = b; }
                }
            const key_t mine_k = best ? key_of(best, at) : 0, k = lanes_max_key<L>(mine_k);
            if (best && k == mine_k) taken |= bit;
            if (mine) write_top(O, r, i, k, F);
        }
    }
}

struct Grads {
    const int64_t* labels;
    const float* stats;
    const float* entropy;
    const int64_t* top_index;
    const float* g_logp;
    const float* g_entropy;
    const float* g_top;
    int64_t ignore_index;
    int classes, top;
};

// What a row's gradient needs: dz_j = -p_j (all + gh (log p_j + h)) + gl [j = label] (+ the likeliest classes').
// A row of -inf alone has no gradient (any = false), and neither has one whose label is ignored and to which nothing else
// flows: a row that is left out may hold NaN or +inf, which times zero would be NaN.
struct RowGrad { float m, log_s, h, gl, gh, all; int label; bool any; };
__device__ __forceinline__ RowGrad row_grad(const Grads& G, int64_t r) {
    const float2 st = *reinterpret_cast<const float2*>(G.stats + 2 * r);
    RowGrad R{st.x, st.y, 0.f, 0.f, 0.f, 0.f, -1, st.y != kInf};
    if (!R.any) return R;
    bool left_out = false;
    if (G.g_entropy) { R.gh = G.g_entropy[r]; R.h = G.entropy[r]; }
    if (G.g_logp) {
        const int64_t y = G.labels[r];
        const float g = G.g_logp[r];
        if (y != G.ignore_index) {
            const bool in = y >= 0 && y < G.classes;
            R.gl = in ? g : __builtin_nanf("");
            R.label = in ? static_cast<int>(y) : -1;
        } else {
            left_out = R.gh == 0.f;
        }
    }
    R.all = R.gl;
    if (G.g_top)
        for (int i = 0; i < G.top; ++i) {
            const float g = G.g_top[r * G.top + i];
            R.all += g;
            left_out = left_out && g == 0.f;
        }
    if (left_out) R.any = false;
    return R;
}
template <bool H>
__device__ __forceinline__ float grad_of(const RowGrad& R, float z, int c) {
    const float lp = (z - R.m) - R.log_s, p = __expf(lp);
    // p = 0: nothing, also where log p is -inf; a NaN goes through
    const float inner = H ? __builtin_fmaf(R.gh, (p == 0.f ? 0.f : lp) + R.h, R.all) : R.all;
    return __builtin_fmaf(-p, inner, c == R.label ? R.gl : 0.f);
}

template <typename T, int V, int L, int NV>
__global__ __launch_bounds__(kThreads) void label_grads_narrow(const T* __restrict__ Z, T* __restrict__ D, int64_t ld, int64_t ldg,
                                                               int rows, Grads G) {
    const int lane = threadIdx.x % L;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
    if (r >= rows) return;
    float v[NV][V];
    load_narrow<T, V, L, NV>(Z + r * ld, lane, G.classes, 0.f, v);
    const RowGrad R = row_grad(G, r);
    // the last vector's overlap belongs to a neighbour; both write the same bits there
    const Place last = place_of<V>((lane + L * (NV - 1)) * V, G.classes);
    T* out = D + r * ldg;
    const bool likeliest = G.g_top && R.any;
    float z[V];
    if (last.at < last.first) {                            // the overlap's values, which load_narrow left out
        const Raw<T, V> raw = load_raw<T, V>(Z + r * ld + last.at);
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = v[NV - 1][i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[NV - 1][i] = z[i];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = j < NV - 1 ? (lane + L * j) * V : last.at;
        if (G.g_entropy) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = R.any ? grad_of<true>(R, v[j][i], at + i) : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = R.any ? grad_of<false>(R, v[j][i], at + i) : 0.f;
        }
    }
    if (likeliest)
        for (int k = 0; k < G.top; ++k) {
            const int64_t c = G.top_index[r * G.top + k];
            const float g = G.g_top[r * G.top + k];
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) v[j][i] += c == (j < NV - 1 ? (lane + L * j) * V : last.at) + i ? g : 0.f;
        }
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (j < NV - 1 || last.first < G.classes) store_from_f32<T, V>(out + (j < NV - 1 ? (lane + L * j) * V : last.at), v[j]);
}

// ---------------------------------------------------------------------------------------------
// wide rows: vector j of thread t covers the columns lo + (t + TH j) V ..
// ---------------------------------------------------------------------------------------------
// Partial results of a split row: Sums, then `top` keys.
__host__ __device__ constexpr int64_t partial_floats(int top) { return 4 + 2 * top; }

template <int TH>
__device__ __forceinline__ key_t block_max_key(key_t k, key_t* lds) {
    k = lanes_max_key<kWave>(k);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = k;
    __syncthreads();
    return lanes_max_key<TH / kWave>(lds[threadIdx.x % (TH / kWave)]);
}

template <typename T, int TH, int NV>
__global__ __launch_bounds__(TH) __attribute__((amdgpu_waves_per_eu(NV <= 4 ? 8 : 4))) void label_scores_wide(const T* __restrict__ Z, int64_t ld, int split_cols,
                                                        float* __restrict__ partial, Outputs O) {
    constexpr int V = 16 / sizeof(T);
    __shared__ key_t list[kList];
    __shared__ key_t found[kMaxTop];
    __shared__ key_t wave_key[TH / kWave];
    __shared__ Sums wave_sums[TH / kWave];
    __shared__ float part_max[kParts];
    __shared__ float bound;
    __shared__ int listed;
    const int64_t r = blockIdx.x;
    const T* row = Z + r * ld;
    const int lo = blockIdx.y * split_cols, hi = min(O.classes, lo + split_cols);
    auto place = [&](int j) { return place_of<V>(lo + (static_cast<int>(threadIdx.x) + TH * j) * V, hi); };
    Raw<T, V> raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j] = load_raw<T, V>(row + place(j).at);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const Place p = place(j);
        if (p.at < p.first) lowest(raw[j], p.first - p.at);
    }
    float my_max = -kInf;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) my_max = fmaxf(my_max, raw[j][i]);
    forget(raw);                                           // unpacked again below: 8 values a vector are too many to keep
    // part g: the columns of TH / kParts neighbouring threads; a NaN does not count for its part
    const float part = lanes_max<TH / kParts>(my_max), wave_max = lanes_max<kWave>(my_max);
    const int lane = threadIdx.x % kWave;
    if (threadIdx.x % (TH / kParts) == 0) part_max[threadIdx.x / (TH / kParts)] = part;
    if (lane == 0) wave_sums[threadIdx.x / kWave].m = wave_max;
    if (threadIdx.x < kMaxTop) found[threadIdx.x] = 0;
    if (threadIdx.x == 0) { listed = 0; bound = -kInf; }
    __syncthreads();
    Sums S{lanes_max<TH / kWave>(wave_sums[lane % (TH / kWave)].m), 0.f, 0.f};
    const float base = S.m == -kInf ? 0.f : S.m;
    if (O.entropy || gridDim.y > 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < V; ++i) take<true>(S, raw[j][i], base);
            __builtin_amdgcn_sched_barrier(0);
        }
        S.t = lanes_sum<kWave>(S.t);
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < V; ++i) take<false>(S, raw[j][i], base);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    const bool odd = S.s != S.s;                           // a NaN or +inf among this thread's values
    S.s = lanes_sum<kWave>(S.s);
    forget(raw);
    if (O.top > 0 && threadIdx.x < kParts) {
        const float mine = part_max[threadIdx.x];
        int above = 0, level = 0;
#pragma unroll 8
        for (int i = 0; i < kParts; ++i) {
            above += part_max[i] > mine ? 1 : 0;
            level += part_max[i] == mine ? 1 : 0;
        }
        if (above < O.top && above + level >= O.top) bound = mine;          // who writes, writes the same
    }
    if (lane == 0) { wave_sums[threadIdx.x / kWave].s = S.s; wave_sums[threadIdx.x / kWave].t = S.t; }
    __syncthreads();
    S.s = lanes_sum<TH / kWave>(wave_sums[lane % (TH / kWave)].s);
    S.t = lanes_sum<TH / kWave>(wave_sums[lane % (TH / kWave)].t);
    if (O.top > 0) {
        const float least = bound;
        if (!(my_max < least) || odd) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const Place p = place(j);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x = raw[j][i];
                    if (p.at + i < p.first || x < least) continue;
                    const int n = atomicAdd(&listed, 1);    // LDS; the ranks below do not depend on the order
                    if (n < kList) list[n] = key_of(order_of(x), p.at + i);
                }
            }
        }
        __syncthreads();
        const int n = listed;
        if (n <= kList) {
            for (int i = threadIdx.x; i < n; i += TH) {
                const key_t k = list[i];
                int above = 0;
                for (int j = 0; j < n; ++j) above += list[j] > k ? 1 : 0;
                if (above < O.top) found[above] = k;
            }
        } else {
            key_t before = ~static_cast<key_t>(0);
            for (int round = 0; round < O.top; ++round) {
                const unsigned limit = static_cast<unsigned>(before >> 32), limit_at = index_of(before);
                unsigned best = 0, at = 0;
                forget(raw);                               // orders of all values would not fit the registers
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const Place p = place(j);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const unsigned o = order_of(raw[j][i]), c = p.at + i;
                        // after the last one found, and better than this thread's best (whose column is lower)
                        if (p.at + i >= p.first && (o < limit || (o == limit && c > limit_at)) && o > best) { best = o; at = c; }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                const key_t k = best ? key_of(best, at) : 0;
                before = block_max_key<TH>(k, wave_key);
                if (threadIdx.x == 0) found[round] = before;
            }
        }
        __syncthreads();
    }
    if (gridDim.y > 1) {
        float* out = partial + (r * gridDim.y + blockIdx.y) * partial_floats(O.top);
        if (threadIdx.x == 0) { out[0] = S.m; out[1] = S.s; out[2] = S.t; }
        if (static_cast<int>(threadIdx.x) < O.top) reinterpret_cast<key_t*>(out + 4)[threadIdx.x] = found[threadIdx.x];
        return;
    }
    const Final F = finish(S);
    if (threadIdx.x == 0) write_scores<T>(O, row, r, F);
    if (static_cast<int>(threadIdx.x) < O.top) write_top(O, r, threadIdx.x, found[threadIdx.x], F);
}

constexpr int kMaxSplits = 64;

// Joins the splits of a row: one workgroup per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void label_scores_join(const T* __restrict__ Z, int64_t ld, int splits,
                                                              const float* __restrict__ partial, Outputs O) {
    __shared__ key_t list[kMaxSplits * kMaxTop];
    const int64_t r = blockIdx.x;
    const float* in = partial + r * splits * partial_floats(O.top);
    const int lane = threadIdx.x % kWave, n = splits * O.top;
    for (int i = threadIdx.x; i < n; i += kThreads)
        list[i] = reinterpret_cast<const key_t*>(in + (i / O.top) * partial_floats(O.top) + 4)[i % O.top];
    Sums S{-kInf, 0.f, 0.f};
    if (lane < splits) {
        const float* p = in + lane * partial_floats(O.top);
        S = Sums{p[0], p[1], p[2]};
    }
    S = lanes_join<kWave>(S);
    const Final F = finish(S);
    if (threadIdx.x == 0) write_scores<T>(O, Z + r * ld, r, F);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const key_t k = list[i];
        if (!k) continue;                                   // a split with fewer columns than `top`
        int above = 0;
        for (int j = 0; j < n; ++j) above += list[j] > k ? 1 : 0;
        if (above < O.top) write_top(O, r, above, k, F);
    }
}

constexpr int kGradVectors = 8;            // most vectors of a thread in the wide backward

template <typename T>
__global__ __launch_bounds__(kThreads) void label_grads_wide(const T* __restrict__ Z, T* __restrict__ D, int64_t ld, int64_t ldg,
                                                             int split_cols, Grads G) {
    constexpr int V = 16 / sizeof(T);
    const int64_t r = blockIdx.x;
    const T* row = Z + r * ld;
    T* out = D + r * ldg;
    const int lo = blockIdx.y * split_cols, hi = min(G.classes, lo + split_cols);
    const RowGrad R = row_grad(G, r);
    const bool h = G.g_entropy != nullptr;
    const int full = (hi - lo) / V;
    if (!R.any) {                                           // the same for the whole workgroup
        const float zeros[V] = {};
        for (int i = threadIdx.x; i < full; i += kThreads) store_from_f32<T, V>(out + lo + i * V, zeros);
        if (lo + full * V + static_cast<int>(threadIdx.x) < hi) out[lo + full * V + threadIdx.x] = static_cast<T>(0.f);
        return;
    }
#pragma unroll 2
    for (int i = threadIdx.x; i < full; i += kThreads) {
        const int c = lo + i * V;
        const Raw<T, V> raw = load_raw<T, V>(row + c);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = h ? grad_of<true>(R, raw[j], c + j) : grad_of<false>(R, raw[j], c + j);
        store_from_f32<T, V>(out + c, v);
    }
    const int c = lo + full * V + threadIdx.x;
    if (c < hi) out[c] = static_cast<T>(grad_of<true>(R, static_cast<float>(row[c]), c));
    if (!G.g_top) return;
    __syncthreads();                                        // the stores above are over: these few go on top of them
    if (static_cast<int>(threadIdx.x) < G.top) {
        const int64_t at = G.top_index[r * G.top + threadIdx.x];
        if (at >= lo && at < hi)
            out[at] = static_cast<T>(grad_of<true>(R, static_cast<float>(row[at]), static_cast<int>(at)) + G.g_top[r * G.top + threadIdx.x]);
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int kNarrowClasses = 1024;
constexpr int kWideThreads = 1024, kWideVectors = 8;

// Splits of a wide row's columns: as many as its length needs (a workgroup's registers hold kWideThreads kWideVectors
// vectors), more where rows are few, for two workgroups per CU of at least 4096 columns each.
struct Splits { int n, cols; };
Splits splits_of(int rows, int classes, int dtype) {
    const int V = 16 / element_bytes(dtype), most = kWideThreads * kWideVectors * V;
    const int need = (classes + most - 1) / most;
    const int want = std::max(need, std::min({kMaxSplits, std::max(1, 512 / std::max(rows, 1)), std::max(1, classes / 4096)}));
    const int cols = ((classes + want - 1) / want + V - 1) / V * V;
    return {(classes + cols - 1) / cols, cols};
}
constexpr int kMaxClasses = CBM_LABELS_MAX_CLASSES;
static_assert(kMaxClasses == kMaxSplits * kWideThreads * kWideVectors * 4, "fp32: the fewest columns a split holds");

#define CBM_LABEL_BY_TYPE(CALL)                          \
    if (dtype == CBM_DTYPE_F32) { CALL(float) }          \
    else if (dtype == CBM_DTYPE_BF16) { CALL(__bf16) }   \
    else { CALL(_Float16) }
// Lanes of a row and vectors of a lane: the fewest lanes that hold the row in at most 16 (two-byte types: 24) values each.
#define CBM_LABEL_BY_WIDTH(T, CALL)                                                     \
    if constexpr (sizeof(T) == 4) {                                                     \
        if (classes < 4) { CALL(T, 1, 4, 1) }                                           \
        else if (classes <= 16) { CALL(T, 4, 4, 1) }                                    \
        else if (classes <= 32) { CALL(T, 4, 4, 2) }                                    \
        else if (classes <= 48) { CALL(T, 4, 4, 3) }                                    \
        else if (classes <= 64) { CALL(T, 4, 4, 4) }                                    \
        else if (classes <= 96) { CALL(T, 4, 8, 3) }                                    \
        else if (classes <= 128) { CALL(T, 4, 8, 4) }                                   \
        else if (classes <= 192) { CALL(T, 4, 16, 3) }                                  \
        else if (classes <= 256) { CALL(T, 4, 16, 4) }                                  \
        else if (classes <= 384) { CALL(T, 4, 32, 3) }                                  \
        else if (classes <= 512) { CALL(T, 4, 32, 4) }                                  \
        else if (classes <= 768) { CALL(T, 4, 64, 3) }                                  \
        else { CALL(T, 4, 64, 4) }                                                      \
    } else {                                                                            \
        if (classes < 8) { CALL(T, 1, 8, 1) }                                           \
        else if (classes <= 32) { CALL(T, 8, 4, 1) }                                    \
        else if (classes <= 64) { CALL(T, 8, 4, 2) }                                    \
        else if (classes <= 96) { CALL(T, 8, 4, 3) }                                    \
        else if (classes <= 128) { CALL(T, 8, 8, 2) }                                   \
        else if (classes <= 192) { CALL(T, 8, 8, 3) }                                   \
        else if (classes <= 256) { CALL(T, 8, 16, 2) }                                  \
        else if (classes <= 384) { CALL(T, 8, 16, 3) }                                  \
        else if (classes <= 512) { CALL(T, 8, 32, 2) }                                  \
        else if (classes <= 768) { CALL(T, 8, 32, 3) }                                  \
        else { CALL(T, 8, 64, 2) }                                                      \
    }
// Threads of a wide row and vectors of a thread: 256 threads up to 32 KiB, 1024 up to 128 KiB.
#define CBM_LABEL_BY_SPLIT(T, CALL)                                                     \
    {                                                                                   \
        const int vectors = (s.cols * static_cast<int>(sizeof(T)) + 15) / 16;           \
        if (vectors <= 256) { CALL(T, 256, 1) }                                         \
        else if (vectors <= 512) { CALL(T, 256, 2) }                                    \
        else if (vectors <= 1024) { CALL(T, 256, 4) }                                   \
        else if (vectors <= 2048) { CALL(T, 256, 8) }                                   \
        else if (vectors <= 4096) { CALL(T, 1024, 4) }                                  \
        else { CALL(T, 1024, 8) }                                                       \
    }

int check_labels(int rows, int classes, int top, int64_t ld, int dtype) {
    if (dtype < CBM_DTYPE_F32 || dtype > CBM_DTYPE_F16) return CBM_ERR_SHAPE;
    if (rows < 0 || classes < 1 || classes > kMaxClasses || top < 0 || top > kMaxTop || top > classes || ld < classes) return CBM_ERR_SHAPE;
    return CBM_OK;
}

unsigned narrow_blocks(int rows, int L) { return static_cast<unsigned>((static_cast<int64_t>(rows) * L + kThreads - 1) / kThreads); }

// Rows of one launch: a grid holds fewer than 2^32 threads along one dimension.
int rows_at_once(int classes) { return classes <= kNarrowClasses ? 1 << 25 : 1 << 21; }      // 64 and 1024 threads a row at most

// The scores of some rows, with s (of the whole call) for wide ones.
int score_rows(const void* logits, const Outputs& O, float* workspace, int rows, int64_t ld, const Splits& s, int dtype, hipStream_t st) {
    const int classes = O.classes;
    if (classes <= kNarrowClasses) {
#define NARROW(T, V, L, NV)                                                                                                  \
    if (O.entropy || O.top > 0)                                                                                                \
        hipLaunchKernelGGL((label_scores_narrow<T, V, L, NV, true>), dim3(narrow_blocks(rows, L)), dim3(kThreads), 0, st,    \
                           static_cast<const T*>(logits), ld, rows, O);                                                      \
    else                                                                                                                     \
        hipLaunchKernelGGL((label_scores_narrow<T, V, L, NV, false>), dim3(narrow_blocks(rows, L)), dim3(kThreads), 0, st,   \
                           static_cast<const T*>(logits), ld, rows, O);
#define BY_WIDTH(T) CBM_LABEL_BY_WIDTH(T, NARROW)
        CBM_LABEL_BY_TYPE(BY_WIDTH)
#undef BY_WIDTH
#undef NARROW
        return check_launch();
    }
#define WIDE(T, TH, NV)                                                                                                     \
    hipLaunchKernelGGL((label_scores_wide<T, TH, NV>), dim3(rows, s.n), dim3(TH), 0, st, static_cast<const T*>(logits), ld, \
                       s.cols, workspace, O);
#define BY_SPLIT(T) CBM_LABEL_BY_SPLIT(T, WIDE)
#define JOIN(T) \
    hipLaunchKernelGGL(label_scores_join<T>, dim3(rows), dim3(kThreads), 0, st, static_cast<const T*>(logits), ld, s.n, workspace, O);
    CBM_LABEL_BY_TYPE(BY_SPLIT)
    if (int rc = check_launch()) return rc;
    if (s.n > 1) { CBM_LABEL_BY_TYPE(JOIN) }
#undef WIDE
#undef BY_SPLIT
#undef JOIN
    return check_launch();
}

int grad_rows(const void* logits, void* grad, const Grads& G, int rows, int64_t ld, int64_t ldg, int cols, int dtype, hipStream_t st) {
    const int classes = G.classes;
    if (classes <= kNarrowClasses) {
#define NARROW(T, V, L, NV)                                                                                             \
    hipLaunchKernelGGL((label_grads_narrow<T, V, L, NV>), dim3(narrow_blocks(rows, L)), dim3(kThreads), 0, st,          \
                       static_cast<const T*>(logits), static_cast<T*>(grad), ld, ldg, rows, G);
#define BY_WIDTH(T) CBM_LABEL_BY_WIDTH(T, NARROW)
        CBM_LABEL_BY_TYPE(BY_WIDTH)
#undef BY_WIDTH
#undef NARROW
        return check_launch();
    }
#define WIDE(T)                                                                                                               \
    hipLaunchKernelGGL(label_grads_wide<T>, dim3(rows, (classes + cols - 1) / cols), dim3(kThreads), 0, st,                   \
                       static_cast<const T*>(logits), static_cast<T*>(grad), ld, ldg, cols, G);
    CBM_LABEL_BY_TYPE(WIDE)
#undef WIDE
    return check_launch();
}

template <typename P>
P* rows_on(P* p, int64_t n) { return p ? p + n : nullptr; }

}  // namespace

extern "C" {

int64_t cbm_label_scores_workspace_floats(int32_t rows, int32_t classes, int32_t top, int32_t dtype) {
    if (check_labels(rows, classes, top, classes, dtype) || rows == 0 || classes <= kNarrowClasses) return 0;
    const Splits s = splits_of(rows, classes, dtype);
    return s.n > 1 ? static_cast<int64_t>(rows) * s.n * partial_floats(top) : 0;
}

int cbm_label_scores(const void* logits, const int64_t* labels, float* logp, float* entropy, float* top_logp, int64_t* top_index,
                     float* stats, float* workspace, int32_t rows, int32_t classes, int32_t top, int64_t ld, int64_t ignore_index,
                     int32_t dtype, void* stream) {
    if (int rc = check_labels(rows, classes, top, ld, dtype)) return rc;
    if (rows == 0) return CBM_OK;
    if (!logits || (logp && !labels) || (top > 0 && (!top_logp || !top_index))) return CBM_ERR_NULL;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Splits s = splits_of(rows, classes, dtype);
    if (classes > kNarrowClasses && s.n > 1 && !workspace) return CBM_ERR_NULL;
    const int most = rows_at_once(classes);
    for (int64_t r = 0; r < rows; r += most) {
        const Outputs O{rows_on(labels, r), rows_on(logp, r), rows_on(entropy, r), rows_on(top_logp, r * top), rows_on(top_index, r * top),
                        rows_on(stats, 2 * r), ignore_index, classes, top};
        if (int rc = score_rows(static_cast<const char*>(logits) + r * ld * element_bytes(dtype), O, workspace,
                                static_cast<int>(std::min<int64_t>(most, rows - r)), ld, s, dtype, st))
            return rc;
    }
    return CBM_OK;
}

int cbm_label_scores_backward(const void* logits, const int64_t* labels, const float* stats, const float* entropy, const int64_t* top_index,
                              const float* g_logp, const float* g_entropy, const float* g_top, void* grad, int32_t rows, int32_t classes,
                              int32_t top, int64_t ld, int64_t ldg, int64_t ignore_index, int32_t dtype, void* stream) {
    if (int rc = check_labels(rows, classes, top, ld, dtype)) return rc;
    if (ldg < classes) return CBM_ERR_SHAPE;
    if (overlap(logits, ld, grad, ldg, rows, classes, element_bytes(dtype))) return CBM_ERR_SHAPE;     // read again while it is written
    if (rows == 0) return CBM_OK;
    if (!logits || !stats || !grad || (g_logp && !labels) || (g_entropy && !entropy) || (g_top && (!top_index || top < 1)))
        return CBM_ERR_NULL;
    hipStream_t st = static_cast<hipStream_t>(stream);
    // a workgroup per share of a row: kGradVectors vectors a thread, fewer where rows are few
    const int V = 16 / element_bytes(dtype), most = rows_at_once(classes);
    int cols = kThreads * kGradVectors * V;
    while (cols > kThreads * V && static_cast<int64_t>(rows) * ((classes + cols - 1) / cols) < 1024) cols >>= 1;
    for (int64_t r = 0; r < rows; r += most) {
        const Grads G{rows_on(labels, r), rows_on(stats, 2 * r), rows_on(entropy, r), rows_on(top_index, r * top), rows_on(g_logp, r),
                      rows_on(g_entropy, r), rows_on(g_top, r * top), ignore_index, classes, top};
        if (int rc = grad_rows(static_cast<const char*>(logits) + r * ld * element_bytes(dtype),
                               static_cast<char*>(grad) + r * ldg * element_bytes(dtype), G,
                               static_cast<int>(std::min<int64_t>(most, rows - r)), ld, ldg, cols, dtype, st))
            return rc;
    }
    return CBM_OK;
}

}  // extern "C"
