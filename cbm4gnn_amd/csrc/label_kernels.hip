// Scores of labels: log probability of the given class, entropy of the distribution and the likeliest classes of
// every row of logits [rows, classes], and the gradient of the logits.
//
//     m = max z,  S = sum exp(z - m),  log p_j = (z_j - m) - log S,  H = log S - sum exp(z - m) (z - m) / S
//     dz_j = gl [j = label] + sum_i gt_i [j = top_i] - p_j (gl + sum_i gt_i + gH (log p_j + H))
//
// m and log S are kept apart (not summed into one float), so logits far from zero cost no digits.
//
// One pass over the logits serves all three: running maximum, sum and weighted sum.  Reading the logits bounds the
// forward, reading them and writing the gradient the backward.
//   narrow   up to 1024 classes: L lanes hold a row in registers (at most 16 values each), 64 / L rows per wavefront;
//   wide     a workgroup per row, 16-byte loads; with few rows the columns are split over workgroups whose partial
//            results a second launch joins.
// Likeliest classes order by (value, lowest index): value and index make ONE 64-bit key, so no two are equal and the
// answer does not depend on who looks at what.  Narrow rows take `top` maxima out of registers.  Wide rows first
// find a bound that at least `top` keys reach (the `top`-th largest of 128 maxima of disjoint parts of the row),
// then collect the few keys above it into LDS and rank them by counting; a row that crowds more than the list holds
// into few parts takes one more pass per class instead.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense_types.h"

namespace {

using namespace cbm_dense;
using key_t = unsigned long long;

constexpr int kMaxTop = CBM_LABELS_MAX_TOP;
constexpr int kNarrowThreads = 256;
constexpr int kWideThreads = 1024;
constexpr int kParts = 128;                // disjoint parts of a wide row whose maxima bound its likeliest classes
constexpr int kList = 2048;                // candidates a wide row keeps
constexpr float kInf = __builtin_inff();

// Order of values as unsigned numbers: -inf lowest, NaN highest, -0 and +0 equal.  0 stands for no value.
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __float_as_uint(v + 0.f);
    if (v != v) return 0xffc00000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ key_t key_of(unsigned order, unsigned index) {
    return (static_cast<key_t>(order) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned index_of(key_t k) { return 0xffffffffu - static_cast<unsigned>(k); }

__device__ __forceinline__ key_t shfl_xor_key(key_t k, int o) {
    const unsigned lo = __shfl_xor(static_cast<unsigned>(k), o), hi = __shfl_xor(static_cast<unsigned>(k >> 32), o);
    return (static_cast<key_t>(hi) << 32) | lo;
}

// Running softmax sums: m the maximum, s = sum exp(z - m), t = sum exp(z - m) (z - m).
struct Sums { float m, s, t; };

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    // a part of -inf alone has s = 0 (or NaN, which stays) and moves by factor 0
    const float fa = a.m == -kInf ? 0.f : __expf(a.m - m), fb = b.m == -kInf ? 0.f : __expf(b.m - m);
    const float ta = fa == 0.f ? 0.f : (a.t + a.s * (a.m - m)) * fa, tb = fb == 0.f ? 0.f : (b.t + b.s * (b.m - m)) * fb;
    return {m, a.s * fa + b.s * fb, ta + tb};
}

// Takes one value into sums whose maximum already covers it; base = m, or 0 while m is -inf.
__device__ __forceinline__ void take(Sums& S, float v, float base) {
    const float d = v - base, e = __expf(d);
    S.s += e;
    S.t += e > 0.f ? e * d : 0.f;                          // exp(-inf) (-inf) counts nothing
}

template <int L>
__device__ __forceinline__ Sums join_lanes(Sums S) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) S = join(S, Sums{__shfl_xor(S.m, o), __shfl_xor(S.s, o), __shfl_xor(S.t, o)});
    return S;
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
    if (O.stats) { O.stats[2 * r] = F.m; O.stats[2 * r + 1] = F.log_s; }
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

// ---------------------------------------------------------------------------------------------
// narrow rows
// ---------------------------------------------------------------------------------------------
template <typename T, int L, int NV>
__global__ __launch_bounds__(kNarrowThreads) void label_scores_narrow(const T* __restrict__ Z, int64_t ld, int rows, Outputs O) {
    const int lane = threadIdx.x % L;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / L) + threadIdx.x / L;
    const T* row = Z + min(r, static_cast<int64_t>(rows - 1)) * ld;
    float v[NV];
    Sums S{-kInf, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = lane + L * j;
        v[j] = c < O.classes ? static_cast<float>(row[c]) : -kInf;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) S.m = fmaxf(S.m, v[j]);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) S.m = fmaxf(S.m, __shfl_xor(S.m, o));
    const float base = S.m == -kInf ? 0.f : S.m;
#pragma unroll
    for (int j = 0; j < NV; ++j) take(S, v[j], base);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        S.s += __shfl_xor(S.s, o);
        S.t += __shfl_xor(S.t, o);
    }
    const Final F = finish(S);
    const bool mine = r < rows && lane == 0;
    if (mine) write_scores<T>(O, row, r, F);
    unsigned taken = 0;
    for (int i = 0; i < O.top; ++i) {
        unsigned best = 0, at = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const unsigned c = lane + L * j;
            const unsigned o = c < static_cast<unsigned>(O.classes) && !(taken >> j & 1u) ? order_of(v[j]) : 0u;
            if (o > best) { best = o; at = c; }
        }
        key_t k = best ? key_of(best, at) : 0;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            const key_t other = shfl_xor_key(k, o);
            k = other > k ? other : k;
        }
        if (best && index_of(k) == at) taken |= 1u << ((at - lane) / L);
        if (mine) write_top(O, r, i, k, F);
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

// What a row's gradient needs: dz_j = -p_j (all + gh (log p_j + h)) + gl [j = label] (+ the likeliest classes')
// A row of -inf alone has no gradient.
struct RowGrad { float m, log_s, h, gl, gh, all; int label; bool any; };
__device__ __forceinline__ RowGrad row_grad(const Grads& G, int64_t r) {
    RowGrad R{G.stats[2 * r], G.stats[2 * r + 1], 0.f, 0.f, 0.f, 0.f, -1, true};
    if (R.log_s == kInf) {
        R.any = false;
        return R;
    }
    if (G.g_entropy) { R.gh = G.g_entropy[r]; R.h = G.entropy[r]; }
    if (G.g_logp) {
        const int64_t y = G.labels[r];
        if (y != G.ignore_index) {
            const bool in = y >= 0 && y < G.classes;
            R.gl = in ? G.g_logp[r] : __builtin_nanf("");
            R.label = in ? static_cast<int>(y) : -1;
        }
    }
    R.all = R.gl;
    if (G.g_top)
        for (int i = 0; i < G.top; ++i) R.all += G.g_top[r * G.top + i];
    return R;
}
__device__ __forceinline__ float grad_of(const RowGrad& R, float z, int c) {
    const float lp = (z - R.m) - R.log_s, p = __expf(lp);
    // p = 0: nothing, also where log p is -inf; a NaN goes through
    const float inner = p == 0.f ? R.all : __builtin_fmaf(R.gh, lp + R.h, R.all);
    return (c == R.label ? R.gl : 0.f) - p * inner;
}

template <typename T, int L, int NV>
__global__ __launch_bounds__(kNarrowThreads) void label_grads_narrow(const T* __restrict__ Z, T* __restrict__ D, int64_t ld, int64_t ldg,
                                                                     int rows, Grads G) {
    const int lane = threadIdx.x % L;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / L) + threadIdx.x / L;
    if (r >= rows) return;
    const T* row = Z + r * ld;
    float v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = lane + L * j;
        v[j] = c < G.classes ? static_cast<float>(row[c]) : 0.f;
    }
    const RowGrad R = row_grad(G, r);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = grad_of(R, v[j], lane + L * j);
    if (G.g_top && R.any)
        for (int i = 0; i < G.top; ++i) {
            const int64_t at = G.top_index[r * G.top + i];
            const float g = G.g_top[r * G.top + i];
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] += at == lane + L * j ? g : 0.f;
        }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = lane + L * j;
        if (c < G.classes) D[r * ldg + c] = static_cast<T>(v[j]);
    }
}

// ---------------------------------------------------------------------------------------------
// wide rows
// ---------------------------------------------------------------------------------------------
// Partial results of a split row: Sums, then `top` keys.
__device__ __forceinline__ int64_t partial_floats(int top) { return 4 + 2 * top; }

// fn(value, column) for the columns lo, lo + 1, ... < hi of this thread, ascending; first(values) once per vector
template <typename T, typename First, typename Fn>
__device__ __forceinline__ void for_columns(const T* __restrict__ row, int lo, int hi, First first, Fn fn) {
    constexpr int V = 16 / sizeof(T);
    const int full = (hi - lo) / V;
    for (int i = threadIdx.x; i < full; i += kWideThreads) {
        float v[V];
        load_as_f32<T, V>(row + lo + static_cast<int64_t>(i) * V, v);
        first(v);
#pragma unroll
        for (int j = 0; j < V; ++j) fn(v[j], lo + i * V + j);
    }
    const int c = lo + full * V + threadIdx.x;
    if (c < hi) {
        float v[1] = {static_cast<float>(row[c])};
        first(v);
        fn(v[0], c);
    }
}

__device__ __forceinline__ key_t block_max_key(key_t k, key_t* lds) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) {
        const key_t other = shfl_xor_key(k, o);
        k = other > k ? other : k;
    }
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = k;
    __syncthreads();
    for (int w = 0; w < kWideThreads / kWave; ++w) k = lds[w] > k ? lds[w] : k;
    return k;
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void label_scores_wide(const T* __restrict__ Z, int64_t ld, int split_cols,
                                                                  float* __restrict__ partial, Outputs O) {
    __shared__ key_t list[kList];
    __shared__ key_t found[kMaxTop];
    __shared__ key_t wave_key[kWideThreads / kWave];
    __shared__ Sums wave_sums[kWideThreads / kWave];
    __shared__ key_t bound;
    __shared__ int listed;
    const int64_t r = blockIdx.x;
    const T* row = Z + r * ld;
    const int lo = blockIdx.y * split_cols, hi = min(O.classes, lo + split_cols);
    Sums S{-kInf, 0.f, 0.f};
    float base = 0.f;
    unsigned best = 0, at = 0;
    const bool top = O.top > 0;
    for_columns<T>(
        row, lo, hi,
        [&](auto& v) {
            float vm = S.m;
            for (float x : v) vm = fmaxf(vm, x);
            if (vm > S.m) {
                S = join(S, Sums{vm, 0.f, 0.f});
                base = vm;
            }
        },
        [&](float x, int c) {
            take(S, x, base);
            if (top) {
                const unsigned o = order_of(x);
                if (o > best) { best = o; at = c; }
            }
        });
    S = join_lanes<kWave>(S);
    if (threadIdx.x % kWave == 0) wave_sums[threadIdx.x / kWave] = S;
    if (threadIdx.x < kMaxTop) found[threadIdx.x] = 0;
    if (threadIdx.x == 0) { listed = 0; bound = 1; }
    if (top) list[threadIdx.x] = best ? key_of(best, at) : 0;
    __syncthreads();
    S = wave_sums[0];
    for (int w = 1; w < kWideThreads / kWave; ++w) S = join(S, wave_sums[w]);
    if (top) {
        // part g: the columns of the threads g, g + kParts, ...
        key_t part = 0;
        if (threadIdx.x < kParts)
            for (int i = threadIdx.x; i < kWideThreads; i += kParts) part = list[i] > part ? list[i] : part;
        __syncthreads();
        if (threadIdx.x < kParts) list[threadIdx.x] = part;
        __syncthreads();
        if (threadIdx.x < kParts) {
            int above = 0;
            for (int i = 0; i < kParts; ++i) above += list[i] > part ? 1 : 0;
            if (above == O.top - 1 && part) bound = part;   // keys differ: one thread at most
        }
        __syncthreads();
        const key_t least = bound;
        const unsigned least_order = static_cast<unsigned>(least >> 32);
        for_columns<T>(row, lo, hi, [](auto&) {}, [&](float x, int c) {
            const unsigned o = order_of(x);
            if (o < least_order) return;
            const key_t k = key_of(o, c);
            if (k < least) return;
            const int n = atomicAdd(&listed, 1);            // LDS; the ranks below do not depend on the order
            if (n < kList) list[n] = k;
        });
        __syncthreads();
        const int n = listed;
        if (n <= kList) {
            for (int i = threadIdx.x; i < n; i += kWideThreads) {
                const key_t k = list[i];
                int above = 0;
                for (int j = 0; j < n; ++j) above += list[j] > k ? 1 : 0;
                if (above < O.top) found[above] = k;
            }
        } else {
            key_t last = ~static_cast<key_t>(0);
            for (int i = 0; i < O.top; ++i) {
                key_t k = 0;
                for_columns<T>(row, lo, hi, [](auto&) {}, [&](float x, int c) {
                    const key_t q = key_of(order_of(x), c);
                    if (q < last && q > k) k = q;
                });
                last = block_max_key(k, wave_key);
                if (threadIdx.x == 0) found[i] = last;
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
__global__ __launch_bounds__(256) void label_scores_join(const T* __restrict__ Z, int64_t ld, int splits, const float* __restrict__ partial,
                                                         Outputs O) {
    __shared__ key_t list[kMaxSplits * kMaxTop];
    const int64_t r = blockIdx.x;
    const float* in = partial + r * splits * partial_floats(O.top);
    const int lane = threadIdx.x % kWave;
    Sums S{-kInf, 0.f, 0.f};
    if (lane < splits) {
        const float* p = in + lane * partial_floats(O.top);
        S = Sums{p[0], p[1], p[2]};
    }
    S = join_lanes<kWave>(S);
    const Final F = finish(S);
    if (threadIdx.x == 0) write_scores<T>(O, Z + r * ld, r, F);
    const int n = splits * O.top;
    for (int i = threadIdx.x; i < n; i += 256)
        list[i] = reinterpret_cast<const key_t*>(in + (i / O.top) * partial_floats(O.top) + 4)[i % O.top];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const key_t k = list[i];
        if (!k) continue;                                   // a split with fewer columns than `top`
        int above = 0;
        for (int j = 0; j < n; ++j) above += list[j] > k ? 1 : 0;
        if (above < O.top) write_top(O, r, above, k, F);
    }
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void label_grads_wide(const T* __restrict__ Z, T* __restrict__ D, int64_t ld, int64_t ldg,
                                                                 int split_cols, Grads G) {
    constexpr int V = 16 / sizeof(T);
    const int64_t r = blockIdx.x;
    const T* row = Z + r * ld;
    T* out = D + r * ldg;
    const int lo = blockIdx.y * split_cols, hi = min(G.classes, lo + split_cols);
    const RowGrad R = row_grad(G, r);
    const int full = (hi - lo) / V;
    for (int i = threadIdx.x; i < full; i += kWideThreads) {
        const int c = lo + i * V;
        float v[V];
        load_as_f32<T, V>(row + c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = grad_of(R, v[j], c + j);
        store_from_f32<T, V>(out + c, v);
    }
    const int c = lo + full * V + threadIdx.x;
    if (c < hi) out[c] = static_cast<T>(grad_of(R, static_cast<float>(row[c]), c));
    if (!G.g_top || !R.any) return;                         // the same for the whole workgroup
    __syncthreads();                                        // the stores above are over: these few go on top of them
    if (static_cast<int>(threadIdx.x) < G.top) {
        const int64_t at = G.top_index[r * G.top + threadIdx.x];
        if (at >= lo && at < hi)
            out[at] = static_cast<T>(grad_of(R, static_cast<float>(row[at]), static_cast<int>(at)) + G.g_top[r * G.top + threadIdx.x]);
    }
}

// Splits of a wide row's columns: enough workgroups for two per CU, at least 4096 columns each.
struct Splits { int n, cols; };
Splits splits_of(int rows, int classes) {
    const int want = std::min({kMaxSplits, std::max(1, 512 / std::max(rows, 1)), std::max(1, classes / 4096)});
    const int cols = ((classes + want - 1) / want + 7) / 8 * 8;
    return {(classes + cols - 1) / cols, cols};
}

constexpr int kNarrowClasses = 1024;

#define CBM_LABEL_BY_TYPE(CALL)                          \
    if (dtype == CBM_DTYPE_F32) { CALL(float) }          \
    else if (dtype == CBM_DTYPE_BF16) { CALL(__bf16) }   \
    else { CALL(_Float16) }
// Lanes of a row: the fewest that leave each at most 8 values (16 in a whole wavefront).
#define CBM_LABEL_BY_WIDTH(T, CALL)                      \
    if (classes <= 32) { CALL(T, 4, 8) }                 \
    else if (classes <= 64) { CALL(T, 8, 8) }            \
    else if (classes <= 128) { CALL(T, 16, 8) }          \
    else if (classes <= 256) { CALL(T, 32, 8) }          \
    else if (classes <= 512) { CALL(T, 64, 8) }          \
    else { CALL(T, 64, 16) }

int check_labels(int rows, int classes, int top, int64_t ld, int dtype) {
    if (dtype < CBM_DTYPE_F32 || dtype > CBM_DTYPE_F16) return CBM_ERR_SHAPE;
    if (rows < 0 || classes < 1 || classes > (1 << 30) || top < 0 || top > kMaxTop || top > classes || ld < classes) return CBM_ERR_SHAPE;
    return CBM_OK;
}

}  // namespace

extern "C" {

int64_t cbm_label_scores_workspace_floats(int32_t rows, int32_t classes, int32_t top) {
    if (rows <= 0 || classes <= kNarrowClasses || top < 0 || top > kMaxTop) return 0;
    const Splits s = splits_of(rows, classes);
    return s.n > 1 ? static_cast<int64_t>(rows) * s.n * (4 + 2 * top) : 0;
}

int cbm_label_scores(const void* logits, const int64_t* labels, float* logp, float* entropy, float* top_logp, int64_t* top_index,
                     float* stats, float* workspace, int32_t rows, int32_t classes, int32_t top, int64_t ld, int64_t ignore_index,
                     int32_t dtype, void* stream) {
    if (int rc = check_labels(rows, classes, top, ld, dtype)) return rc;
    if (rows == 0) return CBM_OK;
    if (!logits || (logp && !labels) || (top > 0 && (!top_logp || !top_index))) return CBM_ERR_NULL;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Outputs O{labels, logp, entropy, top_logp, top_index, stats, ignore_index, classes, top};
    if (classes <= kNarrowClasses) {
#define NARROW(T, L, NV)                                                                                                      \
    hipLaunchKernelGGL((label_scores_narrow<T, L, NV>), dim3((unsigned)((static_cast<int64_t>(rows) * L + kNarrowThreads - 1) / kNarrowThreads)), \
                       dim3(kNarrowThreads), 0, st, static_cast<const T*>(logits), ld, rows, O);
#define BY_WIDTH(T) CBM_LABEL_BY_WIDTH(T, NARROW)
        CBM_LABEL_BY_TYPE(BY_WIDTH)
#undef BY_WIDTH
#undef NARROW
        return check_launch();
    }
    const Splits s = splits_of(rows, classes);
    if (s.n > 1 && !workspace) return CBM_ERR_NULL;
#define WIDE(T)                                                                                                             \
    hipLaunchKernelGGL(label_scores_wide<T>, dim3(rows, s.n), dim3(kWideThreads), 0, st, static_cast<const T*>(logits), ld, \
                       s.cols, workspace, O);
#define JOIN(T) \
    hipLaunchKernelGGL(label_scores_join<T>, dim3(rows), dim3(256), 0, st, static_cast<const T*>(logits), ld, s.n, workspace, O);
    CBM_LABEL_BY_TYPE(WIDE)
    if (int rc = check_launch()) return rc;
    if (s.n > 1) { CBM_LABEL_BY_TYPE(JOIN) }
#undef WIDE
#undef JOIN
    return check_launch();
}

int cbm_label_scores_backward(const void* logits, const int64_t* labels, const float* stats, const float* entropy, const int64_t* top_index,
                              const float* g_logp, const float* g_entropy, const float* g_top, void* grad, int32_t rows, int32_t classes,
                              int32_t top, int64_t ld, int64_t ldg, int64_t ignore_index, int32_t dtype, void* stream) {
    if (int rc = check_labels(rows, classes, top, ld, dtype)) return rc;
    if (ldg < classes) return CBM_ERR_SHAPE;
    if (rows == 0) return CBM_OK;
    if (!logits || !stats || !grad || (g_logp && !labels) || (g_entropy && !entropy) || (g_top && (!top_index || top < 1)))
        return CBM_ERR_NULL;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Grads G{labels, stats, entropy, top_index, g_logp, g_entropy, g_top, ignore_index, classes, top};
    if (classes <= kNarrowClasses) {
#define NARROW(T, L, NV)                                                                                                     \
    hipLaunchKernelGGL((label_grads_narrow<T, L, NV>), dim3((unsigned)((static_cast<int64_t>(rows) * L + kNarrowThreads - 1) / kNarrowThreads)), \
                       dim3(kNarrowThreads), 0, st, static_cast<const T*>(logits), static_cast<T*>(grad), ld, ldg, rows, G);
#define BY_WIDTH(T) CBM_LABEL_BY_WIDTH(T, NARROW)
        CBM_LABEL_BY_TYPE(BY_WIDTH)
#undef BY_WIDTH
#undef NARROW
        return check_launch();
    }
    const Splits s = splits_of(rows, classes);
#define WIDE(T)                                                                                                            \
    hipLaunchKernelGGL(label_grads_wide<T>, dim3(rows, s.n), dim3(kWideThreads), 0, st, static_cast<const T*>(logits),     \
                       static_cast<T*>(grad), ld, ldg, s.cols, G);
    CBM_LABEL_BY_TYPE(WIDE)
#undef WIDE
    return check_launch();
}

}  // extern "C"
