// Newton-Schulz orthogonalisation on the matrix cores, and the optimiser step around it.
//
//     X = G / (|G|_F + eps);   `steps` times:  A = X X^T,  B = b A + c A A,  X = a X + B X      (short side s, long l)
//
// Per step 2 s^2 l + 2 s^3 + 2 s^2 l operations, of which the symmetric products need half: matrix cores bound it.
//
// fp32 in, fp32 out, on fp16 matrix instructions.  Every operand is kept as two fp16 planes
//     x = hi + lo / 2048,   hi = fp16(x),   lo = fp16((x - hi) 2048)
// which hold x to 2^-22 (and, hi being rounded to nearest, to 2^-24 on average); a product is hi hi + (hi lo + lo hi) / 2048
// in two fp32 accumulators, so three matrix instructions stand for one of fp32, at 16 times its rate.  Left out is
// lo lo / 2^22, below 2^-22 of the product.  The factor 2048 keeps lo out of fp16's subnormals wherever hi is out of
// them, and 2^-36 is the absolute error below that; |X| <= 1 in the beginning and its singular values stay below 1.3
// (for the usual coefficients), so nothing comes near fp16's largest value.
//
// X is kept in both orders (rows and columns along memory), so that every product reads both operands along k:
//     gram   A [s, s] = X X^T        rows of X against rows of X;  tiles on and above the diagonal, written twice
//     poly   B [s, s] = b A + c A A  rows of A against rows of A (A is symmetric);  likewise
//     apply  X [s, l] = a X + B X    rows of B against rows of X^T;  writes X, X^T, or the result
// Sides are padded to whole tiles with zeros, which all three products keep: the inner loops check no bounds.
// A list of matrices shares its launches: the tiles of all of them are one grid.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "dense_types.h"

namespace {

using namespace cbm_dense;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxItems = CBM_ORTHO_MAX_ITEMS;
constexpr int kNormBlocks = 64;            // partial sums of squares per matrix
constexpr float kLo = 2048.f;

struct Item {
    const void* src;
    void* dst;
    float* weight;
    float* momentum;
    int64_t ld_src, ld_dst, ld_weight, ld_momentum;
    int rows, cols, sp, lp;                // sp, lp: short and long side, padded
    int64_t base;                          // first half of the item's planes in the workspace
};

struct Items {
    Item it[kMaxItems];
    int n;
};

struct Update {
    float lr, mu, decay;
    int nesterov, on;
};

// Planes of an item, in halves from its base: X hi lo [sp, lp], X^T hi lo [lp, sp] twice (read and written in turns),
// A hi lo and B hi lo [sp, sp].
struct Planes { _Float16 *x, *xt[2], *a, *b; int64_t nx, na; };
__device__ __forceinline__ Planes planes_of(const Item& I, _Float16* ws) {
    Planes P;
    P.nx = static_cast<int64_t>(I.sp) * I.lp;
    P.na = static_cast<int64_t>(I.sp) * I.sp;
    P.x = ws + I.base;
    P.xt[0] = P.x + 2 * P.nx;
    P.xt[1] = P.xt[0] + 2 * P.nx;
    P.a = P.xt[1] + 2 * P.nx;
    P.b = P.a + 2 * P.na;
    return P;
}
int64_t item_halves(int sp, int lp) { return 6LL * sp * lp + 4LL * sp * sp; }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(v);
    lo = static_cast<_Float16>((v - static_cast<float>(hi)) * kLo);
}
__device__ __forceinline__ float whole(_Float16 hi, _Float16 lo) {
    return __builtin_fmaf(static_cast<float>(lo), 1.f / kLo, static_cast<float>(hi));
}

// ---------------------------------------------------------------------------------------------
// |G|_F, the momentum, and the planes of X
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float source(const Item& I, const Update& U, int r, int c) {
    const float g = static_cast<float>(static_cast<const T*>(I.src)[static_cast<int64_t>(r) * I.ld_src + c]);
    if (!U.on) return g;
    const float m = I.momentum[static_cast<int64_t>(r) * I.ld_momentum + c];
    return U.nesterov ? __builtin_fmaf(U.mu, m, g) : m;
}

// Workgroup (block of rows, item): sums of squares in 64 bits (a matrix of 1e20s has no norm in 32).
template <typename T>
__global__ __launch_bounds__(256) void ortho_norms(Items L, Update U, double* __restrict__ partial) {
    __shared__ double red[256];
    const Item& I = L.it[blockIdx.y];
    double sum = 0.0;
    for (int r = blockIdx.x; r < I.rows; r += kNormBlocks)
        for (int c = threadIdx.x; c < I.cols; c += 256) {
            if (U.on) {
                float* m = I.momentum + static_cast<int64_t>(r) * I.ld_momentum + c;
                const float g = static_cast<float>(static_cast<const T*>(I.src)[static_cast<int64_t>(r) * I.ld_src + c]);
                *m = __builtin_fmaf(U.mu, *m, g);
            }
            const double v = source<T>(I, U, r, c);
            sum += v * v;
        }
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if (static_cast<int>(threadIdx.x) < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) partial[blockIdx.y * kNormBlocks + blockIdx.x] = red[0];
}

// Tile of 64 x 64 of X in the orientation short x long: both orders of the planes, zeros in the padding.
template <typename T>
__global__ __launch_bounds__(256) void ortho_split(Items L, Update U, const double* __restrict__ partial, float eps, _Float16* __restrict__ ws) {
    __shared__ float tile[64][65];
    int b = blockIdx.x, k = 0;
    for (;; ++k) {                                          // the grid is the sum of the items' tiles
        const int t = (L.it[k].sp / 64) * (L.it[k].lp / 64);
        if (b < t) break;
        b -= t;
    }
    const Item& I = L.it[k];
    const Planes P = planes_of(I, ws);
    const int i0 = b / (I.lp / 64) * 64, j0 = b % (I.lp / 64) * 64;
    double sum = 0.0;
    for (int i = 0; i < kNormBlocks; ++i) sum += partial[k * kNormBlocks + i];
    const float inv = static_cast<float>(1.0 / (sqrt(sum) + static_cast<double>(eps)));
    const bool tall = I.rows > I.cols;
    const int tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    for (int y = ty; y < 64; y += 4) {
        // memory order: rows of G run along tx
        const int r = (tall ? j0 : i0) + y, c = (tall ? i0 : j0) + tx;
        const float v = r < I.rows && c < I.cols ? source<T>(I, U, r, c) * inv : 0.f;
        tile[tall ? tx : y][tall ? y : tx] = v;             // [short][long]
    }
    __syncthreads();
    for (int y = ty; y < 64; y += 4) {
        _Float16 hi, lo;
        split(tile[y][tx], hi, lo);
        const int64_t at = static_cast<int64_t>(i0 + y) * I.lp + j0 + tx;
        P.x[at] = hi;
        P.x[P.nx + at] = lo;
        split(tile[tx][y], hi, lo);
        const int64_t to = static_cast<int64_t>(j0 + y) * I.sp + i0 + tx;
        P.xt[0][to] = hi;
        P.xt[0][P.nx + to] = lo;
    }
}

// ---------------------------------------------------------------------------------------------
// the products
// ---------------------------------------------------------------------------------------------
enum Kind { kGram, kPoly, kApply, kResult };

struct Poly { float a, b, c; };

// One 16-byte copy per lane from global memory straight to LDS: the wavefront's 1 KiB lands in order from `to`.
__device__ __forceinline__ void copy_to_lds(const _Float16* from, _Float16* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

constexpr int kBK = 64;                    // k per stage: a tile row is 128 bytes, 8 chunks of 16

// Rows of a stage in LDS: chunk c of row r lies at place c ^ (r & 7), so that the 32 rows a wavefront reads at one c
// spread over all banks.  The copy puts lane i at place i, so lane i fetches the chunk that belongs there.
template <int ROWS, int WAVES>
__device__ __forceinline__ void copy_rows(const _Float16* __restrict__ from, int64_t ld, _Float16* to) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    static_assert(ROWS % (8 * WAVES) == 0, "whole copies");
#pragma unroll
    for (int i = 0; i < ROWS / (8 * WAVES); ++i) {
        const int r0 = (i * WAVES + wave) * 8, r = r0 + lane / 8, c = (lane % 8) ^ (r & 7);
        copy_to_lds(from + r * ld + c * 8, to + r0 * kBK);
    }
}
__device__ __forceinline__ half8 chunk_at(const _Float16* tile, int r, int c) {
    return *reinterpret_cast<const half8*>(tile + r * kBK + ((c ^ (r & 7)) * 8));
}

// Workgroup: a TM x TN tile of one product of one item; WM x WN wavefronts, each FM x FN blocks of 32 x 32.
template <typename T, Kind KIND, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(kWave* WM* WN) void ortho_product(Items L, Update U, Poly C, int turn, _Float16* __restrict__ ws) {
    constexpr int FM = TM / WM / 32, FN = TN / WN / 32, WAVES = WM * WN;
    constexpr int kStage = (TM + TN) * kBK * 2;            // halves: P hi, P lo, Q hi, Q lo
    extern __shared__ __align__(16) _Float16 lds[];
    int b = blockIdx.x, k = 0;
    for (;; ++k) {                                          // the grid is the sum of the items' tiles
        const int mt = L.it[k].sp / TM, nt = (KIND == kGram || KIND == kPoly) ? L.it[k].sp / TN : L.it[k].lp / TN;
        const int t = (KIND == kGram || KIND == kPoly) ? mt * (mt + 1) / 2 : mt * nt;
        if (b < t) break;
        b -= t;
    }
    const Item& I = L.it[k];
    const Planes P = planes_of(I, ws);
    int bi, bj;
    if constexpr (KIND == kGram || KIND == kPoly) {
        static_assert(KIND == kApply || KIND == kResult || TM == TN, "symmetric products have square tiles");
        bj = static_cast<int>((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
        while (bj * (bj + 1) / 2 > b) --bj;
        while ((bj + 1) * (bj + 2) / 2 <= b) ++bj;
        bi = b - bj * (bj + 1) / 2;                         // bi <= bj
    } else {
        const int nt = I.lp / TN;
        bi = b / nt;
        bj = b - bi * nt;
    }
    const int i0 = bi * TM, j0 = bj * TN;
    const int K = KIND == kGram ? I.lp : I.sp;
    const _Float16 *ph, *qh;
    int64_t pn, qn;                                         // from the hi plane to the lo plane
    if constexpr (KIND == kGram) { ph = qh = P.x; pn = qn = P.nx; }
    else if constexpr (KIND == kPoly) { ph = qh = P.a; pn = qn = P.na; }
    else { ph = P.b; pn = P.na; qh = P.xt[turn]; qn = P.nx; }
    ph += static_cast<int64_t>(i0) * K;
    qh += static_cast<int64_t>(j0) * K;

    auto fetch = [&](int k0, int stage) {
        _Float16* s = lds + stage * kStage;
        copy_rows<TM, WAVES>(ph + k0, K, s);
        copy_rows<TM, WAVES>(ph + pn + k0, K, s + TM * kBK);
        copy_rows<TN, WAVES>(qh + k0, K, s + 2 * TM * kBK);
        copy_rows<TN, WAVES>(qh + qn + k0, K, s + (2 * TM + TN) * kBK);
    };
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int wi = wave / WN * (TM / WM), wj = wave % WN * (TN / WN);
    const int lr = lane % 32, lk = lane / 32;
    f32x16 main_sum[FM][FN], lo_sum[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) main_sum[m][n][e] = lo_sum[m][n][e] = 0.f;
    fetch(0, 0);
    for (int k0 = 0, stage = 0; k0 < K; k0 += kBK, stage ^= 1) {
        __builtin_amdgcn_s_waitcnt(0);                      // this wavefront's copies have landed ...
        __syncthreads();                                    // ... and everyone's; the other stage is read out
        if (k0 + kBK < K) fetch(k0 + kBK, stage ^ 1);
        const _Float16* s = lds + stage * kStage;
#pragma unroll
        for (int q = 0; q < kBK / 16; ++q) {
            half8 ah[FM], al[FM], bh[FN], bl[FN];
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                ah[m] = chunk_at(s, wi + m * 32 + lr, 2 * q + lk);
                al[m] = chunk_at(s + TM * kBK, wi + m * 32 + lr, 2 * q + lk);
            }
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                bh[n] = chunk_at(s + 2 * TM * kBK, wj + n * 32 + lr, 2 * q + lk);
                bl[n] = chunk_at(s + (2 * TM + TN) * kBK, wj + n * 32 + lr, 2 * q + lk);
            }
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int n = 0; n < FN; ++n) {
                    main_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[m], bh[n], main_sum[m][n], 0, 0, 0);
                    lo_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[m], bl[n], lo_sum[m][n], 0, 0, 0);
                    lo_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[m], bh[n], lo_sum[m][n], 0, 0, 0);
                }
        }
    }
    // element e of a block: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int i = i0 + wi + m * 32 + 8 * (e / 4) + 4 * lk + e % 4, j = j0 + wj + n * 32 + lr;
                float v = __builtin_fmaf(lo_sum[m][n][e], 1.f / kLo, main_sum[m][n][e]);
                _Float16 hi, lo;
                if constexpr (KIND == kGram || KIND == kPoly) {
                    const int64_t at = static_cast<int64_t>(i) * I.sp + j, to = static_cast<int64_t>(j) * I.sp + i;
                    if constexpr (KIND == kPoly) v = __builtin_fmaf(C.b, whole(P.a[at], P.a[P.na + at]), C.c * v);
                    split(v, hi, lo);
                    _Float16* o = KIND == kGram ? P.a : P.b;
                    o[at] = hi;
                    o[P.na + at] = lo;
                    if (bi != bj) { o[to] = hi; o[P.na + to] = lo; }
                } else {
                    const int64_t at = static_cast<int64_t>(i) * I.lp + j, to = static_cast<int64_t>(j) * I.sp + i;
                    v = __builtin_fmaf(C.a, whole(P.x[at], P.x[P.nx + at]), v);
                    if constexpr (KIND == kApply) {
                        split(v, hi, lo);
                        P.x[at] = hi;
                        P.x[P.nx + at] = lo;
                        P.xt[turn ^ 1][to] = hi;
                        P.xt[turn ^ 1][P.nx + to] = lo;
                    } else {
                        const bool tall = I.rows > I.cols;
                        const int r = tall ? j : i, c = tall ? i : j;
                        if (r < I.rows && c < I.cols) {
                            if (U.on) {
                                float* w = I.weight + static_cast<int64_t>(r) * I.ld_weight + c;
                                const float scale = sqrtf(fmaxf(1.f, static_cast<float>(I.rows) / static_cast<float>(I.cols)));
                                *w = *w * (1.f - U.lr * U.decay) - (U.lr * scale) * v;
                            } else {
                                static_cast<T*>(I.dst)[static_cast<int64_t>(r) * I.ld_dst + c] = static_cast<T>(v);
                            }
                        }
                    }
                }
            }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int kTile = 64;
constexpr size_t kLds = static_cast<size_t>(2 * kTile) * kBK * 2 * sizeof(_Float16) * 2;

int padded(int v) { return (v + kTile - 1) / kTile * kTile; }

// Sides of the items of one turn; halves of workspace they need.
int64_t lay_out(const cbm_ortho_item* items, int n, Items& L) {
    int64_t halves = 0;
    L.n = 0;
    for (int i = 0; i < n; ++i) {
        const cbm_ortho_item& s = items[i];
        if (s.rows == 0 || s.cols == 0) continue;
        Item& d = L.it[L.n++];
        d.src = s.src; d.dst = s.dst; d.weight = s.weight; d.momentum = s.momentum;
        d.ld_src = s.ld_src; d.ld_dst = s.ld_dst; d.ld_weight = s.ld_weight; d.ld_momentum = s.ld_momentum;
        d.rows = s.rows; d.cols = s.cols;
        d.sp = padded(std::min(s.rows, s.cols));
        d.lp = padded(std::max(s.rows, s.cols));
        d.base = halves;
        halves += item_halves(d.sp, d.lp);
    }
    return halves;
}

constexpr int64_t kNormBytes = static_cast<int64_t>(kMaxItems) * kNormBlocks * sizeof(double);

template <typename T>
int run_turn(const cbm_ortho_item* items, int n, const Update& U, int steps, const Poly& C, float eps, void* workspace, hipStream_t st) {
    Items L;
    lay_out(items, n, L);
    if (L.n == 0) return CBM_OK;
    double* partial = static_cast<double*>(workspace);
    _Float16* ws = reinterpret_cast<_Float16*>(static_cast<char*>(workspace) + kNormBytes);
    int64_t square = 0, wide = 0, tiles64 = 0;
    for (int i = 0; i < L.n; ++i) {
        const int64_t s = L.it[i].sp / kTile, l = L.it[i].lp / kTile;
        square += s * (s + 1) / 2;
        wide += s * l;
        tiles64 += static_cast<int64_t>(L.it[i].sp / 64) * (L.it[i].lp / 64);
    }
    if (wide > (1LL << 30) || square > (1LL << 30)) return CBM_ERR_SHAPE;
    hipLaunchKernelGGL(ortho_norms<T>, dim3(kNormBlocks, L.n), dim3(256), 0, st, L, U, partial);
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(ortho_split<T>, dim3(static_cast<unsigned>(tiles64)), dim3(256), 0, st, L, U, partial, eps, ws);
    if (int rc = check_launch()) return rc;
    for (int t = 0; t < steps; ++t) {
        hipLaunchKernelGGL((ortho_product<T, kGram, kTile, kTile, 2, 2>), dim3(static_cast<unsigned>(square)), dim3(256), kLds, st, L, U, C, t & 1, ws);
        if (int rc = check_launch()) return rc;
        hipLaunchKernelGGL((ortho_product<T, kPoly, kTile, kTile, 2, 2>), dim3(static_cast<unsigned>(square)), dim3(256), kLds, st, L, U, C, t & 1, ws);
        if (int rc = check_launch()) return rc;
        if (t + 1 < steps)
            hipLaunchKernelGGL((ortho_product<T, kApply, kTile, kTile, 2, 2>), dim3(static_cast<unsigned>(wide)), dim3(256), kLds, st, L, U, C, t & 1, ws);
        else
            hipLaunchKernelGGL((ortho_product<T, kResult, kTile, kTile, 2, 2>), dim3(static_cast<unsigned>(wide)), dim3(256), kLds, st, L, U, C, t & 1, ws);
        if (int rc = check_launch()) return rc;
    }
    return CBM_OK;
}

constexpr int kMaxSide = 1 << 20;

int check_items(const cbm_ortho_item* items, int n, bool update) {
    if (n < 0) return CBM_ERR_SHAPE;
    if (n > 0 && !items) return CBM_ERR_NULL;
    for (int i = 0; i < n; ++i) {
        const cbm_ortho_item& s = items[i];
        if (s.rows < 0 || s.cols < 0 || s.rows > kMaxSide || s.cols > kMaxSide) return CBM_ERR_SHAPE;
        if (s.rows == 0 || s.cols == 0) continue;
        if (!s.src || (update ? !s.weight || !s.momentum : !s.dst)) return CBM_ERR_NULL;
        if (s.ld_src < s.cols || (update ? s.ld_weight < s.cols || s.ld_momentum < s.cols : s.ld_dst < s.cols)) return CBM_ERR_SHAPE;
    }
    return CBM_OK;
}

template <typename T>
int run_all(const cbm_ortho_item* items, int n, const Update& U, int steps, const Poly& C, float eps, void* workspace, hipStream_t st) {
    for (int i = 0; i < n; i += kMaxItems)
        if (int rc = run_turn<T>(items + i, std::min(kMaxItems, n - i), U, steps, C, eps, workspace, st)) return rc;
    return CBM_OK;
}

}  // namespace

extern "C" {

int64_t cbm_ortho_workspace_bytes(const cbm_ortho_item* items, int32_t n) {
    if (!items || n <= 0) return 0;
    int64_t most = 0;
    for (int i = 0; i < n; i += kMaxItems) {
        Items L;
        most = std::max(most, lay_out(items + i, std::min(kMaxItems, n - i), L));
    }
    return most ? kNormBytes + most * static_cast<int64_t>(sizeof(_Float16)) : 0;
}

int cbm_orthogonalise(const cbm_ortho_item* items, int32_t n, int32_t steps, float a, float b, float c, float eps, int32_t dtype,
                      void* workspace, void* stream) {
    if (int rc = check_items(items, n, false)) return rc;
    if (steps < 1 || !(eps >= 0.f) || dtype < CBM_DTYPE_F32 || dtype > CBM_DTYPE_F16) return CBM_ERR_SHAPE;
    if (n > 0 && !workspace && cbm_ortho_workspace_bytes(items, n) > 0) return CBM_ERR_NULL;
    const Update U{0.f, 0.f, 0.f, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == CBM_DTYPE_F32) return run_all<float>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
    if (dtype == CBM_DTYPE_BF16) return run_all<__bf16>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
    return run_all<_Float16>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
}

int cbm_muon_step(const cbm_ortho_item* items, int32_t n, float lr, float mu, float decay, int32_t nesterov, int32_t steps, float a,
                  float b, float c, float eps, void* workspace, void* stream) {
    if (int rc = check_items(items, n, true)) return rc;
    if (steps < 1 || !(eps >= 0.f)) return CBM_ERR_SHAPE;
    if (n > 0 && !workspace && cbm_ortho_workspace_bytes(items, n) > 0) return CBM_ERR_NULL;
    const Update U{lr, mu, decay, nesterov, 1};
    return run_all<float>(items, n, U, steps, Poly{a, b, c}, eps, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
