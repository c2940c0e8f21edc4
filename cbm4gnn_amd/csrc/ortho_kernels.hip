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
//
// Measured (one MI355X, kernel times; rates count the fp16 products done):
//   2 048 x 2 048 fp32, tiles of 128: gram 48 us (0.57 PFLOP/s, 136 tiles for 256 CUs), poly 49, apply 59 (0.87), planes and
//   norm 10 + 7.  Without their epilogues 43, 41 and 45; the rest of a tile is 1.7 times its matrix instructions alone and
//   1.2 times its copies alone, which reach a CU at 62 GB/s.
//   8 x 512 x 1 024 bf16: gram 17, poly 11 (tiles of 64), apply 24 (128), planes and norm 16 + 5
//   333 x 1 001 fp32, tiles of 32: gram 11, poly 4.7, apply 11.5, planes and norm 6.5 + 3.5
//   128 x 602 and 41 x 128 together: gram 6.6, poly 4.3, apply 5.7, planes and norm 5.7 + 4.6: a launch after another, which
//   neither more wavefronts, loads further ahead, other strides nor fewer loads on the way to a tile make shorter
//
// Three shapes of the same product, chosen launch by launch by how many tiles there are and what padding they bring (see choose()):
//     tiles of 128 or 64   operands through LDS, copied there directly (no registers in between) one stage ahead;
//     tiles of 32          for small matrices, where a product is one latency after another: eight wavefronts share a tile
//                          and split k, operands straight to registers, partial sums joined in LDS.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <functional>
#include <memory>
#include <new>

#include "dense_types.h"

namespace {

using namespace cbm_dense;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxItems = CBM_ORTHO_MAX_ITEMS;
constexpr int kNormBlocks = 256;           // partial sums of squares per matrix, at most
constexpr float kLo = 2048.f;

struct Item {
    const void* src;
    void* dst;
    float* weight;
    float* momentum;
    int64_t ld_src, ld_dst, ld_weight, ld_momentum;
    int rows, cols, sp, lp;                // sp, lp: short and long side, padded to tiles
    int ls, ll;                            // halves from row to row of planes whose rows run along the short / long side
    int norm_blocks;
    int64_t base;                          // first half of the item's planes in the workspace
};

// The list a turn works on.  A kernel's arguments lie in host memory, and every workgroup would fetch its item from there:
// the first launch writes the list into the workspace, the others read it there.
enum Grid { kSplitGrid, kSquareGrid, kWideGrid, kGrids };
struct Items {
    Item it[kMaxItems];
    int ends[kGrids][kMaxItems];           // tiles up to and with each item, in each of the grids
    int n;
};

// The item that workgroup b of a grid works on; b becomes its place in the item.  One load, whatever the number of items
// (walking along the list, a load after another, cost 1 us per item).
__device__ __forceinline__ int item_of(const Items& L, Grid grid, int& b) {
    const int end = L.ends[grid][min(static_cast<int>(threadIdx.x) % kWave, kMaxItems - 1)];
    const int k = min(__popcll(__ballot(end <= b)), kMaxItems - 1);
    if (k > 0) b -= __builtin_amdgcn_readlane(end, k - 1);
    return k;
}

struct Update {
    float lr, mu, decay;
    int nesterov, on;
};

// Planes of an item, in halves from its base: X hi lo [sp, ll], X^T hi lo [lp, ls] twice (read and written in turns),
// A hi lo and B hi lo [sp, ls].
struct Planes { _Float16 *x, *xt[2], *a, *b; int64_t nx, nt, na; };   // n: from the hi to the lo plane
__device__ __forceinline__ Planes planes_of(const Item& I, _Float16* ws) {
    Planes P;
    P.nx = static_cast<int64_t>(I.sp) * I.ll;
    P.nt = static_cast<int64_t>(I.lp) * I.ls;
    P.na = static_cast<int64_t>(I.sp) * I.ls;
    P.x = ws + I.base;
    P.xt[0] = P.x + 2 * P.nx;
    P.xt[1] = P.xt[0] + 2 * P.nt;
    P.a = P.xt[1] + 2 * P.nt;
    P.b = P.a + 2 * P.na;
    return P;
}
int64_t item_halves(const Item& I) { return 2LL * I.sp * I.ll + 4LL * I.lp * I.ls + 4LL * I.sp * I.ls; }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(v);
    lo = static_cast<_Float16>((v - static_cast<float>(hi)) * kLo);
}
__device__ __forceinline__ void split4(float v, half4& hi, half4& lo, int e) {
    _Float16 a, b;
    split(v, a, b);
    hi[e] = a;
    lo[e] = b;
}
// Stores of planes go through the XCD's L2 at once (agent scope): the next launch reads them from the other XCDs, and what is
// dirty in the L2 when a launch ends is written back then, with nothing left to overlap it.  8 x 512 x 1024, the whole call:
// 287 us for 310; stores that also skip the last-level cache (non-temporal): 327.
__device__ __forceinline__ void put(_Float16* to, half4 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float whole(_Float16 hi, _Float16 lo) {
    return __builtin_fmaf(static_cast<float>(lo), 1.f / kLo, static_cast<float>(hi));
}

// ---------------------------------------------------------------------------------------------
// |G|_F, the momentum, and the planes of X
// ---------------------------------------------------------------------------------------------
// Workgroup (block of rows, item): sums of squares in 64 bits (a matrix of 1e20s has no norm in 32).  Wavefront w takes
// the rows w of every four, kFetch strides of 64 columns in flight: places outside read the matrix's last element and
// count as nothing, for a branch around each load made the loads wait for one another.
constexpr int kFetch = 8;
template <typename T>
__global__ __launch_bounds__(256) void ortho_norms(Items L, Update U, Items* __restrict__ list, double* __restrict__ partial) {
    __shared__ double red[4];
    const Item I = L.it[blockIdx.y];
    if (blockIdx.x == 0 && threadIdx.x == 0) list->it[blockIdx.y] = I;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kGrids * kMaxItems)
        list->ends[threadIdx.x / kMaxItems][threadIdx.x % kMaxItems] = L.ends[threadIdx.x / kMaxItems][threadIdx.x % kMaxItems];
    if (static_cast<int>(blockIdx.x) >= I.norm_blocks) return;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    double sum = 0.0;
    for (int r = blockIdx.x * 4 + wave; r < I.rows; r += I.norm_blocks * 4) {
        const T* row = static_cast<const T*>(I.src) + static_cast<int64_t>(r) * I.ld_src;
        float* momentum = I.momentum + static_cast<int64_t>(r) * I.ld_momentum;
        for (int c0 = lane; c0 < I.cols; c0 += kWave * kFetch) {
            T g[kFetch];
            float v[kFetch];
#pragma unroll
            for (int f = 0; f < kFetch; ++f) g[f] = row[min(c0 + f * kWave, I.cols - 1)];
            if (U.on) {
#pragma unroll
                for (int f = 0; f < kFetch; ++f) v[f] = momentum[min(c0 + f * kWave, I.cols - 1)];
#pragma unroll
                for (int f = 0; f < kFetch; ++f) {
                    v[f] = __builtin_fmaf(U.mu, v[f], static_cast<float>(g[f]));
                    if (c0 + f * kWave < I.cols) momentum[c0 + f * kWave] = v[f];
                    if (U.nesterov) v[f] = __builtin_fmaf(U.mu, v[f], static_cast<float>(g[f]));
                }
            } else {
#pragma unroll
                for (int f = 0; f < kFetch; ++f) v[f] = static_cast<float>(g[f]);
            }
#pragma unroll
            for (int f = 0; f < kFetch; ++f)
                sum += c0 + f * kWave < I.cols ? static_cast<double>(v[f]) * v[f] : 0.0;
        }
    }
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.y * kNormBlocks + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Tile of 64 x 64 of X in the orientation short x long: both orders of the planes, zeros in the padding.
template <typename T>
__global__ __launch_bounds__(256) void ortho_split(const Items* __restrict__ list, Update U, const double* __restrict__ partial, float eps, _Float16* __restrict__ ws) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const Items& L = *list;
    int b = blockIdx.x;
    const int k = item_of(L, kSplitGrid, b);
    const Item I = L.it[k];
    const Planes P = planes_of(I, ws);
    const int across = (I.lp + 63) / 64, i0 = b / across * 64, j0 = b % across * 64;
    double sum = static_cast<int>(threadIdx.x) < I.norm_blocks ? partial[k * kNormBlocks + threadIdx.x] : 0.0;
    const bool tall = I.rows > I.cols;
    const int tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    // Rows of G run along tx.  As above, the padding reads the matrix's edge, and is set to zero afterwards.
    const int r0 = (tall ? j0 : i0) + ty, c = (tall ? i0 : j0) + tx, cc = min(c, I.cols - 1);
    T g[16];
    float v[16];
#pragma unroll
    for (int y = 0; y < 16; ++y) g[y] = static_cast<const T*>(I.src)[static_cast<int64_t>(min(r0 + 4 * y, I.rows - 1)) * I.ld_src + cc];
    if (U.on) {                                             // the momentum is up to date already
#pragma unroll
        for (int y = 0; y < 16; ++y) v[y] = I.momentum[static_cast<int64_t>(min(r0 + 4 * y, I.rows - 1)) * I.ld_momentum + cc];
#pragma unroll
        for (int y = 0; y < 16; ++y)
            if (U.nesterov) v[y] = __builtin_fmaf(U.mu, v[y], static_cast<float>(g[y]));
    } else {
#pragma unroll
        for (int y = 0; y < 16; ++y) v[y] = static_cast<float>(g[y]);
    }
#pragma unroll
    for (int y = 0; y < 16; ++y)
        if (c >= I.cols || r0 + 4 * y >= I.rows) v[y] = 0.f;
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = sum;
    __syncthreads();
    // in 64 bits: neither a norm beyond fp32 nor the reciprocal of a tiny one costs anything; zeros stay zeros without an eps too
    const double size = sqrt((red[0] + red[1]) + (red[2] + red[3])) + static_cast<double>(eps), inv = size == 0.0 ? 0.0 : 1.0 / size;
#pragma unroll
    for (int y = 0; y < 16; ++y) tile[tall ? tx : ty + 4 * y][tall ? ty + 4 * y : tx] = static_cast<float>(v[y] * inv);     // [short][long]
    __syncthreads();
    const int f = threadIdx.x % 16 * 4;                     // sides are multiples of 32: four halves are inside or outside
#pragma unroll
    for (int y = 0; y < 4; ++y) {
        const int u = threadIdx.x / 16 + 16 * y;
        half4 hi, lo;
        if (i0 + u < I.sp && j0 + f < I.lp) {
#pragma unroll
            for (int e = 0; e < 4; ++e) split4(tile[u][f + e], hi, lo, e);
            const int64_t at = static_cast<int64_t>(i0 + u) * I.ll + j0 + f;
            put(P.x + at, hi);
            put(P.x + P.nx + at, lo);
        }
        if (j0 + u < I.lp && i0 + f < I.sp) {
#pragma unroll
            for (int e = 0; e < 4; ++e) split4(tile[f + e][u], hi, lo, e);
            const int64_t to = static_cast<int64_t>(j0 + u) * I.ls + i0 + f;
            put(P.xt[0] + to, hi);
            put(P.xt[0] + P.nt + to, lo);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// the products
// ---------------------------------------------------------------------------------------------
enum Kind { kGram, kPoly, kApply, kResult };

struct Poly { float a, b, c; };

constexpr bool symmetric(Kind k) { return k == kGram || k == kPoly; }

// Which tile of which item a workgroup computes.
struct Tile { int item, i0, j0; };

// Workgroups are dealt to the 8 XCDs in turn; each gets a contiguous range of the tiles, which run down groups of four
// tile rows, so that an XCD's tiles share their operands in its L2.
template <Kind KIND, int TILE>
__device__ __forceinline__ Tile tile_of(const Items& L) {
    constexpr int kXcds = 8, kGroup = 4;
    const int nb = gridDim.x, x = blockIdx.x % kXcds, q = nb / kXcds, rest = nb % kXcds;
    int b = x * q + min(x, rest) + blockIdx.x / kXcds;
    const int k = item_of(L, symmetric(KIND) ? kSquareGrid : kWideGrid, b);
    if constexpr (symmetric(KIND)) {
        int bj = static_cast<int>((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
        while (bj * (bj + 1) / 2 > b) --bj;
        while ((bj + 1) * (bj + 2) / 2 <= b) ++bj;
        return {k, (b - bj * (bj + 1) / 2) * TILE, bj * TILE};      // i0 <= j0
    } else {
        const int mt = L.it[k].sp / TILE, nt = L.it[k].lp / TILE;
        const int g = b / (kGroup * nt), r = b - g * kGroup * nt, rows = min(kGroup, mt - g * kGroup);
        return {k, (g * kGroup + r % rows) * TILE, r / rows * TILE};
    }
}

// The operands of a tile: P rows from i0, Q rows from j0, along k; the lo plane lies pn (qn) halves after the hi plane.
struct Operands { const _Float16 *p, *q; int64_t pn, qn; int K, ld; };
template <Kind KIND>
__device__ __forceinline__ Operands operands_of(const Item& I, const Planes& P, const Tile& t, int turn) {
    Operands O;
    if constexpr (KIND == kGram) O = {P.x, P.x, P.nx, P.nx, I.lp, I.ll};
    else if constexpr (KIND == kPoly) O = {P.a, P.a, P.na, P.na, I.sp, I.ls};
    else O = {P.b, P.xt[turn], P.na, P.nt, I.sp, I.ls};
    O.p += static_cast<int64_t>(t.i0) * O.ld;
    O.q += static_cast<int64_t>(t.j0) * O.ld;
    return O;
}

// What a product adds to in four rows i .. i + 3 of column j: A (poly) or X^T (apply).
struct Old { half4 hi, lo; };
template <Kind KIND>
__device__ __forceinline__ Old old_values(const Item& I, const Planes& P, int turn, int i, int j) {
    const int64_t at = static_cast<int64_t>(j) * I.ls + i;
    if constexpr (KIND == kPoly) return {*reinterpret_cast<const half4*>(P.a + at), *reinterpret_cast<const half4*>(P.a + P.na + at)};
    else if constexpr (KIND != kGram)
        return {*reinterpret_cast<const half4*>(P.xt[turn] + at), *reinterpret_cast<const half4*>(P.xt[turn] + P.nt + at)};
    else return {};
}

// What a product leaves there, given their sums in v: the new values, which go to X^T, A or B (four halves along memory) and
// come back as words {hi, lo} for the row order, or as they are for the result.
template <Kind KIND>
__device__ __forceinline__ void finish_column(const Item& I, const Planes& P, const Poly& C, int turn, int i, int j, const Old& old,
                                              float (&v)[4], uint32_t (&w)[4]) {
    const int64_t to = static_cast<int64_t>(j) * I.ls + i;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (KIND == kPoly) v[e] = __builtin_fmaf(C.b, whole(old.hi[e], old.lo[e]), C.c * v[e]);
        else if constexpr (KIND != kGram) v[e] = __builtin_fmaf(C.a, whole(old.hi[e], old.lo[e]), v[e]);
    }
    if constexpr (KIND == kResult) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(v[e]);
        return;
    }
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 a, b;
        split(v[e], a, b);
        hi[e] = a;
        lo[e] = b;
        w[e] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, a)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
    }
    _Float16* o = KIND == kGram ? P.a : KIND == kPoly ? P.b : P.xt[turn ^ 1];
    const int64_t n = KIND == kApply ? P.nt : P.na;
    put(o + to, hi);
    put(o + n + to, lo);
}

// Four columns j .. j + 3 of row i from their words, in row order (X, or the mirror image of a tile off the diagonal).
template <Kind KIND>
__device__ __forceinline__ void finish_row(const Item& I, const Planes& P, int i, int j, const uint32_t (&w)[4]) {
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e]));
        lo[e] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e] >> 16));
    }
    _Float16* o = KIND == kGram ? P.a : KIND == kPoly ? P.b : P.x;
    const int64_t n = KIND == kApply ? P.nx : P.na, at = static_cast<int64_t>(i) * (KIND == kApply ? I.ll : I.ls) + j;
    put(o + at, hi);
    put(o + n + at, lo);
}

// Four columns c .. c + 3 of row r of the result, or of the weight it updates.
template <typename T>
__device__ __forceinline__ void write_result(const Item& I, const Update& U, int r, int c, const uint32_t (&w)[4]) {
    if (r >= I.rows || c >= I.cols) return;
    const int n = min(4, I.cols - c);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    if (U.on) {
        float* to = I.weight + static_cast<int64_t>(r) * I.ld_weight + c;
        const float keep = 1.f - U.lr * U.decay;
        const float scale = U.lr * sqrtf(fmaxf(1.f, static_cast<float>(I.rows) / static_cast<float>(I.cols)));
        if (n == 4) {
            float old[4];
            load_as_f32<float, 4>(to, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = old[e] * keep - scale * v[e];
            store_from_f32<float, 4>(to, v);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < n) to[e] = to[e] * keep - scale * v[e];
        }
    } else {
        T* to = static_cast<T*>(I.dst) + static_cast<int64_t>(r) * I.ld_dst + c;
        if (n == 4) {
            store_from_f32<T, 4>(to, v);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < n) to[e] = static_cast<T>(v[e]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// tiles through LDS
// ---------------------------------------------------------------------------------------------
// One 16-byte copy per lane from global memory straight to LDS: the wavefront's 1 KiB lands in order from `to`.
__device__ __forceinline__ void copy_to_lds(const _Float16* from, _Float16* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Four wavefronts, two by two; two stages of 64 along k.  (Measured at 2048 x 2048, where it matters most: stages of 32,
// three to five of them, or eight wavefronts: within 3 % of these.)
constexpr int kWaves = 4, kBk = 64, kStages = 2;

// Rows of a stage in LDS, kBk halves each: the chunk of 16 bytes c of row r lies at place c ^ turn_of(r), so that the 16
// rows that are read at one c in one cycle (256 bytes) lie in different banks.  A copy puts lane i at place i: lane i
// fetches what belongs there.
__device__ __forceinline__ int turn_of(int r) { return r >> 1 & 7; }

// Copy number C of a wavefront's share of a plane of rows.
__device__ __forceinline__ void copy_rows(const _Float16* __restrict__ from, int64_t ld, _Float16* to, int C) {
    constexpr int kChunks = kBk / 8, kRows = kWave / kChunks;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int r0 = (C * kWaves + wave) * kRows, r = r0 + lane / kChunks, c = (lane % kChunks) ^ turn_of(r);
    copy_to_lds(from + r * ld + c * 8, to + r0 * kBk);
}
__device__ __forceinline__ half8 chunk_at(const _Float16* tile, int r, int c) {
    return *reinterpret_cast<const half8*>(tile + r * kBk + ((c ^ turn_of(r)) * 8));
}

// Halves of LDS of a stage: P hi, P lo, Q hi, Q lo.
constexpr int stage_halves(int tile) { return 2 * tile * kBk * 2; }
constexpr size_t lds_bytes(int tile) { return sizeof(_Float16) * stage_halves(tile) * kStages; }

// Meets the other wavefronts once all but the last N of this wavefront's copies have landed (copies land in order) and its
// reads are done.  __syncthreads() would wait for every copy, those of the stages ahead too.
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Orders a wavefront's own writes of LDS before its reads (the unit serves them in order).
__device__ __forceinline__ void wave_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// Asks the scheduler for PRODUCTS matrix instructions with READS reads of LDS, then COPIES copies to LDS spread between
// them.  A copy occupies the address unit for some 16 cycles, which four wavefronts share: issued in one go at the head of
// a stage, they kept the matrix cores waiting for a third of the time.
template <int PRODUCTS, int READS, int COPIES, int X = 0>
__device__ __forceinline__ void interleave() {
    constexpr int kOthers = READS + COPIES;
    if constexpr (X < kOthers) {
        constexpr int n = PRODUCTS * (X + 1) / kOthers - PRODUCTS * X / kOthers;
        if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x008, n, 0);
        __builtin_amdgcn_sched_group_barrier(X < READS ? 0x100 : 0x010, 1, 0);
        interleave<PRODUCTS, READS, COPIES, X + 1>();
    }
}

// Workgroup: a TILE x TILE tile of one product of one item; each wavefront a quarter of it, N x N blocks of 32 x 32;
// kStages of kBk along k in LDS, of which all but the one at work are being filled.
template <typename T, Kind KIND, int TILE>
__global__ __launch_bounds__(kWave* kWaves) void ortho_product(const Items* __restrict__ list, Update U, Poly C, int turn, _Float16* __restrict__ ws) {
    constexpr int N = TILE / 64, kStage = stage_halves(TILE), kPlane = TILE * kBk;
    constexpr int kCopies = kStage / 8 / (kWave * kWaves);  // copies of a wavefront per stage
    constexpr int kSteps = kBk / 16, kShare = kCopies / kSteps, kPer = kCopies / 4;            // ... per step, per plane
    static_assert(kShare * kSteps == kCopies && kPer * 4 == kCopies, "whole copies, equal shares");
    extern __shared__ __align__(16) _Float16 lds[];
    const Tile t = tile_of<KIND, TILE>(*list);
    const Item I = list->it[t.item];
    const Planes P = planes_of(I, ws);
    const Operands O = operands_of<KIND>(I, P, t, turn);
    auto copy = [&](int k0, int stage, int c) {             // copy c of a stage
        const _Float16* from = c < kPer ? O.p : c < 2 * kPer ? O.p + O.pn : c < 3 * kPer ? O.q : O.q + O.qn;
        copy_rows(from + k0, O.ld, lds + stage * kStage + c / kPer * kPlane, c % kPer);
    };
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int wi = wave / 2 * (TILE / 2), wj = wave % 2 * (TILE / 2);
    const int lr = lane % 32, lk = lane / 32;
    f32x16 main_sum[N][N], lo_sum[N][N];
#pragma unroll
    for (int m = 0; m < N; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) main_sum[m][n][e] = lo_sum[m][n][e] = 0.f;
    struct Frags { half8 ah[N], al[N], bh[N], bl[N]; };
    auto read = [&](const _Float16* s, int q, Frags& f) {
#pragma unroll
        for (int m = 0; m < N; ++m) {
            f.ah[m] = chunk_at(s, wi + m * 32 + lr, 2 * q + lk);
            f.al[m] = chunk_at(s + kPlane, wi + m * 32 + lr, 2 * q + lk);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            f.bh[n] = chunk_at(s + 2 * kPlane, wj + n * 32 + lr, 2 * q + lk);
            f.bl[n] = chunk_at(s + 3 * kPlane, wj + n * 32 + lr, 2 * q + lk);
        }
    };
    const int last = O.K - kBk;                              // past the end the last stage is fetched again, for nobody
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
#pragma unroll
        for (int c = 0; c < kCopies; ++c) copy(min(s * kBk, last), s, c);
    int stage = 0;
    for (int k0 = 0; k0 < O.K; k0 += kBk) {
        // stage k0 has landed, everyone's part; the stage before is read out.  The kStages - 2 after k0 may be under way.
        meet<(kStages - 2) * kCopies>();
        const _Float16* s = lds + stage * kStage;
        const int next = min(k0 + (kStages - 1) * kBk, last), into = stage == 0 ? kStages - 1 : stage - 1;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        Frags f[2];
        read(s, 0, f[0]);
#pragma unroll
        for (int q = 0; q < kSteps; ++q) {
            if (q + 1 < kSteps) read(s, q + 1, f[(q + 1) & 1]);
#pragma unroll
            for (int c = 0; c < kShare; ++c) copy(next, into, q * kShare + c);
            const Frags& g = f[q & 1];
#pragma unroll
            for (int m = 0; m < N; ++m)
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    main_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.ah[m], g.bh[n], main_sum[m][n], 0, 0, 0);
                    lo_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.ah[m], g.bl[n], lo_sum[m][n], 0, 0, 0);
                }
#pragma unroll
            for (int m = 0; m < N; ++m)
#pragma unroll
                for (int n = 0; n < N; ++n)
                    lo_sum[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.al[m], g.bh[n], lo_sum[m][n], 0, 0, 0);
        }
        // order: the first step's reads, then each step's matrix instructions with the next step's reads between them
        constexpr int kReads = 4 * N, kProducts = 3 * N * N;
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
#pragma unroll
        for (int q = 0; q + 1 < kSteps; ++q) interleave<kProducts, kReads, kShare>();
        interleave<kProducts, 0, kShare>();
    }
    // what the product adds to, all of it at once: loads between the stores below would wait for one another
    constexpr int kSide = N * 32, kPasses = kSide * kSide / 4 / kWave, kAcross = kSide / 4;
    Old old[kPasses];
#pragma unroll
    for (int x = 0; x < kPasses; ++x)
        old[x] = old_values<KIND>(I, P, turn, t.i0 + wi + (x * kWave + lane) % kAcross * 4, t.j0 + wj + (x * kWave + lane) / kAcross);
    meet<0>();                                              // no copy is under way, nobody reads a stage any more
    // The sums go through LDS, a wavefront's block at a time, so that what lies along memory is read and written in runs
    // of its whole side: buf[j][i].  (Straight from the registers, 16 bytes of a line at a time, this cost as much as a
    // third of the products.)  Element e of a block: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32.
    constexpr int kRow = kSide + 4;
    static_assert(kWaves * kSide * kRow * sizeof(uint32_t) <= lds_bytes(TILE), "fits the stages");
    uint32_t* buf = reinterpret_cast<uint32_t*>(lds) + wave * kSide * kRow;
#pragma unroll
    for (int m = 0; m < N; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t* to = buf + (n * 32 + lr) * kRow + m * 32 + 8 * g + 4 * lk;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    to[e] = __float_as_uint(__builtin_fmaf(lo_sum[m][n][4 * g + e], 1.f / kLo, main_sum[m][n][4 * g + e]));
            }
    wave_lds();
    const bool tall = I.rows > I.cols;
#pragma unroll
    for (int x = 0; x < kPasses; ++x) {
        const int i = (x * kWave + lane) % kAcross * 4, j = (x * kWave + lane) / kAcross;
        uint32_t w[4];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(buf[j * kRow + i + e]);
        finish_column<KIND>(I, P, C, turn, t.i0 + wi + i, t.j0 + wj + j, old[x], v, w);
        if (KIND == kResult && tall) {
            write_result<T>(I, U, t.j0 + wj + j, t.i0 + wi + i, w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) buf[j * kRow + i + e] = w[e];
        }
    }
    if (KIND == kResult ? tall : symmetric(KIND) && t.i0 == t.j0) return;      // (a tile on the diagonal is its own mirror image)
    wave_lds();
#pragma unroll
    for (int x = 0; x < kPasses; ++x) {
        const int j = (x * kWave + lane) % kAcross * 4, i = (x * kWave + lane) / kAcross;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = buf[(j + e) * kRow + i];
        if constexpr (KIND == kResult) write_result<T>(I, U, t.i0 + wi + i, t.j0 + wj + j, w);
        else finish_row<KIND>(I, P, t.i0 + wi + i, t.j0 + wj + j, w);
    }
}

// ---------------------------------------------------------------------------------------------
// tiles of 32 for small matrices
// ---------------------------------------------------------------------------------------------
constexpr int kSmall = 32, kSmallWaves = 8, kSmallAhead = 4;

// Workgroup: a 32 x 32 tile; wavefront w takes its share of the steps of 16 along k, kSmallAhead of them in flight.
template <typename T, Kind KIND>
__global__ __launch_bounds__(kWave* kSmallWaves) void ortho_product_small(const Items* __restrict__ list, Update U, Poly C, int turn, _Float16* __restrict__ ws) {
    __shared__ float part[kSmallWaves][kSmall][kSmall + 1];
    const Tile t = tile_of<KIND, kSmall>(*list);
    const Item I = list->it[t.item];
    const Planes P = planes_of(I, ws);
    const Operands O = operands_of<KIND>(I, P, t, turn);
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, lr = lane % 32, lk = lane / 32;
    const _Float16* p = O.p + static_cast<int64_t>(lr) * O.ld + lk * 8;
    const _Float16* q = O.q + static_cast<int64_t>(lr) * O.ld + lk * 8;
    f32x16 main_sum, lo_sum;
#pragma unroll
    for (int e = 0; e < 16; ++e) main_sum[e] = lo_sum[e] = 0.f;
    const int steps = O.K / 16;
    for (int s0 = wave; s0 < steps; s0 += kSmallWaves * kSmallAhead) {
        half8 ah[kSmallAhead], al[kSmallAhead], bh[kSmallAhead], bl[kSmallAhead];
#pragma unroll
        for (int a = 0; a < kSmallAhead; ++a) {
            const int k = min(s0 + a * kSmallWaves, steps - 1) * 16;
            ah[a] = *reinterpret_cast<const half8*>(p + k);
            al[a] = *reinterpret_cast<const half8*>(p + O.pn + k);
            bh[a] = *reinterpret_cast<const half8*>(q + k);
            bl[a] = *reinterpret_cast<const half8*>(q + O.qn + k);
        }
#pragma unroll
        for (int a = 0; a < kSmallAhead; ++a) {
            if (s0 + a * kSmallWaves >= steps) break;       // the same for the whole wavefront
            main_sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[a], bh[a], main_sum, 0, 0, 0);
            lo_sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[a], bl[a], lo_sum, 0, 0, 0);
            lo_sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[a], bh[a], lo_sum, 0, 0, 0);
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) part[wave][lr][8 * (e / 4) + 4 * lk + e % 4] = __builtin_fmaf(lo_sum[e], 1.f / kLo, main_sum[e]);
    __syncthreads();
    // 256 threads: four rows of a column each, then four columns of a row
    const int u = threadIdx.x / 8, f = threadIdx.x % 8 * 4;
    const bool active = threadIdx.x < 256, tall = I.rows > I.cols;
    uint32_t w[4];
    if (active) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = part[0][u][f + e];
#pragma unroll
            for (int x = 1; x < kSmallWaves; ++x) v[e] += part[x][u][f + e];
        }
        finish_column<KIND>(I, P, C, turn, t.i0 + f, t.j0 + u, old_values<KIND>(I, P, turn, t.i0 + f, t.j0 + u), v, w);
        if (KIND == kResult && tall) write_result<T>(I, U, t.j0 + u, t.i0 + f, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) part[0][u][f + e] = __uint_as_float(w[e]);
    }
    if (KIND == kResult ? tall : symmetric(KIND) && t.i0 == t.j0) return;
    __syncthreads();
    if (!active) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(part[0][f + e][u]);
    if constexpr (KIND == kResult) write_result<T>(I, U, t.i0 + u, t.j0 + f, w);
    else finish_row<KIND>(I, P, t.i0 + u, t.j0 + f, w);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int64_t kMaxTiles = 1LL << 25;   // of 32 x 32 in a turn: far beyond memory, and every grid stays below 2^32 threads

int padded(int v, int unit) { return (v + unit - 1) / unit * unit; }

int64_t tiles_of(const Items& L, bool square, int tile) {
    int64_t n = 0;
    for (int i = 0; i < L.n; ++i) {
        const int64_t s = (L.it[i].sp + tile - 1) / tile, l = (L.it[i].lp + tile - 1) / tile;
        n += square ? s * (s + 1) / 2 : s * l;
    }
    return n;
}

// Operations of the list with sides padded to whole tiles, up to a factor.
double padded_work(const Items& L, int tile) {
    double n = 0.0;
    for (int i = 0; i < L.n; ++i) {
        const double s = padded(L.it[i].sp, tile), l = padded(L.it[i].lp, tile);
        n += s * s * l;
    }
    return n;
}

// Tile size of a launch: a larger tile fetches less for its work, but wants half the chip's 256 CUs to have one, and pads
// every side to itself, work and workspace with it.  How much padding it may bring is measured, whole optimiser steps in us,
// the smaller tile in brackets.  128 for 64, up to a quarter more work: 4 x 200 x 4096 (none) 308 [319], 12 x 96 x 8192 (none)
// 615 [640], 8 x 80 x 2048 (none) 195 [172];  3 x 300 x 4096 (1.44) 402 [332], 24 x 130 x 1030 (1.78) 301 [243], 8 x 64 x 2048
// (4) 197 [155].  64 for 32, up to twice the work: 8 x 40 x 2048 (none) 154 [176], 8 x 130 x 2048 (1.44) 208 [259], 8 x 80 x
// 2048 (1.78) 172 [201];  8 x 16 x 2048 (4) 151 [151] in 12 MiB of workspace [6], 1 x 2^20 (4) 78.0 ms [72.0].
// By the number of tiles, launches in us: 136 symmetric tiles of 128 (side 2048) 49 [58 as 64]; 80 of them, as 288 tiles of 64
// (8 x 512 x 1024), 17.6 [25.7 as 128].  At 96 tiles of 64 (333 x 1001) 64 and 32 are even (11.2, 11.4).
constexpr int kFullGrid = 128;
int choose(const Items& L, bool square) {
    const double least = padded_work(L, 32), middle = padded_work(L, 64);
    if (tiles_of(L, square, 128) >= kFullGrid && padded_work(L, 128) <= 1.25 * middle && middle <= 2.0 * least) return 128;
    return tiles_of(L, square, 64) >= kFullGrid && middle <= 2.0 * least ? 64 : 32;
}

// Sides of the items of one turn; halves of workspace they need.  All sides are padded to the larger tile in use.
struct Choice { int square, wide; };
int64_t lay_out(const cbm_ortho_item* items, int n, Items& L, Choice& choice) {
    L.n = 0;
    for (int i = 0; i < n; ++i) {
        const cbm_ortho_item& s = items[i];
        if (s.rows == 0 || s.cols == 0) continue;
        Item& d = L.it[L.n++];
        d.src = s.src; d.dst = s.dst; d.weight = s.weight; d.momentum = s.momentum;
        d.ld_src = s.ld_src; d.ld_dst = s.ld_dst; d.ld_weight = s.ld_weight; d.ld_momentum = s.ld_momentum;
        d.rows = s.rows; d.cols = s.cols;
        d.sp = std::min(s.rows, s.cols);
        d.lp = std::max(s.rows, s.cols);
        d.norm_blocks = std::max<int64_t>(1, std::min<int64_t>({kNormBlocks, (s.rows + 3) / 4, static_cast<int64_t>(s.rows) * s.cols / 1024}));
    }
    choice = {choose(L, true), choose(L, false)};
    const int unit = std::max(choice.square, choice.wide);
    int64_t halves = 0;
    for (int i = 0; i < L.n; ++i) {
        Item& d = L.it[i];
        d.sp = padded(d.sp, unit);
        d.lp = padded(d.lp, unit);
        d.ls = d.sp;                                        // (rows 128 bytes further apart, off powers of two: no gain)
        d.ll = d.lp;
        d.base = halves;
        halves += item_halves(d);
    }
    int ends[kGrids] = {};
    for (int i = 0; i < kMaxItems; ++i) {
        if (i < L.n) {
            const int64_t s = L.it[i].sp, l = L.it[i].lp, q = s / choice.square;
            if (tiles_of(L, false, 32) <= kMaxTiles) {
                ends[kSplitGrid] += static_cast<int>(((s + 63) / 64) * ((l + 63) / 64));
                ends[kSquareGrid] += static_cast<int>(q * (q + 1) / 2);
                ends[kWideGrid] += static_cast<int>((s / choice.wide) * (l / choice.wide));
            }
        }
        for (int g = 0; g < kGrids; ++g) L.ends[g][i] = i < L.n ? ends[g] : INT_MAX;
    }
    return halves;
}

constexpr int64_t kNormBytes = static_cast<int64_t>(kMaxItems) * kNormBlocks * sizeof(double);
static_assert(sizeof(cbm_ortho_item) == 72, "the layout that bindings mirror");
constexpr int64_t kListBytes = 4096;
static_assert(sizeof(Items) <= kListBytes, "the list");

template <typename T, Kind KIND>
int launch_product(int tile, const Items& L, const Items* list, const Update& U, const Poly& C, int turn, _Float16* ws, hipStream_t st) {
    const unsigned blocks = static_cast<unsigned>(tiles_of(L, symmetric(KIND), tile));
    if (tile == 128) {
        hipLaunchKernelGGL((ortho_product<T, KIND, 128>), dim3(blocks), dim3(kWave * kWaves), lds_bytes(128), st, list, U, C, turn, ws);
    } else if (tile == 64) {
        hipLaunchKernelGGL((ortho_product<T, KIND, 64>), dim3(blocks), dim3(kWave * kWaves), lds_bytes(64), st, list, U, C, turn, ws);
    } else {
        hipLaunchKernelGGL((ortho_product_small<T, KIND>), dim3(blocks), dim3(kWave * kSmallWaves), 0, st, list, U, C, turn, ws);
    }
    return check_launch();
}

template <typename T>
int run_turn(const cbm_ortho_item* items, int n, const Update& U, int steps, const Poly& C, float eps, void* workspace, hipStream_t st) {
    Items L;
    Choice choice;
    lay_out(items, n, L, choice);
    if (L.n == 0) return CBM_OK;
    Items* list = static_cast<Items*>(workspace);
    double* partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + kListBytes);
    _Float16* ws = reinterpret_cast<_Float16*>(static_cast<char*>(workspace) + kListBytes + kNormBytes);
    if (tiles_of(L, false, 32) > kMaxTiles) return CBM_ERR_SHAPE;
    int norm_blocks = 1;
    for (int i = 0; i < L.n; ++i) norm_blocks = std::max(norm_blocks, L.it[i].norm_blocks);
    hipLaunchKernelGGL(ortho_norms<T>, dim3(norm_blocks, L.n), dim3(256), 0, st, L, U, list, partial);
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(ortho_split<T>, dim3(static_cast<unsigned>(tiles_of(L, false, 64))), dim3(256), 0, st, list, U, partial, eps, ws);
    if (int rc = check_launch()) return rc;
    for (int t = 0; t < steps; ++t) {
        if (int rc = launch_product<T, kGram>(choice.square, L, list, U, C, t & 1, ws, st)) return rc;
        if (int rc = launch_product<T, kPoly>(choice.square, L, list, U, C, t & 1, ws, st)) return rc;
        const int rc = t + 1 < steps ? launch_product<T, kApply>(choice.wide, L, list, U, C, t & 1, ws, st)
                                     : launch_product<T, kResult>(choice.wide, L, list, U, C, t & 1, ws, st);
        if (rc) return rc;
    }
    return CBM_OK;
}

constexpr int kMaxSide = 1 << 20;

// Whether what a call writes meets anything else of its list: the items share launches, so their order is open.  By address,
// each matrix is held against those that begin before it ends.
int check_apart(const cbm_ortho_item* items, int n, bool update, int e) {
    struct Matrix { Extent x; intptr_t end; bool written; };
    const std::unique_ptr<Matrix[]> all(new (std::nothrow) Matrix[3 * static_cast<size_t>(n)]);
    if (!all) return CBM_ERR_ALLOC;
    int m = 0;
    auto add = [&](const cbm_ortho_item& s, const void* at, int64_t ld, bool written) {
        const Extent x{at, ld, s.rows, s.cols};
        all[m++] = {x, reinterpret_cast<intptr_t>(at) + ((s.rows - 1) * ld + s.cols) * e, written};
    };
    for (int i = 0; i < n; ++i) {
        const cbm_ortho_item& s = items[i];
        if (s.rows == 0 || s.cols == 0) continue;
        add(s, s.src, s.ld_src, false);
        if (update) {
            add(s, s.weight, s.ld_weight, true);
            add(s, s.momentum, s.ld_momentum, true);
        } else {
            add(s, s.dst, s.ld_dst, true);
        }
    }
    std::sort(all.get(), all.get() + m, [](const Matrix& a, const Matrix& b) { return std::less<const void*>()(a.x.at, b.x.at); });
    for (int i = 0; i < m; ++i)
        for (int j = i + 1; j < m && reinterpret_cast<intptr_t>(all[j].x.at) < all[i].end; ++j)
            if ((all[i].written || all[j].written) && overlap(all[i].x, all[j].x, e)) return CBM_ERR_SHAPE;
    return CBM_OK;
}

int check_items(const cbm_ortho_item* items, int n, bool update, int e) {
    if (n < 0) return CBM_ERR_SHAPE;
    if (n > 0 && !items) return CBM_ERR_NULL;
    for (int i = 0; i < n; ++i) {
        const cbm_ortho_item& s = items[i];
        if (s.rows < 0 || s.cols < 0 || s.rows > kMaxSide || s.cols > kMaxSide) return CBM_ERR_SHAPE;
        if (s.rows == 0 || s.cols == 0) continue;
        if (!s.src || (update ? !s.weight || !s.momentum : !s.dst)) return CBM_ERR_NULL;
        if (s.ld_src < s.cols || (update ? s.ld_weight < s.cols || s.ld_momentum < s.cols : s.ld_dst < s.cols)) return CBM_ERR_SHAPE;
    }
    return check_apart(items, n, update, e);
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
        Choice choice;
        most = std::max(most, lay_out(items + i, std::min(kMaxItems, n - i), L, choice));
    }
    return most ? kListBytes + kNormBytes + most * static_cast<int64_t>(sizeof(_Float16)) : 0;
}

int cbm_ortho_tiles(const cbm_ortho_item* items, int32_t n, int32_t* square, int32_t* wide) {
    if (!square || !wide || (n > 0 && !items)) return CBM_ERR_NULL;
    if (n < 0) return CBM_ERR_SHAPE;
    Items L;
    Choice choice;
    lay_out(items, std::min<int>(n, kMaxItems), L, choice);
    *square = L.n ? choice.square : 0;
    *wide = L.n ? choice.wide : 0;
    return CBM_OK;
}

int cbm_orthogonalise(const cbm_ortho_item* items, int32_t n, int32_t steps, float a, float b, float c, float eps, int32_t dtype,
                      void* workspace, void* stream) {
    if (dtype < CBM_DTYPE_F32 || dtype > CBM_DTYPE_F16) return CBM_ERR_SHAPE;
    if (int rc = check_items(items, n, false, element_bytes(dtype))) return rc;
    if (steps < 1 || !(eps >= 0.f)) return CBM_ERR_SHAPE;
    if (n > 0 && !workspace && cbm_ortho_workspace_bytes(items, n) > 0) return CBM_ERR_NULL;
    const Update U{0.f, 0.f, 0.f, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == CBM_DTYPE_F32) return run_all<float>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
    if (dtype == CBM_DTYPE_BF16) return run_all<__bf16>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
    return run_all<_Float16>(items, n, U, steps, Poly{a, b, c}, eps, workspace, st);
}

int cbm_muon_step(const cbm_ortho_item* items, int32_t n, float lr, float mu, float decay, int32_t nesterov, int32_t steps, float a,
                  float b, float c, float eps, void* workspace, void* stream) {
    if (int rc = check_items(items, n, true, sizeof(float))) return rc;
    if (steps < 1 || !(eps >= 0.f)) return CBM_ERR_SHAPE;
    if (n > 0 && !workspace && cbm_ortho_workspace_bytes(items, n) > 0) return CBM_ERR_NULL;
    const Update U{lr, mu, decay, nesterov, 1};
    return run_all<float>(items, n, U, steps, Poly{a, b, c}, eps, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
