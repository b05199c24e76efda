// Newton-Schulz orthogonalisation of weight updates (gfx950): the singular values of G / |G|_F go through
//   p(s) = a s + b s^3 + c s^5,   (a, b, c) = (3.4445, -4.7750, 2.0315),
// `steps` times, which moves all but the smallest near 1 and leaves the singular vectors alone (the coefficients: K. Jordan et
// al., "Muon: An optimizer for hidden layers in neural networks", 2024).
//
// With m <= n (a taller matrix is taken transposed), A = X X' and Q = a I + b A + c A^2, one step is X <- Q X and makes
// the next Gram matrix A' = Q A Q = Q^2 A: all m x m factors are polynomials of one symmetric matrix, they commute and
// stay symmetric.  So a group of k steps can be taken on m x m matrices alone and applied to X at once,
//   A = X X';  Q_1;  A <- (A Q_1) Q_1;  Q_2;  ...;  X <- (Q_k ... Q_1) X,
// and every m x m product computes its upper tiles only: 3 m^2 n + (4k - 3) m^3 products a group.  What limits k is that a
// Gram matrix carries an error of 2^-24 |A| into directions whose singular value is near 0, where a step multiplies it
// by a^2 = 11.9.  Measured error of five steps against 64 bits, next to float32 products (16 x 144, 256 x 256, 256 x
// 2304):  k = 1  0.9, 0.4, 0.7 times;  k = 2  0.8, 1.2, 1.0 (2.5 on an update of low rank);  k = 3  3.2, 11, 0.7.
//
// Arithmetic: the matrix cores have no fast float32 product, so a number is held as the sum of two float16 numbers
// (hi + lo, 22 bits) times a power of two, and a product is hi hi + hi lo + lo hi in float32 accumulators (the missing
// lo lo is below 2^-22 of the result).  Powers of two put the largest possible entry below float16's limit: entries of
// X are at most 1.25, of A 1.6, of Q products a^3 = 41.  At the other end float16 stops at 2^-24, so entries of X are whole
// multiples of 2^-39, of A of 2^-38, of Q of 2^-34: rows of an update that are far smaller than its norm lose digits, and each
// step multiplies the loss by up to a.  This arithmetic on 64 x 576 with one row, or every other row, smaller by 1e-3 to 1e-11,
// next to float32 products (error of the whole result, emulated on the CPU): at most as much up to 10 steps, 8 times as
// much at 12, 300 times at 15.  Hence the limit of 10 steps.
//
// Packed layout of a matrix: rows of K-contiguous groups of 8 numbers, 16 bytes of hi then 16 bytes of lo.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/azmcts.h"

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int EXP_X = 15, EXP_A = 14, EXP_Q = 10; // stored number = value * 2^EXP
constexpr int MAX_TABLE = 64;                     // matrices per launch when their addresses travel as kernel arguments
constexpr int MAX_BATCH = 4096;                   // and at most
constexpr int CUS = 256;
constexpr int BIG_TILES = 192;                    // 128 x 128 tiles from this number of them on
constexpr int FEW_TILES = CUS;                    // up to here a CU has one workgroup at most
constexpr int NORM_PARTS = 512;                   // partial sums of squares per matrix, at most

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct bf16_t { uint16_t u; };
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(bf16_t v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float as_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t *p, float v)
{
    const uint32_t b = __float_as_uint(v); // to nearest even; a NaN stays one
    p->u = v != v ? (uint16_t)0x7fc0 : (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void put(_Float16 *p, float v) { *p = (_Float16)v; }

// the matrices' addresses: evenly spaced ones (a batch in one tensor) as first and distance, any number of them; others
// as a table
struct Ptrs {
    const char *in0;
    char *out0;
    long long in_step, out_step;
    int even;
    const void *in_at[MAX_TABLE];
    void *out_at[MAX_TABLE];
    __device__ __forceinline__ const void *in(int i) const { return even ? in0 + i * in_step : in_at[i]; }
    __device__ __forceinline__ void *out(int i) const { return even ? out0 + i * out_step : out_at[i]; }
};

// the matrices of a launch: G is rows x cols with row pitch ld (elements), X is G or its transpose, m x n with m <= n
struct Shape {
    int rows, cols, m, n, mp, np; // mp, np: padded with zeros to whole tiles
    long long ld_in, ld_out;
    int tall;
};

// ---- sum of squares, in 64 bits (a float32 square leaves the range at 1e19 and 1e-23)
template <class T> __global__ __launch_bounds__(256) void k_norm(Ptrs p, Shape s, int parts, double *sums)
{
    const T *g = (const T *)p.in(blockIdx.y);
    double acc[4] = {0., 0., 0., 0.};
    // a wavefront takes pieces of 256 cells of a row
    const int pieces = (s.cols + 255) / 256;
    for (long long u = blockIdx.x * 4 + (threadIdx.x >> 6); u < (long long)s.rows * pieces; u += parts * 4) {
        const int i = (int)(u / pieces), j = (int)(u - (long long)i * pieces) * 256 + (threadIdx.x & 63);
        const T *row = g + (size_t)i * s.ld_in;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = as_float(row[min(j + 64 * k, s.cols - 1)]);
#pragma unroll
        for (int k = 0; k < 4; k++) acc[k] = j + 64 * k < s.cols ? fma((double)v[k], (double)v[k], acc[k]) : acc[k];
    }
    double sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    __shared__ double s_w[4];
    if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) sums[(size_t)blockIdx.y * NORM_PARTS + blockIdx.x] = (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]);
}

// hi and lo halves of a number.  It is hidden from the compiler how v came about: it may compute hi twice, once rounded
// from v and once straight from the factors of a product (other bits next to a tie), and take lo from the other one.
template <class V> __device__ __forceinline__ void split1(float v, V &hi, V &lo, int i)
{
    asm("" : "+v"(v));
    hi[i] = (_Float16)v;
    lo[i] = (_Float16)fmaf(-1.f, (float)hi[i], v); // exact (one instruction: an operand may be float16)
}

// of 8 numbers, 32 bytes at p
__device__ __forceinline__ void pack8(char *p, const float (&v)[8])
{
    h8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) split1(v[i], hi, lo, i);
    *(h8 *)p = hi;
    *(h8 *)(p + 16) = lo;
}
// X' = the packed transpose of G / |G| (G itself, row by row, when it is tall), [np][mp]; one 64 x 64 tile of G per workgroup
// (X: also X itself, [mp][np], or NULL)
template <class T> __global__ __launch_bounds__(256) void k_split(Ptrs p, Shape s, int parts, const double *sums, char *XT, char *X)
{
    __shared__ float t[64][65];
    __shared__ double s_scale;
    const int b = blockIdx.z;
    const T *g = (const T *)p.in(b);
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    float v[16]; // all loads are in flight while the sum is taken
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const int r = r0 + (threadIdx.x >> 6) + 4 * k, c = c0 + (threadIdx.x & 63);
        v[k] = as_float(g[(size_t)min(r, s.rows - 1) * s.ld_in + min(c, s.cols - 1)]);
        v[k] = r < s.rows && c < s.cols ? v[k] : 0.f;
    }
    if (threadIdx.x < 64) {
        double sum = 0.;
#pragma unroll
        for (int i = 0; i < NORM_PARTS; i += 64) sum += i + (int)threadIdx.x < parts ? sums[(size_t)b * NORM_PARTS + i + threadIdx.x] : 0.;
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        if (threadIdx.x == 0) s_scale = sum == 0. ? 0. : ldexp(1. / sqrt(sum), EXP_X);
    }
    __syncthreads();
    const double scale = s_scale;
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const int r = (threadIdx.x >> 6) + 4 * k, c = threadIdx.x & 63;
        t[s.tall ? r : c][s.tall ? c : r] = (float)((double)v[k] * scale);
    }
    __syncthreads();
    const int n0 = s.tall ? r0 : c0, m0 = s.tall ? c0 : r0;
    char *out = XT + b * ((size_t)s.mp * s.np * 4);
    for (int e = threadIdx.x; e < 64 * 8; e += 256) {
        const int n = e >> 3, m = (e & 7) * 8;
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = t[n][m + i];
        if (n0 + n < s.np && m0 + m < s.mp) pack8(out + ((size_t)(n0 + n) * s.mp + m0 + m) * 4, w);
        if (X) {
            const int r = e >> 3, c = (e & 7) * 8; // row of X, columns
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = t[c + i][r];
            if (m0 + r < s.mp && n0 + c < s.np) pack8(X + b * ((size_t)s.mp * s.np * 4) + ((size_t)(m0 + r) * s.np + n0 + c) * 4, w);
        }
    }
}

// ---- packed products:  D' = alpha * (A B') + beta * E + gamma * I,  A [M][K], B [N][K] packed
struct Gemm {
    const char *A, *B;
    size_t sA, sB;      // bytes from one matrix of the batch to the next
    int pitchA, pitchB; // bytes per row
    int K;
    int tiles, tiles_m, tiles_n; // tiles per matrix
    int symmetric;      // upper tiles only, each written to both of its places
    float alpha, beta, gamma;
    const char *E;      // packed, same shape as D; or NULL
    size_t sE, sD;
    const char *A2, *B2; // a second product of the same shape in the same launch (no E), or NULL
    char *D2;
    int batch;
    int whole;          // tiles (of all matrices) with a workgroup of their own; of the others ...
    int split;          // ... so many workgroups share the K of each, their float32 sums go to `parts` (k_join)
    float *parts;
    int poly;           // the tile is the whole matrix and D is to hold Q (k_join_poly)
    char *M;            // the packed result by rows too, [M][N], or NULL
    int pitchM;
    char *D;            // packed result, by columns: [N][M]; NULL: to p.out() as G (columns: n, rows: m)
    int pitchD;
};

// 16 bytes per lane straight into LDS; the wavefront's 64 lanes fill 1 KB from `lds` on in lane order
__device__ __forceinline__ void load_lds(const char *g, char *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)g,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// 8 numbers of K for one row of an operand, from two transposing LDS reads of 4: of 16 lanes, lane 4 j + q hands over 4
// neighbouring columns (place q) of row j, and lane l receives column l of the four rows
typedef short s4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ h8 turned(const char *a, const char *b)
{
    union { struct { s4 a, b; } s; h8 h; } u;
    u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)a);
    u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)b);
    return u.h;
}

// Four of those at LDS addresses (bytes) + AT, their second halves FURTHER bytes behind.  The builtin is taken for a read of
// what any load into LDS may still write: the compiler waits for all of them before it, also for the stage that was just
// asked for.  These reads are waited for within the block.
template <int AT, int FURTHER> __device__ __forceinline__ void turned4(unsigned a, unsigned b, unsigned c, unsigned d, h8 &ra, h8 &rb, h8 &rc, h8 &rd)
{
    union { struct { s4 a, b; } s; h8 h; } u, v, w, x;
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(u.s.a), "=&v"(u.s.b), "=&v"(v.s.a), "=&v"(v.s.b), "=&v"(w.s.a), "=&v"(w.s.b), "=&v"(x.s.a), "=&v"(x.s.b)
                 : "v"(a), "v"(b), "v"(c), "v"(d), "n"(AT), "n"(AT + FURTHER)
                 : "memory");
    ra = u.h; rb = v.h; rc = w.h; rd = x.h;
}

constexpr int BK = 32;              // K per stage: 128 bytes of a packed row
// place of 16-byte piece c of row r within the row's 128 bytes: 16 lanes that read the same piece of 16 rows touch
// all 64 banks
__device__ __forceinline__ int place(int r, int c) { return c ^ ((r >> 1) & 7); }
// the same for rows of K: the four rows of a transposing read, 64 bytes of each, touch all 64 banks
__device__ __forceinline__ int place_k(int k, int c) { return c ^ ((k & 1) | (k & 2) << 2); }

constexpr int BAND = 8; // tiles are taken in bands of 8 rows, column by column: 64 neighbours share 8 + 8 panels
__device__ __forceinline__ void tile_at(int i, const Gemm &a, int &ti, int &tj)
{
    for (int first = 0;; first += BAND) {
        const int rows = min(BAND, a.tiles_m - first);
        if (!a.symmetric) {
            const int n = rows * a.tiles_n;
            if (i < n) {
                ti = first + i % rows;
                tj = i / rows;
                return;
            }
            i -= n;
            continue;
        }
        const int corner = rows * (rows + 1) / 2, n = corner + rows * (a.tiles_n - first - rows);
        if (i >= n) {
            i -= n;
            continue;
        }
        if (i < corner) {
            int j = 0;
            while (i > j) i -= ++j;
            ti = first + i;
            tj = first + j;
        } else {
            i -= corner;
            ti = first + i % rows;
            tj = first + rows + i / rows;
        }
        return;
    }
}

// Where a finished tile stands in LDS: [column][row], so that the four rows a lane has of a column are one write, with
// rows exchanged in fours so that reads along the columns find all banks
template <int BM> __device__ __forceinline__ int tile_place(int r, int c) { return c * (BM + 4) + (r ^ (c >> 3 & 7) << 2); }

// A finished tile from LDS to its place, every write a whole group of 8.  The result is stored by columns (D is [N][M]);
// symmetric ones also where the mirror image belongs.
template <int BM, int BN, int THREADS, class T>
__device__ __forceinline__ void store_tile(float *t, const Gemm &a, const Ptrs &p, const Shape &s, int b, int ti, int tj)
{
    const int row0 = ti * BM, col0 = tj * BN; // rows: m, columns: n
    if (!a.D) {
        // 8 neighbours of a row of G per thread: along m where G is X', along n where it is X
        T *out = (T *)p.out(b);
        const bool wide = ((size_t)out | (size_t)s.ld_out * sizeof(T)) % 16 == 0; // whole 16-byte writes
        for (int e = threadIdx.x; e < BM * BN / 8; e += THREADS) {
            const int r = s.tall ? e % (BM / 8) * 8 : e / (BN / 8), c = s.tall ? e / (BM / 8) : e % (BN / 8) * 8;
            __align__(16) T v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) put(v + i, t[s.tall ? tile_place<BM>(r + (i & 4), c) + (i & 3) : tile_place<BM>(r, c + i)]);
            const int left = s.tall ? s.m - row0 - r : s.n - col0 - c;
            if (left <= 0 || (s.tall ? col0 + c >= s.n : row0 + r >= s.m)) continue;
            T *at = s.tall ? out + (size_t)(col0 + c) * s.ld_out + row0 + r : out + (size_t)(row0 + r) * s.ld_out + col0 + c;
            if (wide && left >= 8) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)at)[i] = ((const uint4 *)v)[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < left) at[i] = v[i];
            }
        }
        return;
    }
    char *D = a.D + b * a.sD;
    for (int e = threadIdx.x; e < BM * BN / 8; e += THREADS) {
        const int c = e / (BM / 8), r = e % (BM / 8) * 8;
        float4 *lo4 = (float4 *)(t + tile_place<BM>(r, c)), *hi4 = (float4 *)(t + tile_place<BM>(r + 4, c));
        float4 x = *lo4, y = *hi4;
        float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        const size_t at = (size_t)(col0 + c) * a.pitchD + (size_t)(row0 + r) * 4;
        if (a.E) {
            const h8 hi = *(const h8 *)(a.E + b * a.sE + at), lo = *(const h8 *)(a.E + b * a.sE + at + 16);
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = fmaf(a.beta, (float)hi[i] + (float)lo[i], v[i]) + (col0 + c == row0 + r + i ? a.gamma : 0.f);
            *lo4 = make_float4(v[0], v[1], v[2], v[3]);
            *hi4 = make_float4(v[4], v[5], v[6], v[7]);
        }
        pack8(D + at, v);
    }
    if (a.symmetric ? ti == tj : a.M == nullptr) return;
    char *M = a.symmetric ? D : a.M + b * a.sD;
    const int pitch = a.symmetric ? a.pitchD : a.pitchM;
    __syncthreads();
    for (int e = threadIdx.x; e < BM * BN / 8; e += THREADS) {
        const int r = e / (BN / 8), c = e % (BN / 8) * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = t[tile_place<BM>(r, c + i)];
        pack8(M + (size_t)(row0 + r) * pitch + (size_t)(col0 + c) * 4, v);
    }
}

// BM x BN results per workgroup of 4 wavefronts (2 x 2); per stage and wavefront (BM/64) (BN/64) 2 x 3 matrix
// instructions 32x32x16 on (BM/64 + BN/64) 4 LDS reads.  D places for stages in LDS: D - 1 load while one is used.
// KS groups of 4 wavefronts take every KS-th stage of K, each with stages of its own, and add up at the end: where tiles
// are few a CU needs more loads in flight (what one asks for arrives after 2100 cycles).  Measured with one group and two
// places / several: 256 x 2304, one matrix 225 / 137 us, 4 x 512 x 512 191 / 151 us.  (Every wavefront on its own, a whole
// tile each, with four pieces of K in flight, took 200 us where four groups took 174.)  Large tiles: a CU that has one workgroup of two
// groups is busy, with one of one group it waits (210 symmetric tiles, K = 2560: 60 us; as 820 tiles of 64, four to a CU: 82 us).
// The last tiles may be shared: workgroups take parts of their K and leave float32 sums for k_join.
// TURN: A and B are given as [K][M] and [K][N] (the Gram matrix from X'), and the LDS reads transpose.
template <int BM, int BN, int KS, int D, bool TURN, class T>
__global__ __launch_bounds__(256 * KS, KS < 3 ? 2 : KS) void k_gemm(Gemm a, Ptrs p, Shape s)
{
    constexpr int FM = BM / 64, FN = BN / 64; // 32 x 32 blocks of a wavefront
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int TILE = BN * (BM + 4) * 4;
    __shared__ __align__(16) char lds_all[KS * (D * STAGE > TILE ? D * STAGE : TILE)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int group = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    char *lds = lds_all + group * D * STAGE;
    constexpr bool SHARES = BM == 64 ? TURN && D == 4 : KS == 2; // some tiles may be shared
    // workgroups go round the 8 XCDs: each XCD gets a run of neighbouring tiles, which share operands in its L2
    int item, share = -1, b, ti, tj;
    {
        const bool shared = SHARES && (int)blockIdx.x >= a.whole; // (of the workgroups behind `whole` each XCD gets a run too)
        const int at = shared ? blockIdx.x - a.whole : blockIdx.x, n = shared ? gridDim.x - a.whole : SHARES ? a.whole : gridDim.x;
        const int x = at & 7, i = at >> 3, per = n >> 3, rest = n & 7;
        item = x * per + min(x, rest) + i;
        int tile = item;
        if (shared) {
            tile = item / a.split;
            share = item - tile * a.split;
            tile += a.whole;
        }
        b = tile / a.tiles;
        tile_at(tile - b * a.tiles, a, ti, tj);
    }
    if (a.D2 && b >= a.batch) {
        a.A = a.A2;
        a.B = a.B2;
        a.D = a.D2;
        b -= a.batch;
    }
    const char *A = a.A + b * a.sA + (TURN ? (size_t)ti * BM * 4 : (size_t)ti * BM * a.pitchA);
    const char *B = a.B + b * a.sB + (TURN ? (size_t)tj * BN * 4 : (size_t)tj * BN * a.pitchB);

    constexpr int LOADS = (BM + BN) / 8 / 4; // 1 KB loads per wavefront and stage
    const char *src[LOADS];
    int dst[LOADS];
    size_t next_a = 128, next_b = 128; // from stage to stage
    if (TURN) {
        next_a = (size_t)BK * a.pitchA;
        next_b = (size_t)BK * a.pitchB;
    }
#pragma unroll
    for (int l = 0; l < LOADS; l++) {
        const int kb = l * 4 + wave; // KB of the stage
        dst[l] = kb * 1024;
        if (TURN) {
            constexpr int PA = BM / 4, PB = BN / 4; // 16-byte pieces per row of K
            if (kb < BM / 8) {
                const int k = kb * 64 / PA + lane / PA;
                src[l] = A + (size_t)k * a.pitchA + place_k(k, lane % PA) * 16;
            } else {
                const int k = (kb - BM / 8) * 64 / PB + lane / PB;
                src[l] = B + (size_t)k * a.pitchB + place_k(k, lane % PB) * 16;
            }
        } else {
            const int r = kb * 8 + (lane >> 3), c = place(r, lane & 7);
            src[l] = kb * 8 < BM ? A + (size_t)r * a.pitchA + c * 16 : B + (size_t)(r - BM) * a.pitchB + c * 16;
        }
    }
    const auto load_stage = [&](int k, char *to) {
#pragma unroll
        for (int l = 0; l < LOADS; l++) load_lds(src[l] + (size_t)k * (l * 4 < BM / 8 ? next_a : next_b), to + dst[l]);
    };
    // The small products have accumulators of their own: added to the large ones they would cost a rounding each
    // (three times the error of one step).  They stay in the last product of a bfloat16 result too: without them its error is
    // 2^-12 of |Q| |X|, and Q is a^k = 41 (three steps) where X has next to nothing, four times the type's rounding on an
    // update of low rank.
    f16v acc[FM][FN], low[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = low[i][j][e] = 0.f;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    const int lr = lane & 31, half = lane >> 5;
    int stages = a.K / BK;
    if (SHARES && share >= 0) { // this workgroup's share of them
        const int each = (stages + a.split - 1) / a.split, first = share * each;
        stages = max(0, min(each, stages - first));
#pragma unroll
        for (int l = 0; l < LOADS; l++) src[l] += (size_t)first * (l * 4 < BM / 8 ? next_a : next_b);
    }
#pragma unroll
    for (int d = 0; d < D - 1; d++) {
        if (d * KS + group < stages) load_stage(d * KS + group, lds + d * STAGE);
        asm volatile("" ::: "memory"); // (in this order: the waits below count loads)
    }
    // (one way out of the loop: where there were two the compiler counted the wait states between the last products and the
    // first use of their results along the longer one, and results came without the last products)
    const int rounds = (stages + KS - 1) / KS, mine = KS == 1 ? rounds : (stages - group + KS - 1) / KS; // of all groups, of this one
    int at = 0, to = D - 1; // places of this round's stage and of the one that is asked for
    for (int k = 0; k < mine; k++) {
        // this wavefront's part of the group's stage k has arrived (loads arrive in order, up to D - 2 stages of them stay
        // behind it), and it has read all it wanted of stage k - 1
        static_assert(D == 2 || D == 4, "the waits below");
        const int next = (k + 1) * KS + group;
        if (D == 4 && next + KS < stages) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");
        else if (D == 4 && next < stages) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier(); // (not __syncthreads(), which would wait for all loads)
        asm volatile("" ::: "memory");
        const char *cur = lds + at * STAGE;
        const int after = (k + D - 1) * KS + group;
        if (after < stages) load_stage(after, lds + to * STAGE);
        at = at + 1 == D ? 0 : at + 1;
        to = to + 1 == D ? 0 : to + 1;
        const auto half_stage = [&](auto which) {
            constexpr int ks = decltype(which)::value;
            h8 ah[FM], al[FM], bh[FN], bl[FN];
            if constexpr (TURN) {
                static_assert(!TURN || (FM == 1 && FN == 1 && BM == BN), "one block of each operand");
                const int q = lane & 3, kk = half * 8 + (lane >> 2 & 3), f = place_k(kk, 0), up = (lane >> 4 & 1) * 4 + (q & 2);
                const unsigned at = (unsigned)(size_t)(const __attribute__((address_space(3))) char *)cur + kk * BM * 4 + (q & 1) * 8;
                const int ca = wm / 4 + up, cb = wn / 4 + up;
                turned4<ks * 16 * BM * 4, 4 * BM * 4>(at + (ca ^ f) * 16, at + ((ca + 1) ^ f) * 16, at + BM * 128 + (cb ^ f) * 16,
                                                      at + BM * 128 + ((cb + 1) ^ f) * 16, ah[0], al[0], bh[0], bl[0]);
            } else {
                const int c = (ks * 2 + half) * 2;
#pragma unroll
                for (int i = 0; i < FM; i++) {
                    const int r = wm + i * 32 + lr;
                    ah[i] = *(const h8 *)(cur + r * 128 + place(r, c) * 16);
                    al[i] = *(const h8 *)(cur + r * 128 + place(r, c + 1) * 16);
                }
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    const int r = BM + wn + j * 32 + lr;
                    bh[j] = *(const h8 *)(cur + r * 128 + place(r, c) * 16);
                    bl[j] = *(const h8 *)(cur + r * 128 + place(r, c + 1) * 16);
                }
            }
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], low[i][j], 0, 0, 0);
                    low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], low[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
                }
        };
        half_stage(std::integral_constant<int, 0>());
        half_stage(std::integral_constant<int, 1>());
    }
    if (mine < rounds) __builtin_amdgcn_s_barrier(); // (the last round has no stage for this group)
    __syncthreads();
    float *t = (float *)lds_all, *part = (float *)(lds_all + group * TILE);
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; q++) v[q] = (acc[i][j][e + q] + low[i][j][e + q]) * a.alpha;
                *(float4 *)(part + tile_place<BM>(wm + i * 32 + e * 2 + half * 4, wn + j * 32 + lr)) = make_float4(v[0], v[1], v[2], v[3]);
            }
    __syncthreads();
    if (KS > 1) { // the groups' sums in their order
        for (int e = threadIdx.x; e < BM * BN / 4; e += 256 * KS) {
            const int at = tile_place<BM>(e % (BM / 4) * 4, e / (BM / 4));
            float4 v = *(float4 *)(t + at);
#pragma unroll
            for (int g = 1; g < KS; g++) {
                const float4 o = *(const float4 *)(t + g * (TILE / 4) + at);
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            *(float4 *)(t + at) = v;
        }
        __syncthreads();
    }
    if (SHARES && share >= 0) {
        for (int e = threadIdx.x; e < BM * BN / 4; e += 256 * KS)
            ((float4 *)(a.parts + (size_t)item * BM * BN))[e] = *(const float4 *)(t + tile_place<BM>(e % (BM / 4) * 4, e / (BM / 4)));
        return;
    }
    store_tile<BM, BN, 256 * KS, T>(t, a, p, s, b, ti, tj);
}

// 16-byte piece of a row of M * 4 bytes: rows spread over the banks
template <int M> __device__ __forceinline__ int bank(int r, int piece) { return M == 64 ? piece ^ (r & 15) : piece ^ ((r >> 1) & 7); }
// first of the two pieces (hi, lo) of the 8 columns 16 c + 4 h + {0..3, 8..11} of a packed row
__device__ __forceinline__ int slot(int c, int h) { return (c * 2 + h) * 2; }

__device__ __forceinline__ void split8(const float *v, h8 &hi, h8 &lo)
{
#pragma unroll
    for (int i = 0; i < 8; i++) split1(v[i], hi, lo, i);
}

// A tile (rows 32 i, columns 32 j) of Q = a I + b A + c A^2, times 2^EXP_Q, for A of M x M in LDS (rows of blocks of 16
// columns, in a block the 8 of slot 0, then of slot 1, hi and lo).  A lane's results are four rows side by side of its
// column, so (Q is symmetric) f[c] is what slot `half` of block 2 i + c of row 32 j + lane mod 32 holds, and the elements of
// A that go with it stand in the same place.
template <int M> __device__ __forceinline__ void poly_tile(const char *sA, int i, int j, int lane, float (&f)[2][8])
{
    constexpr int C = M / 16;
    const int lr = lane & 31, half = lane >> 5, ra = i * 32 + lr, rb = j * 32 + lr;
    f16v acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.f;
    h8 ah[C], bh[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        ah[c] = *(const h8 *)(sA + ra * M * 4 + bank<M>(ra, slot(c, half)) * 16);
        bh[c] = *(const h8 *)(sA + rb * M * 4 + bank<M>(rb, slot(c, half)) * 16);
        const h8 al = *(const h8 *)(sA + ra * M * 4 + bank<M>(ra, slot(c, half) + 1) * 16);
        const h8 bl = *(const h8 *)(sA + rb * M * 4 + bank<M>(rb, slot(c, half) + 1) * 16);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh[c], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[c], bl, acc, 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < C; c++) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[c], bh[c], acc, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const char *at = sA + rb * M * 4;
        const h8 hi = *(const h8 *)(at + bank<M>(rb, slot(2 * i + c, half)) * 16), lo = *(const h8 *)(at + bank<M>(rb, slot(2 * i + c, half) + 1) * 16);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            f[c][k] = fmaf((float)hi[k] + (float)lo[k], NS_B * 0x1p-4f, acc[8 * c + k] * (NS_C * 0x1p-18f)); // 2^(EXP_Q - EXP_A), 2^(EXP_Q - 2 EXP_A)
            if (i * 32 + 16 * c + 8 * (k >> 2) + 4 * half + (k & 3) == rb) f[c][k] += NS_A * 0x1p10f;
        }
    }
}
static_assert(EXP_X == 15 && EXP_A == 14 && EXP_Q == 10, "the powers of two written out in poly_tile and k_small");

// the sums of the workgroups that shared a tile, in their order; 64 x 64 of its results per workgroup
template <int BM, class T> __global__ __launch_bounds__(256) void k_join(Gemm a, Ptrs p, Shape s)
{
    constexpr int Q = BM / 64;
    __shared__ __align__(16) float t[64 * 68];
    const int tile = blockIdx.x / (Q * Q), q_row = blockIdx.x % Q, q_col = blockIdx.x / Q % Q;
    int b = (a.whole + tile) / a.tiles, ti, tj;
    tile_at(a.whole + tile - b * a.tiles, a, ti, tj);
    if (a.D2 && b >= a.batch) {
        a.D = a.D2;
        b -= a.batch;
    }
    if (a.symmetric && ti == tj && q_row > q_col) return; // (written with its mirror image)
    const float *part = a.parts + (size_t)tile * a.split * BM * BM + q_col * 64 * BM + q_row * 64;
    float4 v[4];
    for (int i = 0; i < a.split; i++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int e = q * 256 + threadIdx.x;
            const float4 o = *(const float4 *)(part + (size_t)i * BM * BM + e / 16 * BM + e % 16 * 4);
            if (i == 0) v[q] = o;
            else {
                v[q].x += o.x; v[q].y += o.y; v[q].z += o.z; v[q].w += o.w;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int e = q * 256 + threadIdx.x;
        *(float4 *)(t + tile_place<64>(e % 16 * 4, e / 16)) = v[q];
    }
    __syncthreads();
    store_tile<64, 64, 256, T>(t, a, p, s, b, ti * Q + q_row, tj * Q + q_col);
}

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// The same where the tile is the whole Gram matrix (up to 64 rows), and Q at once, packed to a.D: one launch less a step
__global__ __launch_bounds__(256) void k_join_poly(Gemm a)
{
    __shared__ __align__(16) char sA[64 * 256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float4 *part = (const float4 *)(a.parts + (size_t)blockIdx.x * a.split * 64 * 64);
    float4 v[4];
#pragma unroll
    for (int q = 0; q < 4; q++) v[q] = part[q * 256 + threadIdx.x];
    for (int i = 1; i < a.split; i++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float4 o = part[(size_t)i * 1024 + q * 256 + threadIdx.x];
            v[q].x += o.x; v[q].y += o.y; v[q].z += o.z; v[q].w += o.w;
        }
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int e = q * 256 + threadIdx.x, r = e % 16 * 4, c = e / 16; // rows r..r+3 of column c, stored as row c
        const float x[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        h4 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; k++) split1(x[k], hi, lo, k);
        char *row = sA + c * 256 + (r >> 3 & 1) * 8;
        *(h4 *)(row + bank<64>(c, slot(r >> 4, r >> 2 & 1)) * 16) = hi;
        *(h4 *)(row + bank<64>(c, slot(r >> 4, r >> 2 & 1) + 1) * 16) = lo;
    }
    __syncthreads();
    const int i = wave >> 1, j = wave & 1, half = lane >> 5;
    float f[2][8];
    poly_tile<64>(sA, i, j, lane, f);
    char *D = a.D + blockIdx.x * a.sD + (size_t)(j * 32 + (lane & 31)) * a.pitchD;
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int u = 0; u < 2; u++) { // columns 16 (2 i + c) + 8 u + 4 half + {0..3}
            h4 hi, lo;
#pragma unroll
            for (int k = 0; k < 4; k++) split1(f[c][4 * u + k], hi, lo, k);
            char *at = D + (16 * (2 * i + c) + 8 * u) * 4 + 4 * half * 2;
            *(h4 *)at = hi;
            *(h4 *)(at + 16) = lo;
        }
}

// ---------------------------------------------------------------- small matrices: all steps in one launch
//
// A matrix of m <= 32 MT rows and n <= 256 NT columns belongs to one workgroup of 8 wavefronts and stays in registers:
// a wavefront owns NT column tiles of 32 (lane l: column l mod 32; its registers: rows, in the order in which the matrix
// instruction leaves a result), as hi and lo halves.  In that order a tile is at once the operand of the next Q X: only
// Q's columns have to be stored in the same order.  For the Gram matrix the tile is turned through LDS (rows to lanes)
// by transposing reads, every wavefront adds up its own columns and the eight partial sums meet in LDS in a fixed order.  Launches bound the general path here
// (17 of them, 5 us each); this one is bound by the latency of 3 barriers a step (2 up to 32 rows) and
// by one CU's matrix cores and its share of the memory (11 of 40 us at 64 x 576 go into reading and writing).
constexpr int SMALL_WAVES = 8;

__device__ __forceinline__ int row_of(int r) { return (r & ~12) | (r & 4) << 1 | (r & 8) >> 1; }

template <int MT, int NT, class T> __global__ __launch_bounds__(64 * SMALL_WAVES, 2) void k_small(Ptrs p, Shape s, int steps)
{
    constexpr int M = 32 * MT, LD = M + 8, C = 2 * MT; // C: blocks of 16 rows
    constexpr int TURN = 32 * LD * 2;                  // one half (hi or lo) of a tile, [column][row], rows 16 bytes apart
    constexpr int AREA = M * M * 4 > 2 * TURN ? M * M * 4 : 2 * TURN;
    __shared__ __align__(16) char lds[SMALL_WAVES * AREA + MT * M * M * 4]; // (MT == 2: all 160 KB of a CU)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 31, half = lane >> 5;
    char *area = lds + wave * AREA, *sA = lds + SMALL_WAVES * AREA, *sQ = sA + M * M * 4;
    const int tiles = (s.n + 31) / 32;

    // X and |X|.  A lane's registers hold, of each block of 16 rows, rows 4 half + {0..3, 8..11}: hi and lo, 8 each
    h8 xh[NT][C], xl[NT][C];
    {
        float x[NT][C][8];
        const T *g = (const T *)p.in(blockIdx.x);
        const long long pm = s.tall ? 1 : s.ld_in, pn = s.tall ? s.ld_in : 1;
        // (no branch around a load: all of them are in flight together; a row number that is the same in all lanes but for
        // their half is a scalar offset)
        const auto load = [&](auto full) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int n = (t * SMALL_WAVES + wave) * 32 + lr;
                const T *col = g + min(n, s.n - 1) * pn + (decltype(full)::value ? 4 * half * pm : 0);
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int m = c * 16 + 8 * (e >> 2) + (e & 3);
                        if (decltype(full)::value) {
                            const float v = as_float(col[m * pm]);
                            x[t][c][e] = n < s.n ? v : 0.f;
                        } else {
                            const float v = as_float(col[min(m + 4 * half, s.m - 1) * pm]);
                            x[t][c][e] = m + 4 * half < s.m && n < s.n ? v : 0.f;
                        }
                    }
            }
        };
        if (s.m == M && s.tall) { // a lane's rows lie side by side in fours
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int n = (t * SMALL_WAVES + wave) * 32 + lr;
                const T *col = g + min(n, s.n - 1) * pn + 4 * half;
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        T four[4];
                        __builtin_memcpy(four, col + c * 16 + 2 * e, sizeof(four));
#pragma unroll
                        for (int i = 0; i < 4; i++) x[t][c][e + i] = n < s.n ? as_float(four[i]) : 0.f;
                    }
            }
        } else if (s.m == M) load(std::true_type());
        else load(std::false_type());
        double sum = 0.;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) sum = fma((double)x[t][c][e], (double)x[t][c][e], sum);
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) ((double *)lds)[wave] = sum;
        __syncthreads();
        sum = 0.;
#pragma unroll
        for (int w = 0; w < SMALL_WAVES; w++) sum += ((double *)lds)[w];
        __syncthreads();
        // 1 / |X| = f 2^k with f in [1/2, 1]: the power of two first (the smallest float32 numbers lose nothing), then a
        // float32 product, rounded once
        int k;
        const float f = sum == 0. ? 0.f : (float)frexp(1. / sqrt(sum), &k);
        k = sum == 0. ? 0 : k + EXP_X;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int c = 0; c < C; c++) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[t][c][e] = ldexpf(x[t][c][e], k) * f;
                split8(x[t][c], xh[t][c], xl[t][c]);
            }
    }

    for (int step = 0; step < steps; step++) {
        // Gram matrix of this wavefront's columns, upper tiles
        // (two row blocks: the small products apart, so that fewer instructions wait for each other: 16 x 64 x 768 49 -> 44 us;
        // with one row block the sums cost more, 7 x 16 x 144 13.3 -> 14.0 us)
        constexpr bool APART = MT > 1;
        f16v gram[MT * (MT + 1) / 2], low[MT * (MT + 1) / 2];
#pragma unroll
        for (int q = 0; q < MT * (MT + 1) / 2; q++)
#pragma unroll
            for (int e = 0; e < 16; e++) gram[q][e] = low[q][e] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t * SMALL_WAVES + wave >= tiles) continue;
            // turned through LDS: a transposing read hands lane l of 16 the 4 columns of place l of a block of 16 rows, so
            // the operand's rows come with bits 2 and 3 of their number exchanged (row_of)
#pragma unroll
            for (int c = 0; c < C; c++) {
                *(h8 *)(area + (lr * LD + c * 16 + half * 8) * 2) = xh[t][c];
                *(h8 *)(area + TURN + (lr * LD + c * 16 + half * 8) * 2) = xl[t][c];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            h8 hi[MT][2], lo[MT][2];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int n = c * 16 + half * 8 + (lr >> 2 & 3), at = (n * LD + i * 32 + (lr >> 4) * 16 + (lr & 3) * 4) * 2;
                    hi[i][c] = turned(area + at, area + at + 4 * LD * 2);
                    lo[i][c] = turned(area + TURN + at, area + TURN + at + 4 * LD * 2);
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            // (instructions on the same accumulator wait for each other: the tiles in turn)
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int k = 0; k < 3; k++)
#pragma unroll
                    for (int i = 0, q = 0; i < MT; i++)
#pragma unroll
                        for (int j = i; j < MT; j++, q++) {
                            f16v &to = APART && k < 2 ? low[q] : gram[q];
                            to = __builtin_amdgcn_mfma_f32_32x32x16_f16(k == 0 ? lo[i][c] : hi[i][c], k == 1 ? lo[j][c] : hi[j][c], to, 0, 0, 0);
                        }
        }
        if (APART) {
#pragma unroll
            for (int q = 0; q < MT * (MT + 1) / 2; q++)
#pragma unroll
                for (int e = 0; e < 16; e++) gram[q][e] += low[q][e];
        }
        // partial sums to the wavefront's own area, row c holding column c (the matrix is symmetric)
#pragma unroll
        for (int i = 0, q = 0; i < MT; i++)
#pragma unroll
            for (int j = i; j < MT; j++, q++) {
                const int c = row_of(j * 32 + lr);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int r = row_of(i * 32 + 2 * e + 4 * half);
                    *(float4 *)(area + c * M * 4 + bank<M>(c, r >> 2) * 16) = make_float4(gram[q][e], gram[q][e + 1], gram[q][e + 2], gram[q][e + 3]);
                    if (i != j) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            *(float *)(area + (r + k) * M * 4 + bank<M>(r + k, c >> 2) * 16 + (c & 3) * 4) = gram[q][e + k];
                    }
                }
            }
        __syncthreads();
        const int r = threadIdx.x / (M / 8), c16 = threadIdx.x % (M / 8) >> 1, h = threadIdx.x & 1;
        const bool mine = threadIdx.x < M * M / 8;
        float v[8];
        if (mine) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = 0.f;
#pragma unroll
            for (int w = 0; w < SMALL_WAVES; w++) {
                const char *row = lds + w * AREA + r * M * 4;
                const float4 a = *(const float4 *)(row + bank<M>(r, c16 * 4 + h) * 16);
                const float4 b = *(const float4 *)(row + bank<M>(r, c16 * 4 + h + 2) * 16);
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = ldexpf(v[k], EXP_A - 2 * EXP_X);
            h8 hi, lo;
            split8(v, hi, lo);
            *(h8 *)(sA + r * M * 4 + bank<M>(r, slot(c16, h)) * 16) = hi;
            *(h8 *)(sA + r * M * 4 + bank<M>(r, slot(c16, h) + 1) * 16) = lo;
        }
        __syncthreads();
        // one 32 x 32 tile of Q per wavefront, or the only one in every wavefront
        h8 qh1[2], ql1[2];
        if (MT == 1 ? wave < tiles : wave < MT * MT) {
            const int i = MT == 1 ? 0 : wave / MT, j = MT == 1 ? 0 : wave % MT, rb = j * 32 + lr;
            float f[2][8];
            poly_tile<M>(sA, i, j, lane, f);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                split8(f[c], qh1[c], ql1[c]);
                if (MT > 1) {
                    *(h8 *)(sQ + rb * M * 4 + bank<M>(rb, slot(2 * i + c, half)) * 16) = qh1[c];
                    *(h8 *)(sQ + rb * M * 4 + bank<M>(rb, slot(2 * i + c, half) + 1) * 16) = ql1[c];
                }
            }
        }
        if (MT > 1) __syncthreads();
        // X <- Q X
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t * SMALL_WAVES + wave >= tiles) continue;
            float x[C][8];
            f16v acc[MT];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][e] = 0.f;
            // the small products first, then the large ones on top; the row blocks in turn
            h8 qh[MT][C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                h8 ql[MT];
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const int rq = i * 32 + lr;
                    qh[i][c] = MT == 1 ? qh1[c] : *(const h8 *)(sQ + rq * M * 4 + bank<M>(rq, slot(c, half)) * 16);
                    ql[i] = MT == 1 ? ql1[c] : *(const h8 *)(sQ + rq * M * 4 + bank<M>(rq, slot(c, half) + 1) * 16);
                }
#pragma unroll
                for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql[i], xh[t][c], acc[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[i][c], xl[t][c], acc[i], 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[i][c], xh[t][c], acc[i], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[2 * i + (e >> 3)][e & 7] = acc[i][e] * 0x1p-10f; // 2^-EXP_Q
#pragma unroll
            for (int c = 0; c < C; c++) split8(x[c], xh[t][c], xl[t][c]);
        }
    }
    T *out = (T *)p.out(blockIdx.x);
    const long long pm = s.tall ? 1 : s.ld_out, pn = s.tall ? s.ld_out : 1;
    const auto store = [&](auto full) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int n = (t * SMALL_WAVES + wave) * 32 + lr;
            if (n >= s.n) continue;
            T *col = out + n * pn + 4 * half * pm;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int m = c * 16 + 8 * (e >> 2) + (e & 3);
                    const float v = ((float)xh[t][c][e] + (float)xl[t][c][e]) * 0x1p-15f; // 2^-EXP_X
                    if (decltype(full)::value || m + 4 * half < s.m) put(col + m * pm, v);
                }
        }
    };
    if (s.m == M && s.tall) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int n = (t * SMALL_WAVES + wave) * 32 + lr;
            if (n >= s.n) continue;
            T *col = out + n * pn + 4 * half;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    T four[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) put(four + i, ((float)xh[t][c][e + i] + (float)xl[t][c][e + i]) * 0x1p-15f);
                    __builtin_memcpy(col + c * 16 + 2 * e, four, sizeof(four));
                }
        }
    } else if (s.m == M) store(std::true_type());
    else store(std::false_type());
}

// ---------------------------------------------------------------- host side

int launch_ok() { return hipGetLastError() == hipSuccess ? AZ_OK : AZ_ERR_HIP; }

template <class F> void by_type(int dtype, F f)
{
    if (dtype == AZ_F32) f((float *)nullptr);
    else if (dtype == AZ_BF16) f((bf16_t *)nullptr);
    else f((_Float16 *)nullptr);
}

int round_up(int v, int to) { return (v + to - 1) / to * to; }

// (count: matrices of the call)
Shape shape_of(int rows, int cols, int count)
{
    Shape s = {};
    s.rows = rows;
    s.cols = cols;
    s.tall = rows > cols;
    s.m = s.tall ? cols : rows;
    s.n = s.tall ? rows : cols;
    // to whole large tiles only where the product X <- Q X has enough of them (20 x 150 x 300 padded to 128: 131 us, to 64: 115;
    // 4 x 400 x 1100 198 and 180 us)
    const bool big = s.m > 64 && (long long)((s.m + 127) / 128) * ((s.n + 127) / 128) * (count < MAX_BATCH ? count : MAX_BATCH) >= BIG_TILES;
    s.mp = round_up(s.m, big ? 128 : 64);
    s.np = round_up(s.n, big ? 128 : 64);
    return s;
}

struct Plan {
    size_t x, mm;     // bytes of a packed X and of a packed m x m matrix
    size_t sums, parts, total;
};
Plan plan_of(const Shape &s, int batch)
{
    Plan p;
    p.x = (size_t)s.mp * s.np * 4;
    p.mm = (size_t)s.mp * s.mp * 4;
    p.sums = (size_t)batch * NORM_PARTS * sizeof(double);
    const size_t side = s.mp % 128 == 0 ? 128 : 64;
    p.parts = CUS * side * side * 4; // sums of shared tiles: at most one for every CU
    p.total = p.sums + p.parts + batch * (3 * p.x + 5 * p.mm);
    return p;
}

// launches D = alpha A B' + ... over `batch` matrices
void gemm(Gemm a, int M, int N, bool turn, int batch, int dtype, const Ptrs &p, const Shape &s, hipStream_t st)
{
    a.batch = batch;
    if (a.D2) batch *= 2;
    // 128 x 128 tiles halve the operand traffic of 64 x 64 ones, but most CUs should have one (2304 x 2304, 171 symmetric tiles:
    // 53 us either way; 210 of them 60 against 82 us)
    const auto tiles = [&](int t) { return a.symmetric ? (long long)(M / t) * (M / t + 1) / 2 : (long long)(M / t) * (N / t); };
    const bool big = M % 128 == 0 && N % 128 == 0 && tiles(128) * batch >= BIG_TILES;
    const int t = big ? 128 : 64;
    const long long groups = tiles(t) * batch;
    a.tiles = (int)tiles(t);
    a.tiles_m = M / t;
    a.tiles_n = N / t;
    // workgroups that leave CUs with one or two of them get more wavefronts each
    int ks = big ? (groups <= CUS ? 2 : 1) : groups <= FEW_TILES ? 4 : groups <= 2 * FEW_TILES ? 2 : 1;
    a.split = 1;
    long long whole = groups;
    if (turn && ks == 4) {
        // Gram matrices of few tiles and a long K: four stages of a workgroup take about 0.8 us, joining the shares of
        // several workgroups 4.5 us
        const int rounds = (a.K / BK + 3) / 4;
        int most = (int)(FEW_TILES / groups);
        if (most > (rounds + 1) / 2) most = (rounds + 1) / 2;
        if (a.poly || (most > 1 && rounds - (rounds + most - 1) / most >= 6)) {
            a.split = most;
            whole = 0;
        }
    } else if (big && groups > CUS && groups < 4 * CUS) {
        // A few large tiles more than CUs: a CU that gets another one doubles its time, so the last ones are shared by as
        // many workgroups as there are CUs.  272 tiles, K = 4096 / 2048: 151 / 85 us -> 116 + 9 / 67 + 10 us (with the
        // joining); 288 tiles, K = 1024: 46 -> 43 + 7 us, so not there.  The more tiles are left, the fewer share each and the
        // more there is to join, and a short K saves less.  Five steps of one matrix, shared / not, with 256 + `rest` tiles:
        // K = 1024, rest 8: 478 / 479 us;  K = 1280, rest 4: 506 / 516, 14: 497 / 503, 24: 509 / 503, 64: 541 / 529;  K = 1536,
        // rest 8: 652 / 677, 44: 673 / 677, 68: 702 / 700, 116: 767 / 740;  K = 2048, rest 16: 880 / 896, 64: 932 / 943, 80: 959 /
        // 962, 96: 987 / 977, 112: 1013 / 995;  K = 3200, rest 113 and 69: 2272 / 2385.
        const long long rest = groups % CUS;
        if (rest && rest <= CUS / 2 && 12 * rest <= a.K - 1024) {
            ks = 2;
            a.split = (int)(CUS / rest);
            if (a.split > a.K / BK / 4) a.split = a.K / BK / 4;
            whole = groups - rest;
        }
    }
    a.whole = (int)whole;
    const long long shared = groups - whole;
    // Two groups with four places each ask for six stages at once.  That matters more than wavefronts for Gram matrices (1 x
    // 1024 x 1024 199 -> 196 us in all) and up to 12 stages (64 x 100 x 200 207 -> 196 us); other products of 40 stages are
    // faster with four groups (5 x 1201 x 333 193, 206 us).
    const bool deep = ks == 4 && (turn || a.K / BK / a.split <= 12);
    if (deep) ks = 2;
    const dim3 grid((unsigned)(whole + shared * a.split)), block(256 * ks);
    const auto go = [&](auto *kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a, p, s); };
    const auto run = [&](auto turn, auto *d) {
        using T = std::remove_pointer_t<decltype(d)>;
        constexpr bool TURN = decltype(turn)::value;
        if constexpr (!TURN) { // (Gram matrices of large tiles are computed from X by rows)
            if (big) {
                if (ks == 2) go(k_gemm<128, 128, 2, 2, false, T>);
                else go(k_gemm<128, 128, 1, 2, false, T>);
                if (shared) hipLaunchKernelGGL((k_join<128, T>), dim3((unsigned)shared * 4), dim3(256), 0, st, a, p, s);
                return;
            }
        }
        if constexpr (!TURN) {
            if (ks == 4) return go(k_gemm<64, 64, 4, 2, false, T>);
        }
        if (deep) go(k_gemm<64, 64, 2, 4, TURN, T>);
        else if (ks == 2) go(k_gemm<64, 64, 2, 2, TURN, T>);
        else go(k_gemm<64, 64, 1, 2, TURN, T>);
    };
    if (turn) {
        run(std::true_type(), (float *)nullptr);
        if (a.poly) hipLaunchKernelGGL(k_join_poly, dim3((unsigned)groups), dim3(256), 0, st, a);
        else if (shared) hipLaunchKernelGGL((k_join<64, float>), dim3((unsigned)groups), dim3(256), 0, st, a, p, s);
    }
    else if (a.D) run(std::false_type(), (float *)nullptr);
    else by_type(dtype, [&](auto *d) { run(std::false_type(), d); });
}

bool shape_ok(int count, int rows, int cols, int dtype, int steps)
{
    return count >= 0 && rows >= 1 && cols >= 1 && rows <= AZ_MUON_MAX_DIM && cols <= AZ_MUON_MAX_DIM &&
           (long long)rows * cols <= AZ_MUON_MAX_CELLS && dtype >= AZ_F32 && dtype <= AZ_F16 && steps >= 1 && steps <= AZ_MUON_MAX_STEPS;
}

// Matrices that one workgroup holds in registers (128 of them per lane at most)
bool is_small(const Shape &s) { return (s.m <= 32 && s.n <= 2048) || (s.m <= 64 && s.n <= 768); }

int run_small(int batch, const Shape &s, int dtype, int steps, const Ptrs &p, hipStream_t st)
{
    const int nt = (s.n + 255) / 256;
    by_type(dtype, [&](auto *d) {
        using T = std::remove_pointer_t<decltype(d)>;
        const auto go = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3(batch), dim3(64 * SMALL_WAVES), 0, st, p, s, steps); };
        if (s.m <= 32) {
            if (nt <= 1) go(k_small<1, 1, T>);
            else if (nt <= 2) go(k_small<1, 2, T>);
            else if (nt <= 4) go(k_small<1, 4, T>);
            else go(k_small<1, 8, T>);
        } else {
            if (nt <= 1) go(k_small<2, 1, T>);
            else if (nt <= 2) go(k_small<2, 2, T>);
            else go(k_small<2, 3, T>);
        }
    });
    return launch_ok();
}

int run_batch(int batch, Shape s, int dtype, int steps, const Ptrs &p, char *work, hipStream_t st)
{
    const Plan pl = plan_of(s, batch);
    double *sums = (double *)work;
    float *parts_at = (float *)(work + pl.sums);
    char *XT = work + pl.sums + pl.parts, *YT = XT + batch * pl.x, *X = YT + batch * pl.x;
    char *mm[5];
    for (int i = 0; i < 5; i++) mm[i] = X + batch * pl.x + i * batch * pl.mm;
    // Transposing LDS reads are half as fast as plain ones.  That does not matter where loads are waited for, but a Gram
    // matrix of large tiles is bound by LDS with them: there X is kept by rows as well (4096 x 4096 4.89 -> 4.55 ms,
    // 2 x 2048 x 4096 2.34 -> 2.23 ms, 8 x 1024 x 1024 0.78 -> 0.80 ms).
    const bool by_rows = s.mp % 128 == 0 && (long long)(s.mp / 128) * (s.mp / 128 + 1) / 2 * batch >= BIG_TILES;
    if (!by_rows) X = nullptr;
    // workgroups per matrix: two pieces for each wavefront, up to what their joining costs
    const long long parts_l = ((long long)s.rows * ((s.cols + 255) / 256) + 7) / 8;
    const int parts = (int)(parts_l > NORM_PARTS ? NORM_PARTS : parts_l);
    const int rp = s.tall ? s.np : s.mp, cp = s.tall ? s.mp : s.np; // padded rows and columns of G
    by_type(dtype, [&](auto *d) {
        using T = std::remove_pointer_t<decltype(d)>;
        hipLaunchKernelGGL((k_norm<T>), dim3(parts, batch), dim3(256), 0, st, p, s, parts, sums);
        hipLaunchKernelGGL((k_split<T>), dim3((cp + 63) / 64, (rp + 63) / 64, batch), dim3(256), 0, st, p, s, parts, (const double *)sums, XT, X);
    });
    const auto two = [](int e) { return ldexpf(1.f, e); };
    const int pm = s.mp * 4;
    // a symmetric m x m product of two packed ones, 2^ex * 2^ey in the accumulator, stored with 2^eo
    const auto square = [&](const char *x, int ex, const char *y, int ey, char *out, int eo, float f = 1.f, const char *E = nullptr,
                            float beta = 0.f, float gamma = 0.f, const char *x2 = nullptr, const char *y2 = nullptr, char *out2 = nullptr) {
        Gemm g = {};
        g.A = x; g.B = y;
        g.sA = g.sB = g.sE = g.sD = pl.mm;
        g.pitchA = g.pitchB = g.pitchD = pm;
        g.K = s.mp;
        g.symmetric = 1;
        g.alpha = f * two(eo - ex - ey);
        g.E = E; g.beta = beta; g.gamma = gamma;
        g.D = out;
        g.A2 = x2; g.B2 = y2; g.D2 = out2;
        g.parts = parts_at;
        gemm(g, s.mp, s.mp, false, batch, dtype, p, s, st);
    };
    // Steps per group.  float32 results take every step on X (the error stays at or below that of float32 products).
    // Results of 16 bits (half a step: 2^-9, 2^-12) have room for three, which pay as soon as X is wider than high: of five
    // steps' 27.5 m^3 products at n = 1.5 m 23 are left, of 65 at n = 4 m 38.
    // Up to 64 rows a step is three launches, whatever it computes: the Gram matrix, its joining with Q, the product.
    const bool at_once = s.mp == 64 && batch <= FEW_TILES;
    const int group = !at_once && dtype != AZ_F32 && 2 * s.n >= 3 * s.m ? 3 : 1;
    for (int left = steps; left > 0;) {
        // (the odd ones first: the longer groups start from the better conditioned matrix)
        const int k = left > group ? (left % group ? left % group : group) : left;
        char *A = mm[0], *T = mm[1], *Q = mm[2], *W = mm[3], *V = mm[4];
        {
            Gemm g = {};
            g.A = g.B = by_rows ? X : XT;
            g.sA = g.sB = pl.x;
            g.pitchA = g.pitchB = by_rows ? s.np * 4 : pm;
            g.K = s.np;
            g.symmetric = 1;
            g.alpha = two(EXP_A - 2 * EXP_X);
            g.sD = pl.mm;
            g.pitchD = pm;
            g.poly = at_once;
            g.D = at_once ? W : A;
            g.parts = parts_at;
            gemm(g, s.mp, s.mp, !by_rows, batch, dtype, p, s, st);
        }
        const auto poly = [&](char *out) { // a I + b A + c A^2
            square(A, EXP_A, A, EXP_A, out, EXP_Q, NS_C, A, NS_B * two(EXP_Q - EXP_A), NS_A * two(EXP_Q));
        };
        // W, V: Q of the group's latest steps; the product of all of them ends in `total`
        if (!at_once) poly(W);
        const char *total = W;
        if (k > 1) {
            square(A, EXP_A, W, EXP_Q, T, EXP_A);
            square(T, EXP_A, W, EXP_Q, A, EXP_A);
            poly(V);
            if (k == 2) {
                square(V, EXP_Q, W, EXP_Q, Q, EXP_Q);
                total = Q;
            } else { // Q = V W and T = A V do not wait for each other
                static_assert(EXP_Q - 2 * EXP_Q == EXP_A - EXP_A - EXP_Q, "one factor for both");
                square(V, EXP_Q, W, EXP_Q, Q, EXP_Q, 1.f, nullptr, 0.f, 0.f, A, V, T);
                square(T, EXP_A, V, EXP_Q, A, EXP_A);
                poly(W);
                square(W, EXP_Q, Q, EXP_Q, T, EXP_Q);
                total = T;
            }
        }
        left -= k;
        Gemm g = {}; // X <- Q X, by columns
        g.A = total; g.B = XT;
        g.sA = pl.mm; g.sB = pl.x;
        g.pitchA = g.pitchB = pm;
        g.K = s.mp;
        g.alpha = two((left ? EXP_X : 0) - EXP_Q - EXP_X);
        g.parts = parts_at;
        if (left) {
            g.sD = pl.x;
            g.D = YT;
            g.pitchD = pm;
            g.M = X; // (not read by this product)
            g.pitchM = s.np * 4;
        }
        gemm(g, s.mp, s.np, false, batch, dtype, p, s, st);
        char *t = XT;
        XT = YT;
        YT = t;
    }
    return launch_ok();
}

// Matrices per launch: a workspace of 1 GiB at most (matrices that large fill the chip one by one)
int batch_of(const Shape &s, int count)
{
    long long most = MAX_BATCH;
    if (!is_small(s)) {
        const Plan one = plan_of(s, 1);
        const long long fit = (long long)((((size_t)1 << 30) - one.parts) / (one.total - one.parts));
        most = fit < 1 ? 1 : fit < most ? fit : most;
    }
    return (int)(count < most ? count : most);
}

// whether n addresses are evenly spaced
bool spaced(const void *const *p, int n)
{
    for (int i = 2; i < n; i++)
        if ((const char *)p[i] - (const char *)p[i - 1] != (const char *)p[1] - (const char *)p[0]) return false;
    return true;
}

} // namespace

extern "C" {

long long az_muon_work(int count, int rows, int cols)
{
    if (!shape_ok(count, rows, cols, AZ_F32, 1)) return -1;
    if (count == 0) return 0;
    const Shape s = shape_of(rows, cols, count);
    return is_small(s) ? 0 : (long long)plan_of(s, batch_of(s, count)).total;
}

int az_muon_orthogonalise(int count, int rows, int cols, const void *const *d_in, long long ld_in, void *const *d_out,
                          long long ld_out, int dtype, int steps, void *d_work, void *stream)
{
    if (!shape_ok(count, rows, cols, dtype, steps) || ld_in < cols || ld_out < cols) return AZ_ERR_ARG;
    if (count == 0) return AZ_OK;
    if (!d_in || !d_out) return AZ_ERR_ARG;
    for (int i = 0; i < count; i++)
        if (!d_in[i] || !d_out[i]) return AZ_ERR_ARG;
    Shape s = shape_of(rows, cols, count);
    s.ld_in = ld_in;
    s.ld_out = ld_out;
    const bool small = is_small(s);
    if (!small && (!d_work || (uintptr_t)d_work % 16)) return AZ_ERR_ARG;
    const int batch = batch_of(s, count);
    for (int at = 0; at < count;) {
        int n = count - at < batch ? count - at : batch;
        Ptrs p = {};
        p.even = spaced(d_in + at, n) && spaced(d_out + at, n);
        if (!p.even && n > MAX_TABLE) n = MAX_TABLE;
        if (p.even) {
            p.in0 = (const char *)d_in[at];
            p.out0 = (char *)d_out[at];
            p.in_step = n > 1 ? (const char *)d_in[at + 1] - p.in0 : 0;
            p.out_step = n > 1 ? (char *)d_out[at + 1] - p.out0 : 0;
        } else {
            for (int i = 0; i < n; i++) {
                p.in_at[i] = d_in[at + i];
                p.out_at[i] = d_out[at + i];
            }
        }
        const int rc = small ? run_small(n, s, dtype, steps, p, (hipStream_t)stream) : run_batch(n, s, dtype, steps, p, (char *)d_work, (hipStream_t)stream);
        if (rc != AZ_OK) return rc;
        at += n;
    }
    return AZ_OK;
}

} // extern "C"
