// Operators of a policy row (gfx950): log-probabilities of given moves, entropy and the best alternatives over the
// legal moves, with their gradient; and the trainer's loss (src/train.py: KLDivLoss(batchmean) + MSELoss) with its
// gradients.  Everything follows from three numbers of a row x over its legal set L,
//   M = max x_j,   S = sum e^(x_j - M),   U = sum e^(x_j - M) (x_j - M)      (j in L)
//   log p_j = x_j - M - log S,   H = log S - U / S,
// held in 32 bits whatever the logits' type; a row whose legal set is empty (or holds nothing but -inf) has S = 0.
//
// Bound by HBM: a cell is read once, and the operators do 6 to 12 operations on it.
//   rows up to SHORT_MAX actions  one wavefront per row, the row in registers (lane l holds cells l, l + 64, ...),
//                                 so that one pass over memory serves the maximum, the sums and the gradients;
//   longer rows                   one wavefront per chunk of a row; partial (M, S, U) per chunk in a workspace,
//                                 joined by the launch that needs them.
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/azmcts.h"

namespace {

constexpr int WAVES = 4;                 // wavefronts per workgroup
constexpr int SHORT_MAX = 1024;          // longest row held in registers (16 cells per lane)
constexpr int MAX_ACTIONS = 1 << 24;
constexpr int LONG_R = 16;               // cells per lane and step of a long row
constexpr int LONG_STEP = 64 * LONG_R;
constexpr int MAX_CHUNKS = 256;          // chunks per row
// Workgroups of a launch over `units` wavefronts' work; more work per wavefront comes by striding over the grid.  Eight
// workgroups per CU fill it (8 x 4 wavefronts), sixteen do better where memory is the bound: 262144 x 225 loss 165 -> 149 us
// (4.3 -> 4.75 TB/s; the rows of a wavefront are then further apart than a multiple of the memory's interleaving).
constexpr int GRID_MAX = 256 * 16;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NINF = -INFINITY;

struct bf16_t { uint16_t u; };
struct f16_t { _Float16 h; };

__device__ __forceinline__ float get(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float get(const bf16_t *p, size_t i) { return __uint_as_float((uint32_t)p[i].u << 16); }
__device__ __forceinline__ float get(const f16_t *p, size_t i) { return (float)p[i].h; }
__device__ __forceinline__ void put(float *p, size_t i, float v) { p[i] = v; }
__device__ __forceinline__ void put(bf16_t *p, size_t i, float v)
{
    // round to nearest even; a NaN stays one
    const uint32_t b = __float_as_uint(v);
    p[i].u = v != v ? (uint16_t)0x7fc0 : (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void put(f16_t *p, size_t i, float v) { p[i].h = (_Float16)v; }

// e^d for d <= 0 with the hardware's 2^x; |d| log2(e) is rounded once, so the relative error grows with |d| while
// the value falls as e^d: what reaches a sum of probabilities stays below 2^-22
__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

// the value of another lane of the wavefront (0 where the pattern names none), as an operand of the instruction using it
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __uint_as_float(dpp<CTRL>(__float_as_uint(v))); }
__device__ __forceinline__ float lane_of(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
__device__ __forceinline__ float wave_sum(float v)
{
    v += dpp<0x111>(v); // row_shr 1, 2, 4, 8: lane 15 of each row of 16 holds the row's sum
    v += dpp<0x112>(v);
    v += dpp<0x114>(v);
    v += dpp<0x118>(v);
    v += dpp<0x142>(v); // lane 15 / 47 to the next row, lane 31 to the upper half: lane 63 holds all
    v += dpp<0x143>(v);
    return lane_of(v, 63);
}
// unsigned numbers in the order of the floats (0 is below all of them; NaN counts as -inf, -0 as 0)
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t b = __float_as_uint(fmaxf(v, NINF) + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t k) { return __uint_as_float(k ^ ((uint32_t)(~(int32_t)k >> 31) | 0x80000000u)); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = max(v, dpp<0x111>(v));
    v = max(v, dpp<0x112>(v));
    v = max(v, dpp<0x114>(v));
    v = max(v, dpp<0x118>(v));
    v = max(v, dpp<0x142>(v));
    v = max(v, dpp<0x143>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max(float v) { return float_of(wave_max(order_of(v))); } // NaN is ignored
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// the wavefront's number, known to be the same in all lanes: what depends on it alone (a row's address) costs no vector
// instruction
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

struct Rows {
    const void *x;          // logits [n][ld]
    long long ld;
    const float *board;     // [n][2][A] occupied cells of both players, or NULL
    const uint8_t *legal;   // [n][ldl], or NULL
    long long ldl;
    int n, A;
};

__device__ __forceinline__ bool legal_at(const Rows &a, size_t row, int j)
{
    if (a.board) {
        const float *b = a.board + row * 2 * (size_t)a.A;
        return b[j] == 0.f && b[(size_t)a.A + j] == 0.f;
    }
    return a.legal ? a.legal[row * (size_t)a.ldl + j] != 0 : true;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(bf16_t v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float as_float(f16_t v) { return (float)v.h; }

// The row's cells of this lane, -inf where the mask or the row's end leaves nothing (a select: what stands in a masked
// place is never computed with).  The logits are asked for before the mask, so that the row waits for memory once.
// q: numbers that go with the cells, 0 in those places (a legal cell may hold -inf too, and keeps its number).
template <class T, int R> __device__ __forceinline__ void load_row(const Rows &a, size_t row, int lane, float (&x)[R], float *q = nullptr)
{
    const T *p = (const T *)a.x + row * (size_t)a.ld;
    T raw[R];
    bool ok[R];
#pragma unroll
    for (int r = 0; r < R; r++) raw[r] = p[min(r * 64 + lane, a.A - 1)];
    if (a.board) {
        const float *b = a.board + row * 2 * (size_t)a.A;
        float b0[R], b1[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int j = min(r * 64 + lane, a.A - 1);
            b0[r] = b[j];
            b1[r] = b[a.A + j];
        }
#pragma unroll
        for (int r = 0; r < R; r++) ok[r] = b0[r] == 0.f && b1[r] == 0.f;
    } else if (a.legal) {
        const uint8_t *q = a.legal + row * (size_t)a.ldl;
        uint8_t l[R];
#pragma unroll
        for (int r = 0; r < R; r++) l[r] = q[min(r * 64 + lane, a.A - 1)];
#pragma unroll
        for (int r = 0; r < R; r++) ok[r] = l[r] != 0;
    } else {
#pragma unroll
        for (int r = 0; r < R; r++) ok[r] = true;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool in = ok[r] && r * 64 + lane < a.A;
        x[r] = in ? as_float(raw[r]) : NINF;
        if (q) q[r] = in ? q[r] : 0.f;
    }
}

struct Stats { float M, logS, H; bool live; };

// e^(x - M) and x - M of a cell, 0 and a finite number for a cell of -inf.  M must not be -inf.
__device__ __forceinline__ float term(float x, float M, float &d)
{
    const float t = x - M;
    d = fmaxf(t, -FLT_MAX); // (what multiplies it is 0 there)
    return exp_neg(t);
}

// M, log S and the entropy of a row in registers
template <int R> __device__ __forceinline__ Stats row_stats(const float (&x)[R])
{
    float m = x[0];
#pragma unroll
    for (int r = 1; r < R; r++) m = fmaxf(m, x[r]);
    Stats t;
    t.M = wave_max(m);
    const float M = t.M == NINF ? 0.f : t.M;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int r = 0; r < R; r++) {
        float d;
        const float e = term(x[r], M, d);
        s += e;
        u = fmaf(e, d, u);
    }
    s = wave_sum(s);
    u = wave_sum(u);
    t.live = s != 0.f; // (a NaN cell makes s NaN: the row is live and all of it is NaN)
    t.M = t.live && t.M == NINF ? NAN : t.M; // (legal cells that are all NaN)
    t.logS = t.live ? logf(s) : 0.f;
    t.H = t.live ? t.logS - u / s : 0.f;
    return t;
}

// ---- the sorted list of a wavefront: lane t holds the t-th best value and its index
struct Best { float v; int i; };

__device__ __forceinline__ void best_insert(Best &b, float v, int i, int lane) // v, i uniform; equal values stay in front
{
    const int pos = __popcll(__ballot(b.v >= v));
    const float uv = dpp<0x138>(b.v); // from the lane below
    const int ui = (int)dpp<0x138>((uint32_t)b.i);
    b.v = lane < pos ? b.v : lane == pos ? v : uv;
    b.i = lane < pos ? b.i : lane == pos ? i : ui;
}

// The cells of a step, whose indices (first + 64 r + lane) all come after those already listed.  Of many candidates only
// those not below the k-th largest of the 64 lane maxima can be among the k best, few more than k as a rule (the bound is
// found to 16 bits, from below); those are put into the list one by one, in the order of their indices.
template <int R> __device__ __forceinline__ void best_offer(Best &b, const float (&x)[R], int first, int k, int lane)
{
    float limit = lane_of(b.v, k - 1);
    float top = x[0]; // (NaN is ignored by fmaxf, and never above the limit)
#pragma unroll
    for (int r = 1; r < R; r++) top = fmaxf(top, x[r]);
    const unsigned long long some = __ballot(top > limit);
    if (!some) return;
    float least = NINF;
    if (__popcll(some) > k) {
        const uint32_t key = order_of(top);
        uint32_t bound = 0;
        for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
            if (__popcll(__ballot(key >= (bound | bit))) >= k) bound |= bit;
        least = float_of(bound);
        if (!(least > NINF)) least = NINF; // (a bound below every number is no number)
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        unsigned long long todo = __ballot(x[r] > limit && x[r] >= least);
        while (todo) {
            const int l = __ffsll(todo) - 1;
            best_insert(b, lane_of(x[r], l), first + r * 64 + l, lane);
            limit = lane_of(b.v, k - 1);
            todo &= todo - 1;
            todo &= __ballot(x[r] > limit);
        }
    }
}

struct ScoreOut {
    const void *moves;      // [n][m] int32 or int64
    int move_bytes, m, top;
    float *logp;            // [n][m]
    float *entropy;         // [n]
    float *top_logp;        // [n][top]
    int *top_moves;         // [n][top]
    float *stats;           // [n][2]: M and log S (-inf and 0 for an empty row), for the gradient; or NULL
    unsigned long long *bits; // [n][words]: the legal cells of a short row, for the gradient; or NULL
};

__device__ __forceinline__ long long move_at(const void *moves, int bytes, size_t i)
{
    return bytes == 8 ? ((const long long *)moves)[i] : (long long)((const int *)moves)[i];
}

// one wavefront per row; k rounds of "largest cell left" (cost independent of the data, unlike insertion)
template <class T, int R> __global__ __launch_bounds__(64 * WAVES) void k_score(Rows a, ScoreOut o)
{
    const int lane = threadIdx.x & 63;
    const int words = (a.A + 63) / 64;
    for (long long row = (long long)blockIdx.x * WAVES + wave_of(); row < a.n; row += (long long)gridDim.x * WAVES) {
        float x[R];
        const long long mv = lane < o.m ? move_at(o.moves, o.move_bytes, (size_t)row * o.m + lane) : -1;
        load_row<T, R>(a, row, lane, x);
        if (o.bits) { // lane r stores the mask of register r
            unsigned long long mine = 0;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const unsigned long long w = __ballot(x[r] != NINF);
                mine = lane == r ? w : mine;
            }
            if (lane < words) o.bits[(size_t)row * words + lane] = mine;
        }
        const Stats t = row_stats<R>(x);
        if (lane == 0) {
            if (o.entropy) o.entropy[row] = t.H;
            if (o.stats) {
                o.stats[2 * row] = t.live ? t.M : NINF;
                o.stats[2 * row + 1] = t.logS;
            }
        }
        if (o.m) {
            const int at = mv >= 0 && mv < a.A ? (int)mv : -1;
            float v = NINF;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float c = __shfl(x[r], at & 63);
                v = (at >> 6) == r ? c : v;
            }
            if (lane < o.m)
                o.logp[(size_t)row * o.m + lane] = mv < 0 ? 0.f : mv >= a.A ? NAN : v == NINF ? NINF : v - t.M - t.logS;
        }
        if (o.top) {
            float mine_v = NINF;
            int mine_i = -1;
            for (int k = 0; k < o.top; k++) {
                float v = NINF;
                int br = 0;
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const bool more = x[r] > v;
                    v = more ? x[r] : v;
                    br = more ? r : br;
                }
                const float best = wave_max(v);
                if (best == NINF) break;
                int idx = br * 64 + lane;
                unsigned long long who = __ballot(v == best);
                if (who & (who - 1)) { // equal values in several lanes: the lowest index
                    int low = v == best ? idx : 0x7fffffff;
#pragma unroll
                    for (int s = 32; s; s >>= 1) low = min(low, __shfl_xor(low, s));
                    idx = low;
                } else {
                    idx = __builtin_amdgcn_readlane(idx, __ffsll(who) - 1);
                }
#pragma unroll
                for (int r = 0; r < R; r++) x[r] = r * 64 + lane == idx ? NINF : x[r];
                if (lane == k) {
                    mine_v = best;
                    mine_i = idx;
                }
            }
            if (lane < o.top) {
                o.top_logp[(size_t)row * o.top + lane] = mine_i < 0 ? NINF : mine_v - t.M - t.logS;
                o.top_moves[(size_t)row * o.top + lane] = mine_i;
            }
        }
    }
}

struct ScoreGrad {
    const void *moves;
    int move_bytes, m;
    const float *g_logp;    // [n][m] or NULL
    const float *g_entropy; // [n] or NULL
    const float *entropy, *stats;
    const unsigned long long *bits; // or NULL: the mask is read again
    void *dx;               // [n][A], in the logits' type
};

// dx_j = sum_i g_i ([j = move_i] - p_j) - gH p_j (log p_j + H); a move that is none, out of range or illegal has no
// gradient, masked cells and empty rows get zero.  Moves given twice add up in their order.
template <class T, int R> __global__ __launch_bounds__(64 * WAVES) void k_score_grad(Rows a, ScoreGrad o)
{
    const int lane = threadIdx.x & 63;
    const int words = (a.A + 63) / 64;
    for (long long row = (long long)blockIdx.x * WAVES + wave_of(); row < a.n; row += (long long)gridDim.x * WAVES) {
        // everything the row needs is asked for before anything is waited for
        float x[R];
        const bool given = o.m && o.g_logp;
        const long long mv = given && lane < o.m ? move_at(o.moves, o.move_bytes, (size_t)row * o.m + lane) : -1;
        const float up = given && lane < o.m ? o.g_logp[(size_t)row * o.m + lane] : 0.f;
        const float M = o.stats[2 * row], logS = o.stats[2 * row + 1];
        const float gH = o.g_entropy ? o.g_entropy[row] : 0.f;
        const float H = o.g_entropy ? o.entropy[row] : 0.f;
        if (o.bits) {
            Rows plain = a;
            plain.board = nullptr;
            plain.legal = nullptr;
            unsigned long long w[R];
#pragma unroll
            for (int r = 0; r < R; r++) w[r] = o.bits[(size_t)row * words + min(r, words - 1)];
            load_row<T, R>(plain, row, lane, x);
#pragma unroll
            for (int r = 0; r < R; r++) x[r] = (w[r] >> lane) & 1 ? x[r] : NINF;
        } else {
            load_row<T, R>(a, row, lane, x);
        }
        const bool live = !(M == NINF);
        float g = 0.f;
        int at = -1;
        if (given) {
            at = mv >= 0 && mv < a.A ? (int)mv : -1;
            float v = NINF;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float c = __shfl(x[r], at & 63);
                v = (at >> 6) == r ? c : v;
            }
            at = v == NINF ? -1 : at;
            g = at >= 0 ? up : 0.f;
        }
        const float G = given ? wave_sum(g) : 0.f;
        float d[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float lp = x[r] - M - logS;
            const float p = exp_neg(lp);
            const float ent = p == 0.f ? 0.f : gH * p * (lp + H);
            d[r] = x[r] == NINF || !live ? 0.f : -p * G - ent;
        }
        if (given && live) {
            for (int i = 0; i < o.m; i++) {
                const int j = __builtin_amdgcn_readlane(at, i);
                const float gi = lane_of(g, i);
#pragma unroll
                for (int r = 0; r < R; r++) d[r] += r * 64 + lane == j ? gi : 0.f;
            }
        }
        T *out = (T *)o.dx + (size_t)row * a.A;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (r * 64 + lane < a.A) put(out, r * 64 + lane, d[r]);
    }
}

struct Loss {
    const void *value;      // [n], type of the logits or float32
    int value_f32;
    const float *pi;        // [n][A]
    const float *target;    // [n]
    float inv_n;
    const float *scale;     // device scalar the gradients are multiplied by, or NULL
    int only_if_scaled;     // return at once when *scale == 1 (the gradients of an earlier call stand)
    double *part;           // [blocks][2] partial sums of the policy and the value loss, or NULL
    void *dx, *dv;          // [n][A], [n], or NULL
};

// log pi, finite for 0 (which multiplies it); NaN for a negative one
__device__ __forceinline__ float log_of(float pi) { return pi == 0.f ? 0.f : __logf(pi); }

// pi (log pi - d) for d = x - M: 0 without a target, +inf for a target where the difference is -inf
__device__ __forceinline__ float miss_of(float pi, float d) { return pi * (pi == 0.f ? 0.f : __logf(pi) - d); }

// the gradient of a cell, e = e^(x - M) and inv = sum pi / S: 0 where the mask leaves nothing, -pi for a target at -inf
__device__ __forceinline__ float slope_of(float x, float e, float inv, float pi, float f)
{
    const float g = (x == NINF ? 0.f : e * inv) - pi;
    return x == NINF && pi == 0.f ? 0.f : g * f;
}

// sums of a workgroup's wavefronts in wavefront order
template <int W> __device__ __forceinline__ void block_part(double p, double v, double *out)
{
    __shared__ double s_p[W], s_v[W];
    const int wave = threadIdx.x >> 6;
    p = wave_sum(p);
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) {
        s_p[wave] = p;
        s_v[wave] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < W; w++) {
            p += s_p[w];
            v += s_v[w];
        }
        out[0] = p;
        out[1] = v;
    }
}

// the value head's part, one thread per row; returns the thread's sum of (v - r)^2
template <class T> __device__ __forceinline__ double value_part(const Rows &a, const Loss &o, float scale)
{
    double sum = 0.;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < a.n; i += (long long)gridDim.x * blockDim.x) {
        const float v = o.value_f32 ? ((const float *)o.value)[i] : get((const T *)o.value, i);
        const float d = v - o.target[i];
        sum += (double)d * d;
        if (o.dv) {
            const float g = 2.f * d * o.inv_n * scale;
            if (o.value_f32) ((float *)o.dv)[i] = g;
            else put((T *)o.dv, i, g);
        }
    }
    return sum;
}

template <class T, int R> __global__ __launch_bounds__(64 * WAVES) void k_loss(Rows a, Loss o)
{
    const float scale = o.scale ? *o.scale : 1.f;
    if (o.only_if_scaled && scale == 1.f) return;
    const int lane = threadIdx.x & 63;
    double sum = 0.;
    const float f = o.inv_n * scale;
    for (long long row = (long long)blockIdx.x * WAVES + wave_of(); row < a.n; row += (long long)gridDim.x * WAVES) {
        const float *pi = o.pi + (size_t)row * a.A;
        float x[R], q[R];
#pragma unroll
        for (int r = 0; r < R; r++) q[r] = pi[min(r * 64 + lane, a.A - 1)];
        load_row<T, R>(a, row, lane, x, q); // (masked places and cells past the row's end hold no target)
        float m = x[0];
#pragma unroll
        for (int r = 1; r < R; r++) m = fmaxf(m, x[r]);
        m = wave_max(m);
        const float M = m == NINF ? 0.f : m;
        float s = 0.f, w = 0.f, l = 0.f, e[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float d = x[r] - M;
            e[r] = exp_neg(d);
            s += e[r];
            w += q[r];
            l += miss_of(q[r], d);
        }
        s = wave_sum(s);
        w = wave_sum(w);
        const bool live = s != 0.f;
        if (o.part) {
            // sum pi log pi - sum pi (x - M), each lane its share; log S sum pi once
            sum += (double)l;
            if (lane == 0 && live) sum += (double)logf(s) * (double)w;
        }
        if (o.dx) {
            const float inv = live ? w / s : 0.f;
            T *out = (T *)o.dx + (size_t)row * a.A;
#pragma unroll
            for (int r = 0; r < R; r++)
                if (r * 64 + lane < a.A) put(out, r * 64 + lane, slope_of(x[r], e[r], inv, q[r], f));
        }
    }
    const double v = value_part<T>(a, o, scale);
    if (o.part) block_part<WAVES>(sum, v, o.part + 2 * (size_t)blockIdx.x);
}

// the total, and the policy and value parts, from the workgroups' partial sums, added in a fixed order
constexpr int JOIN_WAVES = 16;
__global__ __launch_bounds__(64 * JOIN_WAVES) void k_loss_join(const double *part, int blocks, double inv_n, const float *unless_one, float *loss, float *parts)
{
    if (unless_one && *unless_one == 1.f) return; // (nor have the kernels before written partial sums)
    constexpr int EACH = (GRID_MAX + 64 * JOIN_WAVES - 1) / (64 * JOIN_WAVES);
    double2 in[EACH]; // (all in flight together)
#pragma unroll
    for (int k = 0; k < EACH; k++) in[k] = ((const double2 *)part)[min(k * 64 * JOIN_WAVES + (int)threadIdx.x, blocks - 1)];
    double p = 0., v = 0.;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const bool mine = k * 64 * JOIN_WAVES + (int)threadIdx.x < blocks;
        p += mine ? in[k].x : 0.;
        v += mine ? in[k].y : 0.;
    }
    __shared__ double s_all[2];
    block_part<JOIN_WAVES>(p, v, s_all);
    if (threadIdx.x == 0) {
        loss[0] = (float)((s_all[0] + s_all[1]) * inv_n);
        if (parts) {
            parts[0] = (float)(s_all[0] * inv_n);
            parts[1] = (float)(s_all[1] * inv_n);
        }
    }
}

// ---------------------------------------------------------------- rows longer than SHORT_MAX

struct Chunks { int len, count; }; // cells per chunk (a multiple of LONG_STEP) and chunks per row

// partial numbers of one chunk: M, S, U, and for the loss sum pi, sum pi log pi, sum pi (x - M)
struct Part { float M, S, U, W, E, X; };

struct LongOut {
    Part *part;             // [n][chunks]
    float *list_v;          // [n][chunks][top]
    int *list_i;
    int top;
    const float *pi;        // of the loss
    const float *unless_one; // device scalar: nothing to do when it is 1; or NULL
};

__device__ __forceinline__ void rebase(float &S, float &U, float from, float to) // sums about another maximum
{
    const float d = from - to;
    const float f = S == 0.f ? 0.f : exp_neg(d);
    const float s = S * f;
    U = s == 0.f ? (S != S ? S : 0.f) : U * f + s * d;
    S = s;
}

template <class T, bool LOSS> __global__ __launch_bounds__(64 * WAVES) void k_long_parts(Rows a, Chunks c, LongOut o, long long first)
{
    if (o.unless_one && *o.unless_one == 1.f) return;
    const int lane = threadIdx.x & 63;
    const long long unit = (first + blockIdx.x) * WAVES + wave_of();
    if (unit >= (long long)a.n * c.count) return;
    const long long row = unit / c.count;
    const int chunk = (int)(unit - row * c.count);
    const int begin = chunk * c.len, end = min(a.A, begin + c.len);
    const T *p = (const T *)a.x + (size_t)row * a.ld;
    const float *pi = LOSS ? o.pi + (size_t)row * a.A : nullptr;
    float M = NINF, S = 0.f, U = 0.f, W = 0.f, E = 0.f, X = 0.f; // S, U, W, E, X: this lane's share; M: the wavefront's
    Best best = {NINF, -1};
    for (int j0 = begin; j0 < end; j0 += LONG_STEP) {
        float x[LONG_R], q[LONG_R];
        bool ok[LONG_R];
#pragma unroll
        for (int r = 0; r < LONG_R; r++) x[r] = get(p, min(j0 + r * 64 + lane, end - 1));
        if (LOSS) {
#pragma unroll
            for (int r = 0; r < LONG_R; r++) q[r] = pi[min(j0 + r * 64 + lane, end - 1)];
        }
#pragma unroll
        for (int r = 0; r < LONG_R; r++) ok[r] = legal_at(a, row, min(j0 + r * 64 + lane, end - 1));
        float m = NINF;
#pragma unroll
        for (int r = 0; r < LONG_R; r++) {
            ok[r] = ok[r] && j0 + r * 64 + lane < end;
            x[r] = ok[r] ? x[r] : NINF;
            m = fmaxf(m, x[r]);
        }
        m = wave_max(m);
        if (m > M) {
            if (M != NINF) {
                if (LOSS) X += W == 0.f ? 0.f : W * (M - m);
                rebase(S, U, M, m);
            }
            M = m;
        }
#pragma unroll
        for (int r = 0; r < LONG_R; r++) {
            const float d = x[r] - M;
            const float e = x[r] == NINF ? 0.f : exp_neg(d);
            S += e;
            U += e == 0.f ? 0.f : e * d;
            if (LOSS) {
                const float w = ok[r] ? q[r] : 0.f;
                W += w;
                E += w * log_of(w);
                X += w == 0.f ? 0.f : w * (x[r] == NINF ? NINF : d); // (M is -inf until a cell above it comes)
            }
        }
        if (!LOSS && o.top) best_offer<LONG_R>(best, x, j0, o.top, lane);
    }
    Part out = {M, wave_sum(S), wave_sum(U), wave_sum(W), wave_sum(E), wave_sum(X)};
    if (lane == 0) o.part[unit] = out;
    if (!LOSS && lane < o.top) {
        o.list_v[(size_t)unit * o.top + lane] = best.v;
        o.list_i[(size_t)unit * o.top + lane] = best.i;
    }
}

// the row's numbers from its chunks' (every lane gets them)
__device__ __forceinline__ Part join_parts(const Part *part, int count, int lane)
{
    float m = NINF;
    for (int i = lane; i < count; i += 64) m = fmaxf(m, part[i].M);
    const float M = wave_max(m);
    float S = 0.f, U = 0.f, W = 0.f, E = 0.f, X = 0.f;
    for (int i = lane; i < count; i += 64) {
        Part q = part[i];
        if (q.M == NINF) { // nothing legal, or nothing but NaN
            S += q.S;
            U += q.U;
            W += q.W;
            E += q.E;
            X += q.X;
            continue;
        }
        X += q.X + (q.W == 0.f ? 0.f : q.W * (q.M - M));
        rebase(q.S, q.U, q.M, M);
        S += q.S;
        U += q.U;
        W += q.W;
        E += q.E;
    }
    return Part{M, wave_sum(S), wave_sum(U), wave_sum(W), wave_sum(E), wave_sum(X)};
}

// one workgroup per row: outputs of az_policy_score from the chunks' numbers and lists.  The lists are merged in LDS: a
// lane holds the heads of every 64th list, each round takes the largest head (of equal ones the lowest index)
template <class T> __global__ __launch_bounds__(64 * WAVES) void k_long_score(Rows a, Chunks c, LongOut w, ScoreOut o, long long first)
{
    extern __shared__ float s_list[]; // [chunks][top] values, then indices
    const int lane = threadIdx.x;
    const long long row = first + blockIdx.x;
    const int cells = c.count * o.top;
    int *s_index = (int *)(s_list + cells);
    for (int i = lane; i < cells; i += 64 * WAVES * 4) { // four loads in flight per thread
        float v[4];
        int n[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const size_t at = (size_t)row * cells + min(i + q * 64 * WAVES, cells - 1);
            v[q] = w.list_v[at];
            n[q] = w.list_i[at];
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (i + q * 64 * WAVES < cells) {
                s_list[i + q * 64 * WAVES] = v[q];
                s_index[i + q * 64 * WAVES] = n[q];
            }
    }
    __syncthreads();
    if (lane >= 64) return; // the first wavefront does the rest
    const Part t = join_parts(w.part + (size_t)row * c.count, c.count, lane);
    const bool live = t.S != 0.f;
    const float logS = live ? logf(t.S) : 0.f;
    if (lane == 0) {
        if (o.entropy) o.entropy[row] = live ? logS - t.U / t.S : 0.f;
        if (o.stats) {
            o.stats[2 * row] = live ? (t.M == NINF ? NAN : t.M) : NINF;
            o.stats[2 * row + 1] = logS;
        }
    }
    if (lane < o.m) {
        const long long mv = move_at(o.moves, o.move_bytes, (size_t)row * o.m + lane);
        float r;
        if (mv < 0) r = 0.f;
        else if (mv >= a.A) r = NAN;
        else {
            const float v = legal_at(a, row, (int)mv) ? get((const T *)a.x + (size_t)row * a.ld, (size_t)mv) : NINF;
            r = v == NINF ? NINF : v - t.M - logS;
        }
        o.logp[(size_t)row * o.m + lane] = r;
    }
    if (!o.top) return;
    constexpr int HEADS = MAX_CHUNKS / 64;
    float head[HEADS];
    int place[HEADS]; // where the head stands
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
        const int list = h * 64 + lane;
        head[h] = list < c.count ? s_list[list * o.top] : NINF;
        place[h] = list * o.top;
    }
    float mine_v = NINF;
    int mine_at = -1;
    for (int k = 0; k < o.top; k++) {
        float v = head[0];
        int from = 0;
#pragma unroll
        for (int h = 1; h < HEADS; h++) {
            from = head[h] > v ? h : from; // (lists in the order of their indices: of equal heads the first)
            v = head[h] > v ? head[h] : v;
        }
        const float best = wave_max(v);
        if (best == NINF) break;
        // of the lanes with this value the one whose list comes first holds the lowest index
        int list = v == best ? from * 64 + lane : 0x7fffffff;
        const unsigned long long who = __ballot(v == best);
        if (who & (who - 1)) {
#pragma unroll
            for (int s = 32; s; s >>= 1) list = min(list, __shfl_xor(list, s));
            list = __builtin_amdgcn_readfirstlane(list);
        } else {
            list = __builtin_amdgcn_readlane(list, __ffsll(who) - 1);
        }
        int at = 0;
#pragma unroll
        for (int h = 0; h < HEADS; h++) at = list >> 6 == h ? __builtin_amdgcn_readlane(place[h], list & 63) : at;
        const float after = at + 1 < (list + 1) * o.top ? s_list[at + 1] : NINF; // the list's next head
#pragma unroll
        for (int h = 0; h < HEADS; h++) {
            const bool taken = list == h * 64 + lane;
            head[h] = taken ? after : head[h];
            place[h] += taken ? 1 : 0;
        }
        mine_v = lane == k ? best : mine_v;
        mine_at = lane == k ? at : mine_at;
    }
    if (lane < o.top) {
        o.top_logp[(size_t)row * o.top + lane] = mine_at < 0 ? NINF : mine_v - t.M - logS;
        o.top_moves[(size_t)row * o.top + lane] = mine_at < 0 ? -1 : s_index[mine_at];
    }
}

template <class T> __global__ __launch_bounds__(64 * WAVES) void k_long_score_grad(Rows a, Chunks c, ScoreGrad o, long long first)
{
    const int lane = threadIdx.x & 63;
    const long long unit = (first + blockIdx.x) * WAVES + wave_of();
    if (unit >= (long long)a.n * c.count) return;
    const long long row = unit / c.count;
    const int chunk = (int)(unit - row * c.count);
    const int begin = chunk * c.len, end = min(a.A, begin + c.len);
    const T *p = (const T *)a.x + (size_t)row * a.ld;
    const float M = o.stats[2 * row], logS = o.stats[2 * row + 1];
    const bool live = !(M == NINF);
    float g = 0.f;
    int at = -1;
    if (o.m && o.g_logp) {
        const long long mv = lane < o.m ? move_at(o.moves, o.move_bytes, (size_t)row * o.m + lane) : -1;
        if (mv >= 0 && mv < a.A && legal_at(a, row, (int)mv) && get(p, (size_t)mv) != NINF) {
            at = (int)mv;
            g = o.g_logp[(size_t)row * o.m + lane];
        }
    }
    const float G = o.m && o.g_logp ? wave_sum(g) : 0.f;
    const float gH = o.g_entropy ? o.g_entropy[row] : 0.f;
    const float H = o.g_entropy ? o.entropy[row] : 0.f;
    T *out = (T *)o.dx + (size_t)row * a.A;
    for (int j0 = begin; j0 < end; j0 += LONG_STEP) {
        float x[LONG_R], d[LONG_R];
        bool ok[LONG_R];
#pragma unroll
        for (int r = 0; r < LONG_R; r++) x[r] = get(p, min(j0 + r * 64 + lane, end - 1));
#pragma unroll
        for (int r = 0; r < LONG_R; r++) ok[r] = legal_at(a, row, min(j0 + r * 64 + lane, end - 1));
#pragma unroll
        for (int r = 0; r < LONG_R; r++) {
            const float lp = x[r] - M - logS;
            const float e = exp_neg(lp);
            const float ent = e == 0.f ? 0.f : gH * e * (lp + H);
            d[r] = !ok[r] || x[r] == NINF || !live ? 0.f : -e * G - ent;
        }
        if (o.m && o.g_logp && live) {
            for (int i = 0; i < o.m; i++) {
                const int j = __builtin_amdgcn_readlane(at, i);
                const float gi = lane_of(g, i);
#pragma unroll
                for (int r = 0; r < LONG_R; r++) d[r] += j0 + r * 64 + lane == j ? gi : 0.f;
            }
        }
#pragma unroll
        for (int r = 0; r < LONG_R; r++)
            if (j0 + r * 64 + lane < end) put(out, j0 + r * 64 + lane, d[r]);
    }
}

// the loss of long rows behind k_long_parts: one wavefront per chunk writes its gradients, the first chunk's wavefront
// adds the row's loss  sum pi log pi - sum pi (x - M) + log S sum pi
template <class T> __global__ __launch_bounds__(64 * WAVES) void k_long_loss(Rows a, Chunks c, const Part *part, Loss o)
{
    const float scale = o.scale ? *o.scale : 1.f;
    if (o.only_if_scaled && scale == 1.f) return;
    const int lane = threadIdx.x & 63;
    const float f = o.inv_n * scale;
    double sum = 0.;
    const long long units = (long long)a.n * c.count;
    for (long long unit = (long long)blockIdx.x * WAVES + wave_of(); unit < units; unit += (long long)gridDim.x * WAVES) {
        const long long row = unit / c.count;
        const int chunk = (int)(unit - row * c.count);
        const int begin = chunk * c.len, end = min(a.A, begin + c.len);
        const Part t = join_parts(part + (size_t)row * c.count, c.count, lane);
        const bool live = t.S != 0.f;
        if (chunk == 0 && lane == 0) {
            const float logS = live ? logf(t.S) : 0.f;
            sum += (double)t.E - (double)t.X + (double)logS * (double)t.W;
        }
        if (!o.dx) continue;
        const T *p = (const T *)a.x + (size_t)row * a.ld;
        const float *pi = o.pi + (size_t)row * a.A;
        T *out = (T *)o.dx + (size_t)row * a.A;
        const float inv = live ? t.W / t.S : 0.f;
        for (int j0 = begin; j0 < end; j0 += LONG_STEP) {
            float x[LONG_R], q[LONG_R];
            bool ok[LONG_R];
#pragma unroll
            for (int r = 0; r < LONG_R; r++) {
                x[r] = get(p, min(j0 + r * 64 + lane, end - 1));
                q[r] = pi[min(j0 + r * 64 + lane, end - 1)];
            }
#pragma unroll
            for (int r = 0; r < LONG_R; r++) ok[r] = legal_at(a, row, min(j0 + r * 64 + lane, end - 1));
#pragma unroll
            for (int r = 0; r < LONG_R; r++)
                if (j0 + r * 64 + lane < end)
                    put(out, j0 + r * 64 + lane, ok[r] ? slope_of(x[r], exp_neg(x[r] - t.M), inv, q[r], f) : 0.f);
        }
    }
    const double v = value_part<T>(a, o, scale);
    if (o.part) block_part<WAVES>(sum, v, o.part + 2 * (size_t)blockIdx.x);
}

// ---------------------------------------------------------------- host side

int launch_ok() { return hipGetLastError() == hipSuccess ? AZ_OK : AZ_ERR_HIP; }

int grid_of(long long units)
{
    const long long b = (units + WAVES - 1) / WAVES;
    return (int)(b < GRID_MAX ? b : GRID_MAX);
}

// A launch counts its threads in 32 bits, so workgroups without end come in several launches: f(first, how many)
constexpr long long LAUNCH_MAX = 1ll << 23;
template <class F> void in_launches(long long groups, F f)
{
    for (long long first = 0; first < groups; first += LAUNCH_MAX)
        f(first, dim3((unsigned)(groups - first < LAUNCH_MAX ? groups - first : LAUNCH_MAX)));
}

// Chunks of a long row: about 8192 wavefronts over all rows (32 per CU) when the rows alone are fewer, chunks of at least
// one step, at most as many as one wavefront can merge (their lists in 32 KB of LDS).
Chunks chunks_of(int n, int A, int top)
{
    long long want = n > 0 ? (8192ll + n - 1) / n : 1;
    const long long most = (A + LONG_STEP - 1) / LONG_STEP;
    const long long fit = top > 16 ? MAX_CHUNKS / 2 : MAX_CHUNKS;
    if (want > most) want = most;
    if (want > fit) want = fit;
    if (want < 1) want = 1;
    const long long len = ((A + want - 1) / want + LONG_STEP - 1) / LONG_STEP * LONG_STEP;
    return Chunks{(int)len, (int)((A + len - 1) / len)};
}

// workgroups with a wavefront for each chunk
long long groups_of(int n, const Chunks &c) { return ((long long)n * c.count + WAVES - 1) / WAVES; }

bool rows_ok(const Rows &a, int dtype)
{
    return a.n >= 0 && a.A >= 1 && a.A <= MAX_ACTIONS && a.ld >= a.A && dtype >= AZ_F32 && dtype <= AZ_F16 &&
           (a.legal == nullptr || a.ldl >= a.A || a.ldl == 0) && !(a.board && a.legal);
}

size_t long_work(int n, int A, int top)
{
    const Chunks c = chunks_of(n, A, top);
    return (size_t)n * c.count * (sizeof(Part) + 8 * (size_t)top);
}

// calls f with the cell type and the number of cells per lane of a short row
template <class F> void by_type(int dtype, F f)
{
    if (dtype == AZ_F32) f((float *)nullptr);
    else if (dtype == AZ_BF16) f((bf16_t *)nullptr);
    else f((f16_t *)nullptr);
}
template <int R> struct Width { static constexpr int value = R; };
template <class F> void by_width(int A, F f)
{
    const int w = (A + 63) / 64;
    if (w <= 1) f(Width<1>());
    else if (w == 2) f(Width<2>());
    else if (w == 3) f(Width<3>());
    else if (w == 4) f(Width<4>());
    else if (w == 5) f(Width<5>());
    else if (w == 6) f(Width<6>());
    else if (w == 7) f(Width<7>());
    else if (w == 8) f(Width<8>());
    else if (w <= 12) f(Width<12>());
    else f(Width<16>());
}

} // namespace

extern "C" {

long long az_policy_score_work(int n, int actions, int top)
{
    if (n < 0 || actions < 1 || actions > MAX_ACTIONS || top < 0 || top > AZ_POLICY_MAX_TOP) return -1;
    return actions <= SHORT_MAX ? 0 : (long long)long_work(n, actions, top);
}

int az_policy_mask_words(int actions) { return actions >= 1 && actions <= SHORT_MAX ? (actions + 63) / 64 : 0; }

int az_policy_score(int n, int actions, const void *d_logits, int dtype, long long ld, const float *d_board,
                    const unsigned char *d_legal, long long ld_legal, const void *d_moves, int move_bytes, int m, int top,
                    float *d_logp, float *d_entropy, float *d_top_logp, int *d_top_moves, float *d_stats,
                    unsigned long long *d_mask, void *d_work, void *stream)
{
    const Rows a = {d_logits, ld, d_board, d_legal, ld_legal, n, actions};
    if (!rows_ok(a, dtype) || m < 0 || m > AZ_POLICY_MAX_MOVES || top < 0 || top > AZ_POLICY_MAX_TOP) return AZ_ERR_ARG;
    if (m && move_bytes != 4 && move_bytes != 8) return AZ_ERR_ARG;
    if (n == 0) return AZ_OK;
    if (!d_logits || (m && (!d_moves || !d_logp)) || (top && (!d_top_logp || !d_top_moves))) return AZ_ERR_ARG;
    const ScoreOut o = {d_moves, move_bytes, m, top, d_logp, d_entropy, d_top_logp, d_top_moves, d_stats, d_mask};
    const dim3 block(64 * WAVES);
    const hipStream_t st = (hipStream_t)stream;
    if (actions <= SHORT_MAX) {
        by_type(dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            by_width(actions, [&](auto w) {
                hipLaunchKernelGGL((k_score<T, decltype(w)::value>), dim3(grid_of(n)), block, 0, st, a, o);
            });
        });
        return launch_ok();
    }
    if (!d_work || (uintptr_t)d_work % 16) return AZ_ERR_ARG;
    const Chunks c = chunks_of(n, actions, top);
    LongOut w = {};
    w.part = (Part *)d_work;
    w.list_v = (float *)(w.part + (size_t)n * c.count);
    w.list_i = (int *)(w.list_v + (size_t)n * c.count * top);
    w.top = top;
    by_type(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        in_launches(groups_of(n, c), [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((k_long_parts<T, false>), grid, block, 0, st, a, c, w, first);
        });
        in_launches(n, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((k_long_score<T>), grid, block, (size_t)c.count * top * 8, st, a, c, w, o, first);
        });
    });
    return launch_ok();
}

int az_policy_score_grad(int n, int actions, const void *d_logits, int dtype, long long ld, const float *d_board,
                         const unsigned char *d_legal, long long ld_legal, const unsigned long long *d_mask,
                         const void *d_moves, int move_bytes, int m, const float *d_g_logp, const float *d_g_entropy,
                         const float *d_entropy, const float *d_stats, void *d_dlogits, void *stream)
{
    const Rows a = {d_logits, ld, d_board, d_legal, ld_legal, n, actions};
    if (!rows_ok(a, dtype) || m < 0 || m > AZ_POLICY_MAX_MOVES) return AZ_ERR_ARG;
    if (m && move_bytes != 4 && move_bytes != 8) return AZ_ERR_ARG;
    if (n == 0) return AZ_OK;
    if (!d_logits || !d_stats || !d_dlogits || (m && d_g_logp && !d_moves) || (d_g_entropy && !d_entropy)) return AZ_ERR_ARG;
    if (d_mask && actions > SHORT_MAX) return AZ_ERR_ARG;
    const ScoreGrad o = {d_moves, move_bytes, m, d_g_logp, d_g_entropy, d_entropy, d_stats, d_mask, d_dlogits};
    const dim3 block(64 * WAVES);
    const hipStream_t st = (hipStream_t)stream;
    const Chunks c = chunks_of(n, actions, 0);
    by_type(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (actions <= SHORT_MAX)
            by_width(actions, [&](auto w) {
                hipLaunchKernelGGL((k_score_grad<T, decltype(w)::value>), dim3(grid_of(n)), block, 0, st, a, o);
            });
        else
            in_launches(groups_of(n, c), [&](long long first, dim3 grid) {
                hipLaunchKernelGGL((k_long_score_grad<T>), grid, block, 0, st, a, c, o, first);
            });
    });
    return launch_ok();
}

// the workspace: partial sums of the workgroups, then the chunks' numbers of long rows
long long az_policy_loss_work(int n, int actions)
{
    if (n < 0 || actions < 1 || actions > MAX_ACTIONS) return -1;
    return (long long)(GRID_MAX * 2 * sizeof(double)) + (actions <= SHORT_MAX ? 0 : (long long)long_work(n, actions, 0));
}

int az_policy_loss(int n, int actions, const void *d_logits, int dtype, long long ld, const float *d_board,
                   const unsigned char *d_legal, long long ld_legal, const void *d_value, int value_f32, const float *d_pi,
                   const float *d_r, const float *d_scale, int only_if_scaled, float *d_loss, float *d_parts, void *d_dlogits,
                   void *d_dvalue, void *d_work, void *stream)
{
    const Rows a = {d_logits, ld, d_board, d_legal, ld_legal, n, actions};
    if (!rows_ok(a, dtype) || n < 1) return AZ_ERR_ARG;
    if ((d_loss || actions > SHORT_MAX) && (!d_work || (uintptr_t)d_work % 16)) return AZ_ERR_ARG;
    if (!d_logits || !d_value || !d_pi || !d_r || (only_if_scaled && !d_scale) || (d_parts && !d_loss)) return AZ_ERR_ARG;
    Loss o = {d_value, value_f32, d_pi, d_r, 1.f / (float)n, d_scale, only_if_scaled, d_loss ? (double *)d_work : nullptr, d_dlogits, d_dvalue};
    const dim3 block(64 * WAVES);
    const hipStream_t st = (hipStream_t)stream;
    int blocks = 0;
    if (actions <= SHORT_MAX) {
        blocks = grid_of(n);
        by_type(dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            by_width(actions, [&](auto w) {
                hipLaunchKernelGGL((k_loss<T, decltype(w)::value>), dim3(blocks), block, 0, st, a, o);
            });
        });
    } else {
        const Chunks c = chunks_of(n, actions, 0);
        LongOut w = {};
        w.part = (Part *)((char *)d_work + GRID_MAX * 2 * sizeof(double));
        w.pi = d_pi;
        w.unless_one = only_if_scaled ? d_scale : nullptr;
        blocks = grid_of((long long)n * c.count);
        by_type(dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            in_launches(groups_of(n, c), [&](long long first, dim3 grid) {
                hipLaunchKernelGGL((k_long_parts<T, true>), grid, block, 0, st, a, c, w, first);
            });
            hipLaunchKernelGGL((k_long_loss<T>), dim3(blocks), block, 0, st, a, c, (const Part *)w.part, o);
        });
    }
    if (d_loss) hipLaunchKernelGGL(k_loss_join, dim3(1), dim3(64 * JOIN_WAVES), 0, st, (const double *)d_work, blocks, 1. / n,
                                   only_if_scaled ? d_scale : nullptr, d_loss, d_parts);
    return launch_ok();
}

} // extern "C"
