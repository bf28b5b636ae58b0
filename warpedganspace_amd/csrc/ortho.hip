// Orthogonalised updates: the quintic Newton-Schulz iteration on matrices, alone or between a momentum and a weight update.
//
//   X_0 = X / (|X|_F + eps), on the wide side (m rows, n >= m columns);   A_t = X_t X_t^T,  B_t = a I + b A_t + c A_t^2,  X_{t+1} = B_t X_t
//
// Every A_t and B_t is a polynomial in A_0, so within a PHASE of k iterations only m x m matrices are needed:
//   A_{t+1} = B_t A_t B_t,  Q = B_{t+k-1} ... B_t,  X_{t+k} = Q X_t
// and all of them are symmetric: their products compute the tiles on and under the diagonal and write each twice.
//
// Arithmetic.  The iteration multiplies small singular values by a = 3.44 each time (A's eigenvalues by a^2), and the noise of the products with
// them, so the products keep about fp32's precision (plan_of has the measured distances): an operand is an fp16 pair hi + lo = value * 2^s (22 bits),
// a product lo*hi + hi*lo + hi*hi on the 16-bit matrix cores with fp32 accumulation — 3 / 2 500 of a TFLOP instead of 1 / 157 on the fp32 ones.  Exponents: X from its largest
// entry; A_t, X_t from bounds on their entries (|A_ij| <= max_i |x_i|^2, times the largest |a + b l + c l^2|^2 on the interval that the
// eigenvalues can reach, iteration by iteration); B, Q from the same polynomial's maximum.  16-bit inputs are their own hi part (one product in
// the first Gram matrix, two in its phase's Q X).  Norms are summed in fp64.
#include "wgs_common.h"
#include "../../include/wgs.h"
#include <math.h>
#include <type_traits>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int frag __attribute__((ext_vector_type(4)));      // half8 in storage (vectors of halves are kept one half a register across branches)
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr int MAX_MATS = 24;             // matrices of one launch (they travel as kernel arguments)
constexpr int MAX_STEPS = 16;
constexpr int INFO = 64;                 // floats of an instance's scalars: f0, then sA[t], sX[t]
constexpr int I_SA = 4, I_SX = I_SA + MAX_STEPS + 1;
constexpr int STAT_BLOCKS = 256;         // partial norms of an instance
// Long sums over few 64 x 64 tiles are split over workgroups, at least SPLIT_NK chunks each: the parts go to the workspace, and a second launch adds
// them, in order, and does the epilogue.  (One launch whose last workgroup a tile adds the parts was slower: the fence that makes them visible
// between XCDs writes back a whole L2, some hundred times.)
constexpr int SPLIT_NK = 12, SPLIT_ITEMS = 1024;
constexpr int64_t SPLIT_BYTES = (int64_t)SPLIT_ITEMS * 64 * 64 * 4;
constexpr int BK = 32, ROW = 64;         // K values (bytes) of an LDS row
constexpr int OOB = (int)0x80000000;     // byte offset behind every plane: the load gives zeros

struct Mat {
    const void* in;          // the matrix (orthogonalise) or the gradient (step)
    void* out;               // the result or the weight
    float* momentum;         // step only
    int64_t in_bs, out_bs;   // elements between instances of a batch
    int64_t ws;              // byte offset of instance 0's planes
    int in_rs, out_rs;       // elements between rows
    int M, N, batch, first;  // first: number of instances before this entry
    float step, decay;       // step only: W <- decay W - step O
};
struct Group {
    unsigned char* ws;
    int count, instances;
    int npx, nt, ns;         // planes of X / X^T, buffers of X^T, m x m buffers
    int stat_blocks;
    int dtype, step;         // element type of in / out; a weight update rather than the bare factor
    int64_t info;            // byte offset of the scalars, INFO floats an instance
    int64_t part;            // byte offset of the partial tiles of split sums (0: none)
    Mat mat[MAX_MATS];
};
// dimensions of an entry's planes
struct Dims {
    int m, n, mp, np;        // small / large side, padded to BK
    int64_t szx, szt, szs;   // bytes of one plane of X [m][np], X^T [n][mp], an m x m matrix [m][mp]
};
__host__ __device__ __forceinline__ int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
__host__ __device__ __forceinline__ Dims dims_of(int M, int N) {
    Dims d;
    d.m = M < N ? M : N; d.n = M < N ? N : M;
    d.mp = (int)up(d.m, BK); d.np = (int)up(d.n, BK);
    d.szx = up((int64_t)d.m * d.np * 2, 256); d.szt = up((int64_t)d.n * d.mp * 2, 256); d.szs = up((int64_t)d.m * d.mp * 2, 256);
    return d;
}
__host__ __device__ __forceinline__ int64_t instance_bytes(const Dims& d, int npx, int nt, int ns) {
    return npx * d.szx + (int64_t)nt * npx * d.szt + (int64_t)ns * 2 * d.szs;
}
// Buffers of an instance: 0 = X, 1 / 2 = X^T (the second one where a phase's result is another phase's input), 3.. = m x m
enum { BUF_X = 0, BUF_T0 = 1, BUF_T1 = 2, BUF_S = 3 };
// A matrix of pairs keeps, row by row, 32 hi parts and their 32 lo parts in turn: one cache line holds what a row gives a chunk of the sum.  (As two
// planes, 64 bytes of a row each, the loads fetch half lines: measured half the rate into the LDS.)  A matrix of hi parts alone is plain.
struct Plane { unsigned char* p; int ld, pair; };
__device__ __forceinline__ int row_bytes(const Plane& q) { return q.ld * (q.pair ? 4 : 2); }
__device__ __forceinline__ unsigned char* at_hi(const Plane& q, int r, int k) {      // the lo part: 64 bytes on
    return q.p + (int64_t)r * row_bytes(q) + (q.pair ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
}
__device__ __forceinline__ Plane plane_of(const Group& g, const Mat& a, const Dims& d, int inst, int buf, bool pair = true) {
    unsigned char* p = g.ws + a.ws + inst * instance_bytes(d, g.npx, g.nt, g.ns);
    if (buf == BUF_X) return Plane{p, d.np, pair};
    if (buf < BUF_S) return Plane{p + g.npx * d.szx + (int64_t)(buf - 1) * g.npx * d.szt, d.mp, pair};
    return Plane{p + g.npx * d.szx + (int64_t)g.nt * g.npx * d.szt + (int64_t)(buf - BUF_S) * 2 * d.szs, d.mp, 1};
}
// header of the workspace: partial norms, then the scalars of every instance
struct Part { double ss; float amax; float pad; };
__device__ __forceinline__ Part* parts_of(const Group& g, int inst) { return (Part*)g.ws + (int64_t)inst * g.stat_blocks; }
__device__ __forceinline__ float* info_of(const Group& g, int inst) { return (float*)(g.ws + g.info) + (int64_t)inst * INFO; }
__host__ __device__ __forceinline__ int parts_of_sum(int nk, int most) { const int s = nk / SPLIT_NK; return s < 1 ? 1 : (s < most ? s : most); }
// instance -> its entry (a scalar search over at most MAX_MATS entries)
__device__ __forceinline__ int entry_of(const Group& g, int inst) {
    int e = 0;
    while (e + 1 < g.count && inst >= g.mat[e + 1].first) ++e;
    return e;
}

template <int DT> __device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if (DT == WGS_F32) return ((const float*)p)[i];
    if (DT == WGS_BF16) return (float)((const __bf16*)p)[i];
    return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ float load_as(int dt, const void* p, int64_t i) {
    return dt == WGS_F32 ? load_elem<WGS_F32>(p, i) : dt == WGS_BF16 ? load_elem<WGS_BF16>(p, i) : load_elem<WGS_F16>(p, i);
}
__device__ __forceinline__ void store_as(int dt, void* p, int64_t i, float v) {
    if (dt == WGS_F32) ((float*)p)[i] = v;
    else if (dt == WGS_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}
// 16 bytes -> 4 (fp32) or 8 floats
template <int DT> __device__ __forceinline__ void unpack_as(uint4 q, float* v) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == WGS_F32) v[i] = __uint_as_float(w[i]);
        else if (DT == WGS_BF16) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            const h2 h = __builtin_bit_cast(h2, w[i]);
            v[2 * i] = (float)h[0]; v[2 * i + 1] = (float)h[1];
        }
    }
}
// The update that is orthogonalised.  STEP: momentum <- mu momentum + g, u = g + mu momentum (nesterov) or momentum.
struct Momentum { float mu, grad_scale; int nesterov; };
template <int DT, bool STEP>
__device__ __forceinline__ float update_of(const Mat& a, int64_t i, int64_t mi, const Momentum& mo, bool write) {
    float v = load_elem<DT>(a.in, i);
    if (STEP) {
        const float gr = v * mo.grad_scale;
        float b = a.momentum[mi];
        if (write) { b = __builtin_fmaf(mo.mu, b, gr); a.momentum[mi] = b; }
        v = mo.nesterov ? __builtin_fmaf(mo.mu, b, gr) : b;
    }
    return v;
}

// ---- 1. partial norms (and the new momentum) ----------------------------------------------------------------------------------------
// Memory-bound: 16-byte loads, four in flight, where the matrix is dense and aligned (one element at a time otherwise).  Squares are summed in
// fp64: neither 1e30 nor 1e-30 leaves its range.
template <int DT, bool STEP>
__global__ __launch_bounds__(512) void ortho_norm_kernel(const Group g, const Momentum mo) {
    constexpr int V = DT == WGS_F32 ? 4 : 8;
    __shared__ double rs[8];
    __shared__ float rm[8];
    const int inst = blockIdx.x / (unsigned)g.stat_blocks, blk = blockIdx.x % (unsigned)g.stat_blocks, t = threadIdx.x;
    const Mat& a = g.mat[entry_of(g, inst)];
    const int b = inst - a.first;
    const int64_t total = (int64_t)a.M * a.N, off = b * a.in_bs, moff = b * total;
    const int64_t per = up((total + g.stat_blocks - 1) / g.stat_blocks, 512 * V);
    const int64_t e0 = blk * per, e1 = e0 + per < total ? e0 + per : total;
    double ss = 0.0;
    float amax = 0.f;
    auto take = [&](float v) { ss = __builtin_fma((double)v, (double)v, ss); amax = fmaxf(amax, fabsf(v)); };
    int64_t tail = e0;
    const bool dense = a.in_rs == a.N && ((uintptr_t)a.in & 15) == 0 && off % V == 0 && (!STEP || (((uintptr_t)a.momentum & 15) == 0 && moff % 4 == 0));
    if (dense) {
        const int64_t n = e1 > e0 ? (e1 - e0) / V : 0;
        const uint4* src = (const uint4*)((const char*)a.in + (off + e0) * (DT == WGS_F32 ? 4 : 2));
        float4* mom = STEP ? (float4*)(a.momentum + moff + e0) : nullptr;
        constexpr int U = STEP ? 2 : 4;
        for (int64_t i0 = 0; i0 < n; i0 += 512 * U) {
            uint4 q[U];
            float4 m[U][V / 4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = i0 + u * 512 + t;
                q[u] = make_uint4(0, 0, 0, 0);
                if (i < n) {
                    q[u] = src[i];
                    if (STEP)
#pragma unroll
                        for (int w = 0; w < V / 4; ++w) m[u][w] = mom[i * (V / 4) + w];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = i0 + u * 512 + t;
                if (i >= n) continue;
                float v[V];
                unpack_as<DT>(q[u], v);
                if (STEP) {
#pragma unroll
                    for (int w = 0; w < V / 4; ++w) {
                        float* x = &m[u][w].x;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float gr = v[4 * w + k] * mo.grad_scale;
                            x[k] = __builtin_fmaf(mo.mu, x[k], gr);
                            v[4 * w + k] = mo.nesterov ? __builtin_fmaf(mo.mu, x[k], gr) : x[k];
                        }
                        mom[i * (V / 4) + w] = m[u][w];
                    }
                }
#pragma unroll
                for (int k = 0; k < V; ++k) take(v[k]);
            }
        }
        tail = e0 + n * V;
    }
    for (int64_t e = tail + t; e < e1; e += 512) {
        const int64_t i = a.in_rs == a.N ? e : (e / a.N) * a.in_rs + e % a.N;
        take(update_of<DT, STEP>(a, off + i, moff + e, mo, true));
    }
    ss = wave_sum_d(ss);
    amax = wave_max(amax);
    if ((t & 63) == 0) { rs[t >> 6] = ss; rm[t >> 6] = amax; }
    __syncthreads();
    if (t == 0) {
        double x = 0.0;
        float y = 0.f;
        for (int w = 0; w < 8; ++w) { x += rs[w]; y = fmaxf(y, rm[w]); }
        Part* p = parts_of(g, inst) + blk;
        p->ss = x; p->amax = y;
    }
}

// ---- matrices of up to 16 rows (or columns): everything in 64 bits, one launch ------------------------------------------------------------------
// The whole run is X_K = Q X_0 with Q a polynomial in A_0, and in 64 bits A_0's rounding is far under the input's own even after 16 joined steps.  (As
// fp16 pairs, few and short sums leave a matrix of up to 8 rows up to 2.5 times as far from the exact factor as the iteration on 32-bit products: the
// pairs' rounding, the dropped lo * lo and the matrix cores' truncation of the smaller products of a group do not average out.)  One workgroup a matrix:
// a wave's share of A_0 from 16 columns at a time, their sum in the same order in every wave, the chain of 16 x 16 products in registers — a result's
// layout (register v: row 4 v + lane / 16, column lane % 16) is that of either operand of the next product, all of them being symmetric —, then Q
// times 16 columns at a time.  (As the left operand a result is its transpose: A is made symmetric in every step, else its antisymmetric rounding grows,
// to 4e-10 in place of 6e-13 where one direction is 1000 times the rest.)  The update that is orthogonalised stays in the workspace between the two passes, in fp32, its own precision.
// Bound by latency: of its dependent products for few columns, of one CU's loads for many.  fp32, us, the pairs' forms in brackets: 16 x 16 15 (22; 15 is
// a host call's length), 16 x 256 15 (27), 16 x 1024 28 (45), 16 x 2048 49 (49), 16 x 4096 93 (164), 16 x 8192 180 (167); a step of one matrix 9 (27), 15 (33),
// 44 (47), 75 (52), 144 (168), 274 (171).  So up to 4096 columns in fp32, beyond which sums are long enough for the pairs (at 4 x 1025 .. 4 x 2100 a
// third of all matrices were over 1.5 times as far as 32-bit products, at 4 x 16000 none); in 16 bits, where joined steps take 49 at 2048 and 55 at
// 4096 and the result's rounding hides the difference, up to 1024.
constexpr int TINY_M = 16, TINY_N = 4096, TINY_N_16BIT = 1024, TINY_WAVES = 4;
bool is_tiny(const Dims& d, int dtype) { return d.m <= TINY_M && d.n <= (dtype == WGS_F32 ? TINY_N : TINY_N_16BIT); }
__host__ __device__ __forceinline__ int64_t tiny_bytes(const Dims& d) { return up((int64_t)d.m * d.n * 4, 256); }
typedef double double4v __attribute__((ext_vector_type(4)));
struct TinyArgs { double a, b, c; float eps; int steps; };
template <int DT, bool STEP>
__global__ __launch_bounds__(64 * TINY_WAVES) void ortho_tiny_kernel(const Group g, const Momentum mo, const TinyArgs ar) {
    constexpr int U = 4;                      // groups of 16 columns in flight
    __shared__ double part[TINY_WAVES][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4, inst = blockIdx.x;
    const Mat& mat = g.mat[entry_of(g, inst)];
    const Dims d = dims_of(mat.M, mat.N);
    const int b = inst - mat.first;
    const bool wide = mat.M <= mat.N;
    const int64_t off = b * mat.in_bs, moff = (int64_t)b * mat.M * mat.N, ob = b * mat.out_bs;
    float* const xs = (float*)(g.ws + mat.ws + b * tiny_bytes(d));          // [m][n]
    auto mul = [](double x, double y, double4v z) { return __builtin_amdgcn_mfma_f64_16x16x4f64(x, y, z, 0, 0, 0); };
    auto product = [&](const double4v& x, const double4v& y) {
        double4v z = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int s = 0; s < 4; ++s) z = mul(x[s], y[s], z);
        return z;
    };
    double4v A = {0.0, 0.0, 0.0, 0.0};
    // Loads go to clamped addresses, unconditionally: they are in flight together.
#pragma unroll 1
    for (int k0 = 16 * U * wave; k0 < d.n; k0 += 16 * U * TINY_WAVES) {
        float v[U][4], mm[U][4];
        auto at = [&](int u, int t, bool& ok, int& r, int& c) {
            const int k = k0 + 16 * u + 4 * t + q, kk = k < d.n ? k : d.n - 1, ii = i < d.m ? i : d.m - 1;
            ok = k == kk && i == ii;
            r = wide ? ii : kk; c = wide ? kk : ii;
        };
        bool ok;
        int r, c;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                at(u, t, ok, r, c);
                v[u][t] = load_elem<DT>(mat.in, off + (int64_t)r * mat.in_rs + c);
                if (STEP) mm[u][t] = mat.momentum[moff + (int64_t)r * mat.N + c];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                at(u, t, ok, r, c);
                float x = v[u][t];
                if (STEP) {
                    const float gr = x * mo.grad_scale, b2 = __builtin_fmaf(mo.mu, mm[u][t], gr);
                    if (ok) mat.momentum[moff + (int64_t)r * mat.N + c] = b2;
                    x = mo.nesterov ? __builtin_fmaf(mo.mu, b2, gr) : b2;
                }
                x = ok ? x : 0.f;
                if (ok) xs[i * d.n + k0 + 16 * u + 4 * t + q] = x;
                A = mul((double)x, (double)x, A);
            }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) part[wave][v][lane] = A[v];
    __syncthreads();                          // (the workgroup's own writes of the update, too)
    double ss = 0.0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        A[v] = part[0][v][lane];
#pragma unroll
        for (int w = 1; w < TINY_WAVES; ++w) A[v] += part[w][v][lane];
        if (4 * v + q == i) ss += A[v];
    }
    ss = wave_sum_d(ss);
    // false for NaN and infinity: NaN throughout
    const double inv = ss < 1e300 ? (ss > 0.0 ? 1.0 / (sqrt(ss) + (double)ar.eps) : 0.0) : (double)NAN;
    A *= inv * inv;
    double4v Q = A;
    for (int t = 0; t < ar.steps; ++t) {
        double4v B = product(A, A);
#pragma unroll
        for (int v = 0; v < 4; ++v) B[v] = (4 * v + q == i ? ar.a : 0.0) + ar.b * A[v] + ar.c * B[v];
        Q = t ? product(B, Q) : B;
        if (t + 1 == ar.steps) break;
        const double4v P = product(B, A);
        A = 0.5 * (product(P, B) + product(B, P));       // each the other's transpose, bit for bit
    }
    Q *= inv;
#pragma unroll 1
    for (int j0 = 16 * U * wave; j0 < d.n; j0 += 16 * U * TINY_WAVES) {
        float x[U][4], w[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = 4 * s + q, j = j0 + 16 * u + i, kk = k < d.m ? k : d.m - 1, jj = j < d.n ? j : d.n - 1;
                x[u][s] = xs[kk * d.n + jj];
                if (STEP) w[u][s] = load_elem<DT>(mat.out, ob + (int64_t)(wide ? kk : jj) * mat.out_rs + (wide ? jj : kk));
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 16 * u + i;
            double4v o = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int s = 0; s < 4; ++s) o = mul(Q[s], 4 * s + q < d.m && j < d.n ? (double)x[u][s] : 0.0, o);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int k = 4 * v + q;
                if (k >= d.m || j >= d.n) continue;
                float y = (float)o[v];
                if (STEP) y = mat.decay * w[u][v] - mat.step * y;
                store_as(DT, mat.out, ob + (int64_t)(wide ? k : j) * mat.out_rs + (wide ? j : k), y);
            }
        }
    }
}

// ---- 2. scalars and the planes of X and X^T -----------------------------------------------------------------------------------------
struct Bounds { float eps; int steps; float grow[MAX_STEPS + 1], cap[MAX_STEPS + 1]; };      // |A_t| <= min(D0 grow[t], cap[t])
__device__ __forceinline__ float pow2_under(float bound, int top, int lo, int hi) {        // 2^(top - ceil(log2 bound)), clamped
    int e;
    frexpf(bound, &e);                       // bound < 2^e
    int s = top - e;
    s = s < lo ? lo : (s > hi ? hi : s);
    return ldexpf(1.f, s);
}
__device__ __forceinline__ void split_pair(float v, _Float16& h, _Float16& l) {
    asm volatile("" : "+v"(v));              // the value as rounded to fp32: a product may not be fused into one of the two conversions alone
    h = (_Float16)v;
    l = (_Float16)(v - (float)h);
}
// N values at once, two a conversion (to nearest)
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
template <int N, typename V> __device__ __forceinline__ void split_many(const float* v, V& h, V& l) {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        float2v x = {v[k], v[k + 1]};
        asm volatile("" : "+v"(x));
        const half2v p = __builtin_convertvector(x, half2v);
        const float2v r = {__builtin_fmaf((float)p[0], -1.f, x[0]), __builtin_fmaf((float)p[1], -1.f, x[1])};
        const half2v q = __builtin_convertvector(r, half2v);
        h[k] = p[0]; h[k + 1] = p[1]; l[k] = q[0]; l[k + 1] = q[1];
    }
}
// the input's own power of two: its largest entry between 2^14 and 2^15
__device__ __forceinline__ float scale_of(double ss, float amax) { return (ss < 1e300 && amax > 0.f) ? pow2_under(amax, 15, -120, 120) : 1.f; }
// the scalars of an instance from its sum of squares and largest entry
__device__ __forceinline__ void write_info(float* info, double ss, float amax, float mult, int n, const Bounds& bd) {
    const bool finite = ss < 1e300;          // false for NaN and infinity: NaN throughout
    const double inv = ss > 0.0 ? 1.0 / (sqrt(ss) + (double)bd.eps) : 0.0;
    info[0] = finite ? (float)(inv / (double)mult) : NAN;
    const double top = (double)amax * inv;
    const double d0 = finite ? (double)n * top * top : 1.0;
    for (int k = 0; k <= bd.steps; ++k) {
        double v = d0 * (double)bd.grow[k];
        v = v < (double)bd.cap[k] ? v : (double)bd.cap[k];
        info[I_SA + k] = pow2_under((float)(v > 1e-30 ? v : 1e-30), 14, -60, 60);
        info[I_SX + k] = pow2_under((float)sqrt(v > 1e-70 ? v : 1e-70), 14, -60, 110);
    }
}
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ortho_split_kernel(const Group g, const Momentum mo, const Bounds bd, int tiles) {
    constexpr bool LO = DT == WGS_F32 || STEP;
    __shared__ float tile[64][65];
    __shared__ double rs[4];
    __shared__ float rm[4];
    const int t = threadIdx.x;
    // block -> (instance, 64 x 64 tile)
    int bid = blockIdx.x, e = 0, tn = 0, tm = 0;
    for (;; ++e) {
        const Mat& a = g.mat[e];
        tm = (int)(up(a.M, BK) + 63) / 64; tn = (int)(up(a.N, BK) + 63) / 64;
        const int c = a.batch * tm * tn;
        if (bid < c || e + 1 == g.count) break;
        bid -= c;
    }
    const Mat& a = g.mat[e];
    const Dims d = dims_of(a.M, a.N);
    const int b = bid / (tm * tn), tt = bid % (tm * tn), inst = a.first + b;
    const int r0 = (tt / tn) * 64, c0 = (tt % tn) * 64;
    // the norm of the instance: every workgroup adds the partial ones itself
    double ss = 0.0;
    float amax = 0.f;
    const Part* p = parts_of(g, inst);
    if (t < g.stat_blocks) { ss = p[t].ss; amax = p[t].amax; }
    ss = wave_sum_d(ss);
    amax = wave_max(amax);
    if ((t & 63) == 0) { rs[t >> 6] = ss; rm[t >> 6] = amax; }
    __syncthreads();
    ss = rs[0] + rs[1] + rs[2] + rs[3];
    amax = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
    const float mult = scale_of(ss, amax);
    if (tt == 0 && t == 0) write_info(info_of(g, inst), ss, amax, mult, d.n, bd);
    const int64_t off = b * a.in_bs, moff = (int64_t)b * a.M * a.N;
    const bool vec = r0 + 64 <= a.M && c0 + 64 <= a.N && a.in_rs % 8 == 0 && off % 8 == 0 && ((uintptr_t)a.in & 15) == 0 &&
                     (!STEP || (a.N % 4 == 0 && moff % 4 == 0 && ((uintptr_t)a.momentum & 15) == 0));
    if (vec) {
        constexpr int V = DT == WGS_F32 ? 4 : 8, PER = 64 / V;
#pragma unroll
        for (int i = t; i < 64 * PER; i += 256) {
            const int r = i / PER, c = (i % PER) * V;
            float v[V];
            unpack_as<DT>(*(const uint4*)((const char*)a.in + (off + (int64_t)(r0 + r) * a.in_rs + c0 + c) * (DT == WGS_F32 ? 4 : 2)), v);
            if (STEP) {
                const float4* m = (const float4*)(a.momentum + moff + (int64_t)(r0 + r) * a.N + c0 + c);
#pragma unroll
                for (int w = 0; w < V / 4; ++w) {
                    const float4 q = m[w];
                    const float x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * w + k] = mo.nesterov ? __builtin_fmaf(mo.mu, x[k], v[4 * w + k] * mo.grad_scale) : x[k];
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) tile[r][c + k] = v[k] * mult;
        }
    } else {
        for (int i = t; i < 64 * 64; i += 256) {
            const int r = r0 + (i >> 6), c = c0 + (i & 63);
            float v = 0.f;
            if (r < a.M && c < a.N) v = update_of<DT, STEP>(a, off + (int64_t)r * a.in_rs + c, moff + (int64_t)r * a.N + c, mo, false) * mult;
            tile[i >> 6][i & 63] = v;
        }
    }
    __syncthreads();
    const bool wide = a.M <= a.N;
    const Plane nat = plane_of(g, a, d, b, wide ? BUF_X : BUF_T0, LO), tra = plane_of(g, a, d, b, wide ? BUF_T0 : BUF_X, LO);
    // natural: rows r < M, columns up to the padding; transposed: rows c < N, columns r up to the padding.  Eight columns (16 bytes) a thread;
    // the padded lengths are multiples of 32.
    auto put = [&](const Plane& p, int row, int col, const float (&v)[8]) {
        half8 h, l;
        split_many<8>(v, h, l);
        unsigned char* q = at_hi(p, row, col);
        *reinterpret_cast<half8*>(q) = h;
        if (LO) *reinterpret_cast<half8*>(q + 64) = l;
    };
#pragma unroll
    for (int i = t; i < 64 * 8; i += 256) {
        const int x = i >> 3, y = (i & 7) * 8;
        float v[8];
        if (r0 + x < a.M && c0 + y < nat.ld) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = tile[x][y + k];
            put(nat, r0 + x, c0 + y, v);
        }
        if (c0 + x < a.N && r0 + y < tra.ld) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = tile[y + k][x];
            put(tra, c0 + x, r0 + y, v);
        }
    }
}

// ---- small matrices: everything in one launch, or a launch a step -------------------------------------------------------------------------------------------------
// m <= 32 MT <= 64, n <= SMALL_N: one workgroup a matrix, the m x m matrices in LDS.  X lies in blocks of 32 columns as the operand "lane = column j,
// 8 rows i": the product's own result layout (lane = column, rows 8 q + 4 half + 0..3) is an operand again once the sum's index is taken in that
// order, B's fragments being read from LDS in the same one.  The next Gram matrix needs X with lane = row: the transposed product X^T B, from the
// same two operands, has it, and is used and dropped block by block.  A block's fragments stay with one wave, which stores and loads them lane by
// lane (1 KB at a time) through the caches: in registers they do not fit beside the accumulators.  The waves' partial Gram matrices are added in
// a fixed order.  Bound by the latency of its steps and one CU's matrix cores; the many launches of the general path cost more where all_small says so.
constexpr int SMALL_N = 2048, SMALL_WAVES = 8;
// With many columns it is a launch a step instead, a block a wave (WHOLE = false; the norm comes from its kernel): a workgroup adds the partial Gram
// matrices of its matrix's workgroups, in order, forms B, applies it to its blocks and leaves its part of the next Gram matrix.  (Workgroups of four
// and two waves have more parts to add and fewer threads to do it: 4 x 64 x 576 fp32 68 us with eight, 74, 85.)
struct SmallArgs { Bounds bd; float sb[MAX_STEPS]; float a, b, c; int t, parts; };      // WHOLE = false: the step (-1: the operands), most workgroups a matrix
__host__ __device__ __forceinline__ bool is_small(const Dims& d) { return d.m <= 64 && d.n <= SMALL_N; }
__host__ __device__ __forceinline__ int64_t small_parts(const Dims& d) { return (d.np / 32 + SMALL_WAVES - 1) / SMALL_WAVES; }
__host__ __device__ __forceinline__ int64_t small_bytes(const Dims& d) { return 64 * (int64_t)d.np * 4 + 2 * small_parts(d) * (3 * 1024 * 4); }      // X, two sets of partial Gram matrices
template <int MT, bool WHOLE>
__global__ __launch_bounds__(64 * SMALL_WAVES, 1) void ortho_small_kernel(const Group g, const Momentum mo, const SmallArgs ar) {
    constexpr int W = SMALL_WAVES, TRI = MT * (MT + 1) / 2, LD = 32 * MT + 8, TURNS = 16 * MT, U = 16;
    __shared__ float part[W][TRI][32][33];
    __shared__ __attribute__((aligned(16))) _Float16 sa[2][32 * MT][LD], sbm[2][32 * MT][LD];
    __shared__ double rs[W];
    __shared__ float rm[W];
    __shared__ float info[INFO];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, lh = lane >> 5;
    const int inst = WHOLE ? blockIdx.x : blockIdx.x / (unsigned)ar.parts, pw = WHOLE ? 0 : blockIdx.x % (unsigned)ar.parts;
    const Mat& mat = g.mat[entry_of(g, inst)];
    const int b = inst - mat.first;
    const Dims d = dims_of(mat.M, mat.N);
    const int parts = WHOLE ? 1 : (int)small_parts(d);
    if (pw >= parts) return;
    const bool wide = mat.M <= mat.N;
    const int64_t off = b * mat.in_bs, moff = (int64_t)b * mat.M * mat.N, ob = b * mat.out_bs;
    float* const sums = (float*)(g.ws + mat.ws + b * small_bytes(d) + 64 * (int64_t)d.np * 4);       // [2][parts][TRI][1024]
    float* tr = &part[wave][0][0][0];          // a wave's own [32 MT rows i][33]
    const int blocks = d.np / 32, k0 = pw * W + wave, kstep = parts * W, active = blocks - pw * W < W ? blocks - pw * W : W;
    frag* const frags = (frag*)(g.ws + mat.ws + b * small_bytes(d)) + lane;      // block k: [tile][half][hi, lo][64 lanes]
    auto at = [&](int k, int t, int ks, int pl) { return frags + (((int64_t)k * MT + t) * 4 + ks * 2 + pl) * 64; };
    auto split = [&](const float* v, frag& fh, frag& fl) {
        half8 h, l;
        split_many<8>(v, h, l);
        fh = __builtin_bit_cast(frag, h); fl = __builtin_bit_cast(frag, l);
    };
    auto mul = [](frag x, frag y, f32x16 z) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), z, 0, 0, 0); };

    // Element e of block k: lane and turn own it, in the two passes over the input (norm and new momentum first, then the scaled operands, from
    // the caches) and in the one over the result.  Loads go to clamped addresses, unconditionally: they are in flight together.
    auto typed = [&](auto f) __attribute__((always_inline)) {
        if (g.dtype == WGS_F32) f(std::integral_constant<int, WGS_F32>());
        else if (g.dtype == WGS_BF16) f(std::integral_constant<int, WGS_BF16>());
        else f(std::integral_constant<int, WGS_F16>());
    };
    // A lane's elements of block k: column c of the matrix, rows r0, r0 + dr, ...; in LDS at t0, t0 + dt, ...
    struct Own { int r0, dr, c, t0, dt; };
    auto own = [&](int k) {
        int ln = lane;
        asm volatile("" : "+v"(ln));            // (formed here, not kept in registers through the kernel)
        const int hi = ln / (32 * MT), lo = ln & (32 * MT - 1);
        return wide ? Own{ln >> 5, 2, k * 32 + (ln & 31), (ln >> 5) * 33 + (ln & 31), 66} : Own{k * 32 + hi, 2 / MT, lo, lo * 33 + hi, 2 / MT};
    };
    auto input = [&](bool first, int k, float mult, auto take) __attribute__((always_inline)) {
        typed([&](auto dt) __attribute__((always_inline)) {
            constexpr int DT = decltype(dt)::value;
            const Own o = own(k);
            const int cc = o.c < mat.N ? o.c : mat.N - 1;
#pragma unroll 1
            for (int it0 = 0; it0 < TURNS; it0 += U) {
                float v[U], mm[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    int r = o.r0 + (it0 + u) * o.dr;
                    r = r < mat.M ? r : mat.M - 1;
                    v[u] = load_elem<DT>(mat.in, off + cc + (int64_t)r * mat.in_rs);
                    mm[u] = 0.f;
                    if (g.step) mm[u] = mat.momentum[moff + cc + r * mat.N];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = o.r0 + (it0 + u) * o.dr;
                    const bool ok = r < mat.M && o.c < mat.N;
                    if (g.step) {
                        const float gr = v[u] * mo.grad_scale;
                        if (first) {
                            mm[u] = __builtin_fmaf(mo.mu, mm[u], gr);
                            if (ok) mat.momentum[moff + cc + r * mat.N] = mm[u];
                        }
                        v[u] = mo.nesterov ? __builtin_fmaf(mo.mu, mm[u], gr) : mm[u];
                    }
                    take(o.t0 + (it0 + u) * o.dt, ok ? v[u] * mult : 0.f);
                }
            }
        });
    };
    f32x16 gr[TRI];
    auto gram = [&](const frag (&ih)[MT][2], const frag (&il)[MT][2]) __attribute__((always_inline)) {       // adds one block: lane = row i, 8 columns a fragment
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int pr = 0; pr < 3; ++pr)
#pragma unroll
                for (int t = 0; t < TRI; ++t) {
                    const int p = t == 0 ? 0 : 1, q = t == 2 ? 1 : 0;
                    gr[t] = mul(pr == 0 ? il[p][ks] : ih[p][ks], pr == 1 ? il[q][ks] : ih[q][ks], gr[t]);
                }
    };
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < TRI; ++t)
#pragma unroll
            for (int q = 0; q < 16; ++q) gr[t][q] = 0.f;
    };
    auto leave = [&](int l31, int lh) __attribute__((always_inline)) {          // a wave's part of the Gram matrix into the LDS
        if (wave < active)
#pragma unroll
            for (int k = 0; k < TRI; ++k)
#pragma unroll
                for (int q = 0; q < 16; ++q) part[wave][k][8 * (q >> 2) + 4 * lh + (q & 3)][l31] = gr[k][q];
        __syncthreads();
    };
    auto publish = [&](int t) __attribute__((always_inline)) {                  // WHOLE = false: the workgroup's part, for step t
        leave(l31, lh);
        float* o = sums + ((t & 1) * parts + pw) * (TRI * 1024);
        for (int e = tid; e < TRI * 1024; e += 64 * W) {
            const int k = e >> 10, r = (e >> 5) & 31, c = e & 31;
            float v = part[0][k][r][c];
            for (int w = 1; w < active; ++w) v += part[w][k][r][c];
            o[e] = v;
        }
    };
    if (WHOLE || ar.t < 0) {
    double ss = 0.0;
    float amax = 0.f;
    if (!WHOLE) {
        const Part* p = parts_of(g, inst);
        if (tid < g.stat_blocks) { ss = p[tid].ss; amax = p[tid].amax; }
    } else
#pragma unroll 1
    for (int k = wave; k < blocks; k += W)
        input(true, k, 1.f, [&](int, float v) {
            ss = __builtin_fma((double)v, (double)v, ss);
            amax = fmaxf(amax, fabsf(v));
        });
    ss = wave_sum_d(ss);
    amax = wave_max(amax);
    if (lane == 0) { rs[wave] = ss; rm[wave] = amax; }
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) { ss += rs[w]; amax = fmaxf(amax, rm[w]); }
    const float mult = scale_of(ss, amax);
    if (tid == 0 && pw == 0) write_info(WHOLE ? info : info_of(g, inst), ss, amax, mult, d.n, ar.bd);

    // the operands, through LDS: lane = column to stay, lane = row for the first Gram matrix
    clear();
#pragma unroll 1
    for (int k = k0; k < blocks; k += kstep) {
        asm volatile("" ::: "memory");
        input(false, k, mult, [&](int i, float v) { tr[i] = v; });
        asm volatile("" ::: "memory");
        frag ih[MT][2], il[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float v[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = tr[(32 * t + 8 * (q >> 2) + 4 * lh + (q & 3)) * 33 + l31];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                frag h, l;
                split(v + 8 * ks, h, l);
                *at(k, t, ks, 0) = h; *at(k, t, ks, 1) = l;
            }
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = tr[(32 * t + l31) * 33 + 8 * (q >> 2) + 4 * lh + (q & 3)];
            split(v, ih[t][0], il[t][0]);
            split(v + 8, ih[t][1], il[t][1]);
        }
        gram(ih, il);
    }
    if (!WHOLE) { publish(0); return; }
    }
    frag nh[MT][2], nl[MT][2];               // the next block's fragments
    auto load = [&](int k) {
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) { nh[u][ks] = *at(k, u, ks, 0); nl[u][ks] = *at(k, u, ks, 1); }
    };
    if (!WHOLE && k0 < blocks) load(k0);
    const float* const inf = WHOLE ? info : info_of(g, inst);
#pragma unroll 1
    for (int t = WHOLE ? 0 : ar.t; t < (WHOLE ? ar.bd.steps : ar.t + 1); ++t) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid) :: "memory");       // (nor the LDS addresses from step to step)
        const int lane = tid & 63, l31 = lane & 31, lh = lane >> 5;
        constexpr int EACH = TRI * 1024 / (64 * W);
        float sum[EACH];
        if (WHOLE) leave(l31, lh);
        else {
            const float* src = sums + (t & 1) * parts * (TRI * 1024) + tid;
#pragma unroll
            for (int it = 0; it < EACH; ++it) sum[it] = src[it * 64 * W];
#pragma unroll 2
            for (int w = 1; w < parts; ++w)
#pragma unroll
                for (int it = 0; it < EACH; ++it) sum[it] += src[w * (TRI * 1024) + it * 64 * W];
        }
        const float fx = t == 0 ? inf[0] : 1.f / inf[I_SX + t], sA = inf[I_SA + t], ga = fx * fx * sA;
#pragma unroll
        for (int it = 0; it < EACH; ++it) {
            const int e = it * 64 * W + tid, k = e >> 10, r = (e >> 5) & 31, c = e & 31;
            const int p = k == 0 ? 0 : 1, q = k == 2 ? 1 : 0;
            if (p == q && r < c) continue;
            float v = WHOLE ? part[0][k][r][c] : sum[it];
            if (WHOLE)
                for (int w = 1; w < active; ++w) v += part[w][k][r][c];
            _Float16 h, l;
            split_pair(v * ga, h, l);
            sa[0][32 * p + r][32 * q + c] = h; sa[1][32 * p + r][32 * q + c] = l;
            sa[0][32 * q + c][32 * p + r] = h; sa[1][32 * q + c][32 * p + r] = l;
        }
        __syncthreads();
        if (wave < TRI) {
            const int p = wave == 0 ? 0 : 1, q = wave == 2 ? 1 : 0;
            f32x16 s0, s1;
#pragma unroll
            for (int k = 0; k < 16; ++k) { s0[k] = 0.f; s1[k] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < 2 * MT; ++ks) {
                const int kc = 16 * ks + 8 * lh;
                const half8 ah = *reinterpret_cast<const half8*>(&sa[0][32 * p + l31][kc]), al = *reinterpret_cast<const half8*>(&sa[1][32 * p + l31][kc]);
                const half8 bh = *reinterpret_cast<const half8*>(&sa[0][32 * q + l31][kc]), bl = *reinterpret_cast<const half8*>(&sa[1][32 * q + l31][kc]);
                s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, s0, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, s1, 0, 0, 0);
                s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, s0, 0, 0, 0);
            }
            const float isa = 1.f / sA;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int r = 8 * (k >> 2) + 4 * lh + (k & 3), c = l31;
                const float A = ((float)sa[0][32 * p + r][32 * q + c] + (float)sa[1][32 * p + r][32 * q + c]) * isa;
                const float v = ((p == q && r == c ? ar.a : 0.f) + (ar.b * A + ar.c * ((s0[k] + s1[k]) * isa * isa))) * ar.sb[t];
                _Float16 h, l;
                split_pair(v, h, l);
                if (p != q || r >= c) {
                    sbm[0][32 * p + r][32 * q + c] = h; sbm[1][32 * p + r][32 * q + c] = l;
                    sbm[0][32 * q + c][32 * p + r] = h; sbm[1][32 * q + c][32 * p + r] = l;
                }
            }
        }
        __syncthreads();
        const bool last = t + 1 == ar.bd.steps;
        const float fo = last ? fx / ar.sb[t] : fx * inf[I_SX + t + 1] / ar.sb[t];
        clear();
        if (WHOLE && k0 < blocks) load(k0);
#pragma unroll 1
        for (int k = k0; k < blocks; k += kstep) {
            frag vh[MT][2], vl[MT][2];
#pragma unroll
            for (int u = 0; u < MT; ++u)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) { vh[u][ks] = nh[u][ks]; vl[u][ks] = nl[u][ks]; }
            if (WHOLE) load(k + W < blocks ? k + W : k);
            // B X (lane = column) and, from the same operands in the other order, X^T B (lane = row)
            f32x16 dd[MT], de[MT];
#pragma unroll
            for (int u = 0; u < MT; ++u)
#pragma unroll
                for (int q = 0; q < 16; ++q) { dd[u][q] = 0.f; de[u][q] = 0.f; }
            asm volatile("" ::: "memory");          // (B's fragments are read again for every block: kept, they would not fit)
#pragma unroll
            for (int ks = 0; ks < 2 * MT; ++ks) {
                const int kb = 16 * ks + 4 * lh;
                frag bh[MT], bl[MT];
#pragma unroll
                for (int u = 0; u < MT; ++u) {
                    const int2 h0 = *reinterpret_cast<const int2*>(&sbm[0][32 * u + l31][kb]), h1 = *reinterpret_cast<const int2*>(&sbm[0][32 * u + l31][kb + 8]);
                    const int2 l0 = *reinterpret_cast<const int2*>(&sbm[1][32 * u + l31][kb]), l1 = *reinterpret_cast<const int2*>(&sbm[1][32 * u + l31][kb + 8]);
                    bh[u] = frag{h0.x, h0.y, h1.x, h1.y};
                    bl[u] = frag{l0.x, l0.y, l1.x, l1.y};
                }
                const frag ph = vh[ks >> 1][ks & 1], pl = vl[ks >> 1][ks & 1];
#pragma unroll
                for (int pr = 0; pr < 3; ++pr)
#pragma unroll
                    for (int u = 0; u < MT; ++u) {
                        const frag x = pr == 0 ? pl : ph, y = pr == 1 ? bl[u] : bh[u];
                        dd[u] = mul(x, y, dd[u]);
                        if (!last) de[u] = mul(y, x, de[u]);
                    }
            }
            if (last) {
                // lane = row i: to LDS as [i][j], then out in rows of the result
                asm volatile("" ::: "memory");
#pragma unroll
                for (int u = 0; u < MT; ++u)
#pragma unroll
                    for (int q = 0; q < 16; ++q) tr[(32 * u + l31) * 33 + 8 * (q >> 2) + 4 * lh + (q & 3)] = dd[u][q] * fo;
                asm volatile("" ::: "memory");
                typed([&](auto dt) __attribute__((always_inline)) {
                    constexpr int DT = decltype(dt)::value;
                    const Own o = own(k);
                    const int cc = o.c < mat.N ? o.c : mat.N - 1;
#pragma unroll 1
                    for (int it0 = 0; it0 < TURNS; it0 += U) {
                        float w[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            int r = o.r0 + (it0 + u) * o.dr;
                            r = r < mat.M ? r : mat.M - 1;
                            w[u] = 0.f;
                            if (g.step) w[u] = load_elem<DT>(mat.out, ob + cc + (int64_t)r * mat.out_rs);
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int r = o.r0 + (it0 + u) * o.dr;
                            float v = tr[o.t0 + (it0 + u) * o.dt];
                            if (g.step) v = mat.decay * w[u] - mat.step * v;
                            if (r < mat.M && o.c < mat.N) store_as(DT, mat.out, ob + cc + (int64_t)r * mat.out_rs, v);
                        }
                    }
                });
                continue;
            }
            frag ih[MT][2], il[MT][2];
            float v[16];
#pragma unroll
            for (int u = 0; u < MT; ++u) {
#pragma unroll
                for (int q = 0; q < 16; ++q) v[q] = dd[u][q] * fo;
                split(v, ih[u][0], il[u][0]); split(v + 8, ih[u][1], il[u][1]);
            }
            gram(ih, il);
#pragma unroll
            for (int u = 0; u < MT; ++u) {
#pragma unroll
                for (int q = 0; q < 16; ++q) v[q] = de[u][q] * fo;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    frag h, l;
                    split(v + 8 * ks, h, l);
                    *at(k, u, ks, 0) = h; *at(k, u, ks, 1) = l;
                }
            }
        }
        if (!WHOLE && !last) publish(t + 1);
    }
}

// ---- 3. products ----------------------------------------------------------------------------------------------------------------------
enum { GRAM, POLY, PROD, PROD_A, APPLY_MID, APPLY_OUT };
struct Job {
    int kind;                // what becomes of the product
    int p, r;                // operands: D[i][j] = sum_k p[i][k] r[j][k]
    int dst, dst2;           // buffers written (APPLY_MID: X and X^T)
    int src;                 // POLY: A
    int t, t2;               // iteration of the operands' / the result's scale
    int first;               // X is the input (its scale is f0)
    float mul;               // factor known on the host
    float a, b, c;           // POLY
};
struct Jobs { Job job[2]; int count; int sym; int kgram; };      // kgram: sums over the n columns, not over m

// tile number -> tile coordinates, in squares of 4 x 4 tiles: the tiles that run side by side on an XCD share operands in its L2
__device__ __forceinline__ void tile_full(int t, int tm, int tn, int& ti, int& tj) {
    const int strip = 4 * tn, s = t / strip, in = t % strip;
    const int h = tm - 4 * s < 4 ? tm - 4 * s : 4;
    ti = 4 * s + in % h; tj = in / h;
}
__device__ __forceinline__ void tile_lower(int t, int tm, int& ti, int& tj) {
    int s = 0;
    for (;; ++s) {                                      // strips of four tile rows; at most tm / 4 of them
        const int h = tm - 4 * s < 4 ? tm - 4 * s : 4, c = 4 * s * h + h * (h + 1) / 2;
        if (t < c || 4 * (s + 1) >= tm) {
            if (t < 4 * s * h) { ti = 4 * s + t % h; tj = t / h; return; }
            t -= 4 * s * h;
            int r = 0;
            while (t > r) { t -= r + 1; ++r; }
            ti = 4 * s + r; tj = 4 * s + t;
            return;
        }
        t -= c;
    }
}

// E: side of the square blocks in which a wave hands its results through LDS to the stores (32 / 64 / 96)
template <int NA, int NB, int BM, int WAVES_M, int WAVES_N, int NS, int E, bool SPLIT = false>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 1) void ortho_gemm_kernel(const Jobs js, int total, int run, int most, int join, const Group g) {
    constexpr int BN = BM, NW = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
    constexpr int RA = NA * ROW, RB = NB * ROW, A_BYTES = BM * RA, B_BYTES = BN * RB, CHUNK = A_BYTES + B_BYTES;      // bytes of a row, an operand, a chunk
    constexpr int KC = BM == 64 ? 2 : 1, STAGE = KC * CHUNK;                                                          // chunks of a stage
    constexpr int GA = 1024 / RA, GB = 1024 / RB, AI = BM / GA / NW, BI = BN / GB / NW, CP = AI + BI, NPIECE = KC * CP;               // rows of a load, loads of a wave
    static_assert(AI * GA * NW == BM && BI * GB * NW == BN && TM * 32 * WAVES_M == BM && TN * 32 * WAVES_N == BN, "tile / wave count mismatch");
    static_assert(WM % E == 0 && WN % E == 0, "epilogue block");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;

    // The arguments' lines all at once: read where they are needed, each would be a round trip to memory of its own.
    {
        const Mat& m0 = g.mat[0];
        const Job& j0 = js.job[0];
        asm volatile("" :: "s"(m0.M), "s"(m0.ws), "s"(m0.out), "s"(g.ws), "s"(g.info), "s"(js.sym), "s"(j0.kind), "s"(j0.first), "s"(js.job[1].kind), "s"(total));
    }
    // Workgroups go round the 8 XCDs: runs of at most 32 tiles in turn, equally many each, so that an XCD's CUs work on neighbouring tiles and every
    // entry is spread over the XCDs.  Entries come in the caller's order; a launch of uneven sums ends with its longest tile (in the first Gram launch of
    // a transformer block of width 2048 some tiles' sums are four times the others', and it takes twice its work's time at full spread).
    const int idx = (int)(blockIdx.x >> 3);
    int tile = (idx / run * 8 + (int)(blockIdx.x & 7)) * run + idx % run;
    if (tile >= total) return;
    int parts = 1, slots = 0, before = 0, slot0 = 0;
    const int half = js.count == 2 ? total / 2 : total;
    const Job& J = js.job[tile >= half ? 1 : 0];
    if (tile >= half) tile -= half;
    int e = 0, tm = 0, tn = 0, per = 0;
    for (;; ++e) {
        const Dims q = dims_of(g.mat[e].M, g.mat[e].N);
        tm = (q.m + BM - 1) / BM; tn = (q.n + BN - 1) / BN;
        per = js.sym ? tm * (tm + 1) / 2 : tm * tn;
        if (SPLIT) { parts = parts_of_sum((js.kgram ? q.np : q.mp) / BK, most); if (!join) per *= parts; slots = g.mat[e].batch * per * (join ? parts : 1); }
        const int c = g.mat[e].batch * per;
        if (tile < c || e + 1 == g.count) break;
        tile -= c;
        if (SPLIT) before += slots;
    }
    const Mat& mat = g.mat[e];
    const Dims d = dims_of(mat.M, mat.N);
    const int b = tile / per, inst = mat.first + b;
    int part = 0;
    if (SPLIT) {                         // slot of the (first) part in the workspace; parts of a tile are neighbours
        slot0 = before + (join ? tile * parts : tile);
        if (!join) { tile -= b * per; part = tile % parts; tile /= parts; per /= parts; tile += b * per; }
        if (join && parts == 1) return;
    }
    int ti, tj;
    if (js.sym) tile_lower(tile % per, tm, ti, tj);
    else tile_full(tile % per, tm, tn, ti, tj);
    const int i0 = ti * BM, j0 = tj * BN;
    const Plane P = plane_of(g, mat, d, b, J.p, NA == 2), R = plane_of(g, mat, d, b, J.r, NB == 2);
    const int nk_all = P.ld / BK, k0 = SPLIT ? nk_all * part / parts : 0, nk = SPLIT ? nk_all * (part + 1) / parts - k0 : nk_all;
    const int rows_r = J.kind >= APPLY_MID ? d.n : d.m;
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(P.p, 0, (unsigned)(d.m * row_bytes(P)), 0x00020000);
    const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(R.p, 0, (unsigned)(rows_r * row_bytes(R)), 0x00020000);
    // An LDS load writes wave base + lane * 16: one instruction fills 8 rows of 128 bytes (32 hi, 32 lo) or 16 of 64.  The 16-byte slots of a row
    // are permuted by the row's number, on the address that is fetched and on the one that is read, so that the rows of a fragment read spread
    // over all banks.
    auto twist = [](int row, int n) { return n == 2 ? (row >> 1) & 7 : (row >> 2) & 3; };
    int a_off[AI], b_off[BI];
#pragma unroll
    for (int j = 0; j < AI; ++j) {
        const int row = (wave * AI + j) * GA + lane / (64 / GA), lc = lane % (64 / GA) ^ twist(row, NA);
        a_off[j] = i0 + row < d.m ? (i0 + row) * row_bytes(P) + lc * 16 : OOB;
    }
#pragma unroll
    for (int j = 0; j < BI; ++j) {
        const int row = (wave * BI + j) * GB + lane / (64 / GB), lc = lane % (64 / GB) ^ twist(row, NB);
        b_off[j] = j0 + row < rows_r ? (j0 + row) * row_bytes(R) + lc * 16 : OOB;
    }
    // piece x of the next chunk (chunk nC, behind the last one that one again: its data is not used) into stage buf
    int nC = 0;
    auto piece = [&](int buf, int y) {
        const int x = y % CP, c1 = nC * KC + y / CP;
        const bool past = KC == 2 && c1 >= nk;                  // (an odd number of chunks: zeros)
        const int c = k0 + (c1 < nk ? c1 : nk - 1);
        lds_byte* st = (lds_byte*)(smem + buf * STAGE + y / CP * CHUNK);
        if (x < AI) {
            const int off = past ? OOB : a_off[x];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, st + (wave * AI + x) * 1024, 16, off, c * RA, 0, 0);
        } else {
            const int off = past ? OOB : b_off[x - AI];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rr, st + A_BYTES + (wave * BI + x - AI) * 1024, 16, off, c * RB, 0, 0);
        }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int l31 = lane & 31, lh = lane >> 5;
    const int a_rd = (wm * WM + l31) * RA, a_sl = (lh ^ twist(l31, NA)) * 16, b_rd = A_BYTES + (wn * WN + l31) * RB, b_sl = (lh ^ twist(l31, NB)) * 16;
    struct Frags { half8 a[TM][NA], b[TN][NB]; };
    constexpr int READS = TM * NA + TN * NB, PRODS = (NA > 1) + (NB > 1) + 1, MMAS = PRODS * TM * TN;
    auto read = [&](int buf, int ks, int x, Frags& f) {      // fragment x of half ks of a chunk
        const unsigned char* base = smem + buf * STAGE;      // slot = half of the lane, half chunk, hi / lo: bits 0, 1, 2
        if (x < TM * NA) f.a[x / NA][x % NA] = *reinterpret_cast<const half8*>(base + a_rd + (x / NA) * 32 * RA + (a_sl ^ (ks * 32 + (x % NA) * 64)));
        else { const int y = x - TM * NA; f.b[y / NB][y % NB] = *reinterpret_cast<const half8*>(base + b_rd + (y / NB) * 32 * RB + (b_sl ^ (ks * 32 + (y % NB) * 64))); }
    };
    // The products of one half chunk, small terms first and neighbours on different accumulators, with the reads of the next half's fragments and
    // the loads of a later chunk spread between them: the matrix pipe is never without a product that is ready.
#define ORTHO_MMA(F, G2, BUF, KS, LOADS, LBUF)                                                                                              \
    _Pragma("unroll") for (int n = 0; n < MMAS; ++n) {                                                                                      \
        constexpr int SIDE = READS + LOADS * NPIECE;                                                                                        \
        const int pr = PRODS == 3 ? n / (TM * TN) : PRODS == 2 ? 2 * (n / (TM * TN)) : 2, i = (n % (TM * TN)) / TN, j = n % TN;               \
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(F.a[i][pr == 0 ? NA - 1 : 0], F.b[j][pr == 1 ? NB - 1 : 0], acc[i][j], 0, 0, 0);  \
        _Pragma("unroll") for (int s = n * SIDE / MMAS; s < (n + 1) * SIDE / MMAS; ++s) {                                                   \
            if (s < READS) read(BUF, KS, s, G2);                                                                                            \
            else piece(LBUF, s - READS);                                                                                                    \
        }                                                                                                                                   \
        __builtin_amdgcn_sched_barrier(0);                                                                                                  \
    }
    auto landed = [&](auto left) {       // all chunks in flight but the newest `left` are complete, in every wave, and so are all reads
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(decltype(left)::value * NPIECE) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // Fragments are read one half chunk ahead of their products; the barrier sits between the two halves, behind products already issued, and
    // frees the stage whose second half has just been read: its refill has NS - 1 chunks of products to arrive in.
    Frags f0, f1;
    if (!SPLIT || !join)
#pragma unroll
    for (int s = 0; s < NS; ++s, ++nC)
#pragma unroll
        for (int x = 0; x < NPIECE; ++x) piece(s, x);
    // the scalars of the epilogue, fetched behind the first loads
    const float* info = info_of(g, inst);
    const float fx = J.first ? info[0] : 1.f / info[I_SX + J.t];
    float mult = J.mul;
    if (J.kind == GRAM) mult = fx * fx * info[I_SA + J.t];
    else if (J.kind == POLY) mult = 1.f / (info[I_SA + J.t] * info[I_SA + J.t]);
    else if (J.kind == PROD_A) mult = J.mul * (info[I_SA + J.t2] / info[I_SA + J.t]);
    else if (J.kind == APPLY_MID) mult = J.mul * fx * info[I_SX + J.t2];
    else if (J.kind == APPLY_OUT) mult = J.mul * fx;
    const float isa = J.kind == POLY ? 1.f / info[I_SA + J.t] : 0.f;
    if (!SPLIT || !join) {
        landed(std::integral_constant<int, NS - 1>());
        if (KC == 1)
#pragma unroll
            for (int x = 0; x < READS; ++x) read(0, 0, x, f0);
    }
    int cur = 0;
    if constexpr (KC == 2) {
        // One 32 x 32 block a wave: three products a half chunk, over before a fragment read or a barrier is.  So a stage of two chunks at a time: its
        // four halves' fragments are read under the products of the stage before, cross terms into an accumulator of their own.
        static_assert(TM == 1 && TN == 1, "one block a wave");
        Frags e[4], o[4];
        f32x16 cross;
#pragma unroll
        for (int r = 0; r < 16; ++r) cross[r] = 0.f;
        auto read4 = [&](int buf, int x, Frags (&f)[4]) {
            const unsigned char* base = smem + buf * STAGE + (x >> 1) * CHUNK;
#pragma unroll
            for (int pl = 0; pl < NA; ++pl) f[x].a[0][pl] = *reinterpret_cast<const half8*>(base + a_rd + (a_sl ^ ((x & 1) * 32 + pl * 64)));
#pragma unroll
            for (int pl = 0; pl < NB; ++pl) f[x].b[0][pl] = *reinterpret_cast<const half8*>(base + b_rd + (b_sl ^ ((x & 1) * 32 + pl * 64)));
        };
        auto mma4 = [&](const Frags& f) {
            if (NA > 1) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[0][NA - 1], f.b[0][0], cross, 0, 0, 0);
            acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[0][0], f.b[0][0], acc[0][0], 0, 0, 0);
            if (NB > 1) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[0][0], f.b[0][NB - 1], cross, 0, 0, 0);
        };
        auto step = [&](const Frags (&f)[4], Frags (&nf)[4]) {
            landed(std::integral_constant<int, NS - 2>());          // the next stage; this one's fragments are in registers
            const int old = cur;
            cur = cur + 1 == NS ? 0 : cur + 1;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                read4(cur, h, nf);
#pragma unroll
                for (int x = h * NPIECE / 4; x < (h + 1) * NPIECE / 4; ++x) piece(old, x);
                mma4(f[h]);
                __builtin_amdgcn_sched_barrier(0);
            }
            ++nC;
        };
        const int stages = SPLIT && join ? 0 : (nk + 1) / 2;
        if (!SPLIT || !join)
#pragma unroll
            for (int h = 0; h < 4; ++h) read4(0, h, e);
        for (int t = 0; t < stages; t += 2) {                   // (a stage behind the last one is zeros)
            step(e, o);
            step(o, e);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][0][r] += cross[r];
    } else
    for (int kt = 0; kt < nk; ++kt) {
        ORTHO_MMA(f0, f1, cur, 1, 0, 0)
        landed(std::integral_constant<int, NS - 2>());
        const int old = cur;
        cur = cur + 1 == NS ? 0 : cur + 1;
        ORTHO_MMA(f1, f0, cur, 0, 1, old)      // (behind the last chunk the fragments read are not used)
        ++nC;
    }
#undef ORTHO_MMA
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // the loads behind the last chunk: the LDS is used again below
    __syncthreads();
    if constexpr (SPLIT) {
        static_assert(TM == 1 && TN == 1, "one block a wave");
        float* slot = (float*)(g.ws + g.part) + (int64_t)slot0 * (BM * BN) + (wave * 256 + lane) * 4;
        if (parts > 1 && !join) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(slot + q * 256) = make_float4(acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]);
            return;
        }
        if (join)
#pragma unroll 4
            for (int s = 0; s < parts; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = *reinterpret_cast<const float4*>(slot + (int64_t)s * (BM * BN) + q * 256);
                    acc[0][0][4 * q] += v.x; acc[0][0][4 * q + 1] += v.y; acc[0][0][4 * q + 2] += v.z; acc[0][0][4 * q + 3] += v.w;
                }
    }

    // ---- epilogue: a lane holds column lane & 31 and rows 8 q + 4 (lane >> 5) + 0..3 of every 32 x 32 block.  A wave puts E x E results into its
    // own part of the LDS and reads them back in rows of either orientation: 16-byte stores over whole cache lines.
    constexpr int LDH = 2 * E + 8;                    // bytes of an fp16 row in LDS (E rows of each plane)
    constexpr int LDF = E + 4;                        // floats of an fp32 row in LDS
    unsigned char* mine = smem + wave * (E * LDF * 4);
    static_assert(2 * E * LDH == E * LDF * 4, "one region for both forms");
    auto fence = [&]() { asm volatile("" ::: "memory"); };      // a wave's LDS operations execute in order

    if (J.kind == APPLY_OUT) {
        const bool wide = mat.M <= mat.N;             // rows of the result are rows of X, or of X^T
        const int64_t ob = b * mat.out_bs;
        const int size = g.dtype == WGS_F32 ? 4 : 2;
        const bool vec = mat.out_rs % 4 == 0 && ob % 4 == 0 && ((uintptr_t)mat.out & (4 * size - 1)) == 0;
        const int rows = wide ? d.m : d.n, cols = wide ? d.n : d.m;
        float* lds = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int bi = 0; bi < WM / E; ++bi)
#pragma unroll
            for (int bj = 0; bj < WN / E; ++bj) {
                fence();
#pragma unroll
                for (int i = 0; i < E / 32; ++i)
#pragma unroll
                    for (int j = 0; j < E / 32; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const f32x16& v = acc[bi * (E / 32) + i][bj * (E / 32) + j];
                            const int c = j * 32 + l31, r = i * 32 + 8 * q + 4 * lh;
                            if (wide) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) lds[(r + k) * LDF + c] = v[4 * q + k] * mult;
                            } else {
                                *reinterpret_cast<float4*>(lds + c * LDF + r) = make_float4(v[4 * q] * mult, v[4 * q + 1] * mult, v[4 * q + 2] * mult, v[4 * q + 3] * mult);
                            }
                        }
                fence();
                const int rb = i0 + wm * WM + bi * E, cb = j0 + wn * WN + bj * E;
                const int r0 = wide ? rb : cb, c0 = wide ? cb : rb;
#pragma unroll 4
                for (int x = lane; x < E * E / 4; x += 64) {
                    const int r = x / (E / 4), c = (x % (E / 4)) * 4;
                    const float4 f = *reinterpret_cast<const float4*>(lds + r * LDF + c);
                    float v[4] = {f.x, f.y, f.z, f.w};
                    if (r0 + r >= rows || c0 + c >= cols) continue;
                    const int64_t at = ob + (int64_t)(r0 + r) * mat.out_rs + c0 + c;
                    const bool full = vec && c0 + c + 4 <= cols;
                    char* o = (char*)mat.out + at * size;
                    if (g.step) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (full || c0 + c + k < cols) v[k] = mat.decay * load_as(g.dtype, mat.out, at + k) - mat.step * v[k];
                    }
                    if (full) {
                        if (size == 4) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
                        else if (g.dtype == WGS_BF16) {
                            typedef __bf16 b4 __attribute__((ext_vector_type(4)));
                            *reinterpret_cast<b4*>(o) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
                        } else *reinterpret_cast<half4*>(o) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (c0 + c + k < cols) store_as(g.dtype, mat.out, at + k, v[k]);
                    }
                }
            }
        return;
    }
    const bool mid = J.kind == APPLY_MID;
    const Plane D = plane_of(g, mat, d, b, J.dst);                              // [i][j]
    const Plane T = mid ? plane_of(g, mat, d, b, J.dst2) : D;                   // [j][i]
    const Plane S = J.kind == POLY ? plane_of(g, mat, d, b, J.src) : D;
    const int nc = mid ? d.n : d.m;
    unsigned char* lo = mine + E * LDH;               // LDS: [c][r] of the hi parts, then of the lo parts
#pragma unroll
    for (int bi = 0; bi < WM / E; ++bi)
#pragma unroll
        for (int bj = 0; bj < WN / E; ++bj) {
            const int rb = i0 + wm * WM + bi * E, cb = j0 + wn * WN + bj * E;
            // A tile on the diagonal computes both triangles, whose roundings differ where the factors do not quite commute: the strict upper
            // one is dropped, else the iteration amplifies the antisymmetric part (measured: ten times the error on spiked spectra).
            if (!mid && rb < cb) continue;
            const bool half = !mid && rb == cb;
            fence();
            if (J.kind == POLY) {                     // A's block, by symmetry in rows c
#pragma unroll 4
                for (int x = lane; x < E * E / 8; x += 64) {
                    const int c = x / (E / 8), r = (x % (E / 8)) * 8;
                    if (cb + c < d.m && rb + r < S.ld) {
                        const unsigned char* q = at_hi(S, cb + c, rb + r);
                        const uint4 h = *reinterpret_cast<const uint4*>(q), l = *reinterpret_cast<const uint4*>(q + 64);
                        uint2* wh = reinterpret_cast<uint2*>(mine + c * LDH + r * 2);
                        uint2* wl = reinterpret_cast<uint2*>(lo + c * LDH + r * 2);
                        wh[0] = make_uint2(h.x, h.y); wh[1] = make_uint2(h.z, h.w);
                        wl[0] = make_uint2(l.x, l.y); wl[1] = make_uint2(l.z, l.w);
                    }
                }
                fence();
            }
#pragma unroll
            for (int i = 0; i < E / 32; ++i)
#pragma unroll
                for (int j = 0; j < E / 32; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x16& av = acc[bi * (E / 32) + i][bj * (E / 32) + j];
                        const int c = j * 32 + l31, r = i * 32 + 8 * q + 4 * lh;
                        half4* ph = reinterpret_cast<half4*>(mine + c * LDH + r * 2);
                        half4* pl = reinterpret_cast<half4*>(lo + c * LDH + r * 2);
                        half4 sh, sl;
                        if (J.kind == POLY) { sh = *ph; sl = *pl; }
                        half4 h, l;
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            v[k] = av[4 * q + k] * mult;
                            if (J.kind == POLY) {
                                const float A = ((float)sh[k] + (float)sl[k]) * isa;
                                v[k] = ((rb + r + k == cb + c ? J.a : 0.f) + (J.b * A + J.c * v[k])) * J.mul;
                            }
                            if (rb + r + k >= d.m || cb + c >= nc) v[k] = 0.f;      // the padding of both planes
                        }
                        split_many<4>(v, h, l);
                        *ph = h; *pl = l;
                    }
            fence();
            auto at = [&](const unsigned char* plane, int c, int r) { return *reinterpret_cast<const unsigned short*>(plane + c * LDH + r * 2); };
            // rows c of T; a block on the diagonal takes what lies over it from the other side
#pragma unroll 2
            for (int x = lane; x < E * E / 8; x += 64) {
                const int c = x / (E / 8), r = (x % (E / 8)) * 8;
                if (cb + c >= nc || rb + r >= T.ld) continue;
                unsigned char* o = at_hi(T, cb + c, rb + r);
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    const unsigned char* src = pl ? lo : mine;
                    const uint2 u0 = *reinterpret_cast<const uint2*>(src + c * LDH + r * 2), u1 = *reinterpret_cast<const uint2*>(src + c * LDH + r * 2 + 8);
                    unsigned w[4] = {u0.x, u0.y, u1.x, u1.y};
                    if (half && r < c) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (r + k < c) {
                                const unsigned v = at(src, r + k, c);
                                w[k / 2] = (k & 1) ? (w[k / 2] & 0xffffu) | (v << 16) : (w[k / 2] & 0xffff0000u) | v;
                            }
                    }
                    *reinterpret_cast<uint4*>(o + pl * 64) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            if (half) continue;
            // rows r of D
#pragma unroll 2
            for (int x = lane; x < E * E / 8; x += 64) {
                const int r = x / (E / 8), c = (x % (E / 8)) * 8;
                if (rb + r >= d.m || cb + c >= D.ld) continue;
                unsigned char* o = at_hi(D, rb + r, cb + c);
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    const unsigned char* src = pl ? lo : mine;
                    unsigned w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = at(src, c + 2 * k, r) | (unsigned)at(src, c + 2 * k + 1, r) << 16;
                    *reinterpret_cast<uint4*>(o + pl * 64) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
}

// ---- 4. a whole phase's polynomial for m <= 128, one workgroup a matrix -----------------------------------------------------------------------------
// From the Gram matrix A (read once) to Q (written once): per iteration B = aI + bA + cA^2, P = B A beside Q <- B Q, A = P B, with A (or P) and B in
// LDS as hi and lo planes and Q in registers: a wave a block of 32 columns, whose result layout is the next product's operand (as in the small
// kernel).  Symmetric products: the tiles on and under the diagonal, written twice.  Some 14 us an iteration at
// m = 128 (the latency of its dependent products and LDS) instead of three launches of some 9: 64 x 128x512 fp16 176 -> 132 us, one in bf16 158 -> 91.
constexpr int CHAIN_M = 128;
struct ChainArgs { int t0, len, src, dst; float a, b, c; float sb[MAX_STEPS], grow[MAX_STEPS], sq[MAX_STEPS]; };      // grow: 2^ceil log2 of B's bound; sq: Q' scale / (Q scale sb)
template <int MT>
__global__ __launch_bounds__(512, 1) void ortho_chain_kernel(const Group g, const ChainArgs ar) {
    constexpr int S = 32 * MT, LD = S + 8, TRI = MT * (MT + 1) / 2;
    typedef _Float16 plane_t[S][LD];
    __shared__ __attribute__((aligned(16))) plane_t la[2], lb[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, lh = lane >> 5;
    const Mat& mat = g.mat[entry_of(g, blockIdx.x)];
    const int b = blockIdx.x - mat.first;
    const Dims d = dims_of(mat.M, mat.N);
    const float* info = info_of(g, blockIdx.x);
    const Plane A = plane_of(g, mat, d, b, ar.src), Q = plane_of(g, mat, d, b, ar.dst);

    for (int e = tid; e < S * (S / 8); e += 512) {
        const int r = e / (S / 8), c = (e % (S / 8)) * 8;
        uint4 h = make_uint4(0, 0, 0, 0), l = h;
        if (r < d.m && c < d.mp) { h = *reinterpret_cast<const uint4*>(at_hi(A, r, c)); l = *reinterpret_cast<const uint4*>(at_hi(A, r, c) + 64); }
        *reinterpret_cast<uint4*>(&la[0][r][c]) = h;
        *reinterpret_cast<uint4*>(&la[1][r][c]) = l;
    }
    auto place = [](int t, int& p, int& q) { p = 0; while (t > p) { t -= p + 1; ++p; } q = t; };
    auto product = [&](const plane_t (&x)[2], const plane_t (&y)[2], int p, int q) {      // rows of tile p of x times rows of tile q of y
        f32x16 s, w;
#pragma unroll
        for (int k = 0; k < 16; ++k) { s[k] = 0.f; w[k] = 0.f; }
#pragma unroll
        for (int ks = 0; ks < 2 * MT; ++ks) {
            const int kc = 16 * ks + 8 * lh;
            const half8 ah = *reinterpret_cast<const half8*>(&x[0][32 * p + l31][kc]), al = *reinterpret_cast<const half8*>(&x[1][32 * p + l31][kc]);
            const half8 bh = *reinterpret_cast<const half8*>(&y[0][32 * q + l31][kc]), bl = *reinterpret_cast<const half8*>(&y[1][32 * q + l31][kc]);
            w = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, w, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, s, 0, 0, 0);
            w = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, w, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) s[k] += w[k];
        return s;
    };
    auto put = [&](plane_t (&x)[2], int p, int q, int k4, float (&v)[4]) {      // elements 4 k4 .. + 3 of tile (p, q), rows r .. r + 3 of a column, and their mirror
        const int r = 32 * p + 8 * k4 + 4 * lh, c = 32 * q + l31;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r + k >= d.m || c >= d.m) v[k] = 0.f;
        half4 h, l;
        split_many<4>(v, h, l);
        _Float16 *dh = &x[0][r][c], *dl = &x[1][r][c], *mh = &x[0][c][r], *ml = &x[1][c][r];
        if (p != q) {
            *reinterpret_cast<half4*>(mh) = h;
            *reinterpret_cast<half4*>(ml) = l;
#pragma unroll
            for (int k = 0; k < 4; ++k) { dh[k * LD] = h[k]; dl[k * LD] = l[k]; }
        } else {                                                                   // not the strict upper triangle of a diagonal tile
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (r + k >= c) { dh[k * LD] = h[k]; dl[k * LD] = l[k]; mh[k] = h[k]; ml[k] = l[k]; }
        }
    };
    frag qh[MT][2], ql[MT][2];          // waves 0 .. 3: Q's columns 32 wave ..: lane = column, 8 rows a fragment
    __syncthreads();
    for (int it = 0; it < ar.len; ++it) {
        const int t = ar.t0 + it;
        const float sA = info[I_SA + t], isa = 1.f / sA, sb = ar.sb[it];
        const bool last = it + 1 == ar.len;
        for (int e = wave; e < TRI; e += 8) {
            int p, q;
            place(e, p, q);
            const f32x16 s = product(la, la, p, q);
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
                const int r = 32 * p + 8 * k4 + 4 * lh, c = 32 * q + l31;
                const half4 h = *reinterpret_cast<const half4*>(&la[0][c][r]), l = *reinterpret_cast<const half4*>(&la[1][c][r]);      // A by symmetry
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[k] = ((r + k == c ? ar.a : 0.f) + (ar.b * (((float)h[k] + (float)l[k]) * isa) + ar.c * (s[4 * k4 + k] * isa * isa))) * sb;
                put(lb, p, q, k4, v);
            }
        }
        __syncthreads();
        f32x16 acc[3];
        if (wave >= 4) {
            if (!last)
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (wave - 4 + 4 * i < TRI) {
                        int p, q;
                        place(wave - 4 + 4 * i, p, q);
                        acc[i] = product(lb, la, p, q);
                    }
        } else if (wave < MT) {
            auto pick = [&](int pl, int row, int k0) {          // 8 values of a row of B in the order of a result's rows
                const int2 u = *reinterpret_cast<const int2*>(&lb[pl][row][k0 + 4 * lh]), w = *reinterpret_cast<const int2*>(&lb[pl][row][k0 + 4 * lh + 8]);
                return frag{u.x, u.y, w.x, w.y};
            };
            if (it == 0) {
#pragma unroll
                for (int u = 0; u < MT; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) { qh[u][h] = pick(0, 32 * wave + l31, 32 * u + 16 * h); ql[u][h] = pick(1, 32 * wave + l31, 32 * u + 16 * h); }
            } else {
                f32x16 s[MT];
#pragma unroll
                for (int u = 0; u < MT; ++u) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) s[u][k] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < 2 * MT; ++ks) {
                        const half8 bh = __builtin_bit_cast(half8, pick(0, 32 * u + l31, 16 * ks)), bl = __builtin_bit_cast(half8, pick(1, 32 * u + l31, 16 * ks));
                        const half8 vh = __builtin_bit_cast(half8, qh[ks >> 1][ks & 1]), vl = __builtin_bit_cast(half8, ql[ks >> 1][ks & 1]);
                        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl, vh, s[u], 0, 0, 0);
                        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh, vl, s[u], 0, 0, 0);
                        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh, vh, s[u], 0, 0, 0);
                    }
                }
                const float f = ar.sq[it];
#pragma unroll
                for (int u = 0; u < MT; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[8];
                        half8 x, y;
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = s[u][8 * h + k] * f;
                        split_many<8>(v, x, y);
                        qh[u][h] = __builtin_bit_cast(frag, x); ql[u][h] = __builtin_bit_cast(frag, y);
                    }
            }
        }
        if (last) break;
        __syncthreads();
        if (wave >= 4) {
            const float f = 1.f / (ar.grow[it] * sb);
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (wave - 4 + 4 * i < TRI) {
                    int p, q;
                    place(wave - 4 + 4 * i, p, q);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v[4] = {acc[i][4 * k] * f, acc[i][4 * k + 1] * f, acc[i][4 * k + 2] * f, acc[i][4 * k + 3] * f};
                        put(la, p, q, k, v);
                    }
                }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (wave + 8 * i < TRI) {
                int p, q;
                place(wave + 8 * i, p, q);
                acc[i] = product(la, lb, p, q);
            }
        __syncthreads();
        const float f = ar.grow[it] / sb * (info[I_SA + t + 1] / sA);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (wave + 8 * i < TRI) {
                int p, q;
                place(wave + 8 * i, p, q);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[4] = {acc[i][4 * k] * f, acc[i][4 * k + 1] * f, acc[i][4 * k + 2] * f, acc[i][4 * k + 3] * f};
                    put(la, p, q, k, v);
                }
            }
        __syncthreads();
    }
    const int row = 32 * wave + l31;          // Q is symmetric: a lane's column is a row
    if (wave < MT && row < d.m)
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int k = 32 * u + 16 * h + 8 * x + 4 * lh;
                    if (k < d.mp) {
                        *reinterpret_cast<int2*>(at_hi(Q, row, k)) = make_int2(qh[u][h][2 * x], qh[u][h][2 * x + 1]);
                        *reinterpret_cast<int2*>(at_hi(Q, row, k) + 64) = make_int2(ql[u][h][2 * x], ql[u][h][2 * x + 1]);
                    }
                }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
struct Plan { int phases, len[MAX_STEPS]; int planes, npx, nt, ns; };
// Iterations of a phase.  Longer phases leave out products with the n columns, but A_t then carries its own rounding through a^2 a step instead
// of being formed anew from X_t.  Distance from the exact factor before the result is rounded (relative, Frobenius; 48 x 600 .. 2048 x 2048, fp32
// in and out), against the iteration on 32-bit library products:
//                                        32-bit    single    (3, 2)    five
//   noise, rows of uneven size           5e-6      2e-6      6e-6      9e-6
//   one direction in noise of 0.1        5e-6      2e-6      5e-6      3e-4
//   ... of 0.01                          5e-5      2e-5      2e-5      6e-4
//   ... of 0.001, 0.0001                 4e-4      1.3e-4    1.3e-4    6e-4
//   eight directions in noise of 0.01    6e-5      4e-5      3e-5      2e-4
//   a third of the rank; 5 decades       9e-6      1.3e-5    8e-6      3e-4
// Single iterations are at most 1.4 times as far as 32-bit products (mostly nearer: the sums have fewer roundings), (3, 2) as good as they.  (A single
// matrix of 17 .. 24 rows can be up to 2.5 times as far: two draws of a few roundings.  Up to 16 rows go through ortho_tiny_kernel.)
// Five are not: they put a bf16 result up to 11 % further from the exact factor than its rounding does, and save 1.4 ms of 6.1 at 4096 x 16384
// (single iterations: 10.3), 30 us of 136 at 64 of 128 x 512.  So bf16 takes five, fp16 three, fp32 one, where the caller names no number;
// nearly square matrices of over 128 rows, whose products with X cost no more than those they replace, one whatever the type (bf16 singles / (3, 2) /
// five: 1024^2 217 / 251 / 245 us, 2048^2 874 / 977 / 958, 4096^2 3.45 / 3.69 / 3.75 ms; but 4096 x 4608 4.47 / 4.06 / 3.89).
Plan plan_of(int dtype, bool step, int steps, const wgs_matrix* mats, int count) {
    Plan p;
    int most = count ? mats[0].joined : 1;
    if (!most) {
        most = 1;
        if (dtype != WGS_F32)
            for (int i = 0; i < count; ++i) {
                const Dims d = dims_of(mats[i].rows, mats[i].cols);
                if (mats[i].batch && !is_tiny(d, dtype) && (d.m <= 128 || d.n - d.m > d.m / 16)) most = dtype == WGS_BF16 ? 5 : 3;
            }
    }
    p.phases = (steps + most - 1) / most;
    int longest = 0;
    for (int i = 0, left = steps; i < p.phases; ++i) {
        p.len[i] = (left + p.phases - i - 1) / (p.phases - i);
        left -= p.len[i];
        if (p.len[i] > longest) longest = p.len[i];
    }
    p.planes = (dtype == WGS_F32 || step) ? 2 : 1;
    p.npx = p.phases > 1 ? 2 : p.planes;
    p.nt = p.phases > 1 ? 2 : 1;
    p.ns = longest > 1 ? 5 : 2;
    return p;
}

constexpr int64_t CHUNK_BYTES = 4LL << 30;       // planes of the matrices that go through the launches together
// Workgroups of 512 of the norm's launch: a grid has fewer than 2^32 threads.  (All matrices of a run take the largest one's number of parts: without
// the limit one of 2048^2 beside a batch of 33000 single entries would pass it.)
constexpr int64_t NORM_BLOCKS = 1 << 22;
int norm_blocks(int64_t elements) {               // 64 elements a thread where the matrix is large
    const int64_t sb = elements / 16384;
    return sb < 1 ? 1 : (sb > STAT_BLOCKS ? STAT_BLOCKS : (int)sb);
}

constexpr int64_t TINY_BLOCKS = 1 << 22;         // (the same for the matrices of up to 16 rows, a workgroup of 256 each)

// The matrices, those of up to 16 rows or the others, in runs of at most MAX_MATS entries, NORM_BLOCKS (TINY_BLOCKS) and CHUNK_BYTES (or one matrix);
// batches are cut where they have to be.
struct Cursor { int entry = 0, done = 0; };
int64_t next_chunk(const wgs_matrix* mats, int count, const Plan& p, bool tiny, Cursor& c, Group& g) {
    int64_t bytes = 0;
    g.count = 0; g.instances = 0;
    int64_t most = 0;
    while (c.entry < count && g.count < MAX_MATS) {
        const wgs_matrix& w = mats[c.entry];
        const int left = w.batch - c.done;
        const Dims d = dims_of(w.rows, w.cols);
        if (left <= 0 || is_tiny(d, g.dtype) != tiny) { ++c.entry; c.done = 0; continue; }
        int64_t one = tiny ? tiny_bytes(d) : instance_bytes(d, p.npx, p.nt, p.ns);
        if (!tiny && is_small(d) && small_bytes(d) > one) one = small_bytes(d);
        const int64_t elements = (int64_t)w.rows * w.cols, largest = elements > most ? elements : most;
        int64_t fit = (CHUNK_BYTES - bytes) / one;
        if (fit < 1 && !g.count) fit = 1;
        const int64_t room = (tiny ? TINY_BLOCKS : NORM_BLOCKS / norm_blocks(largest)) - g.instances;
        if (fit > room) fit = room;
        if (fit < 1) break;
        const int take = fit < left ? (int)fit : left;
        Mat& m = g.mat[g.count++];
        m.in_bs = w.in_batch_stride; m.out_bs = w.out_batch_stride;
        m.momentum = nullptr;
        m.ws = bytes; m.in_rs = (int)w.in_row_stride; m.out_rs = (int)w.out_row_stride;
        m.M = w.rows; m.N = w.cols; m.batch = take; m.first = g.instances; m.step = w.step; m.decay = w.decay;
        // instances before this part of the batch
        const int64_t size = g.dtype == WGS_F32 ? 4 : 2;
        m.in = (const char*)w.in + (int64_t)c.done * w.in_batch_stride * size;
        m.out = (char*)w.out + (int64_t)c.done * w.out_batch_stride * size;
        if (w.momentum) m.momentum = w.momentum + (int64_t)c.done * w.rows * w.cols;
        g.instances += take;
        bytes += one * take;
        most = largest;
        c.done += take;
        if (c.done == w.batch) { ++c.entry; c.done = 0; }
        if (take < left) break;
    }
    if (!g.count) return 0;
    if (tiny) return bytes;
    g.stat_blocks = norm_blocks(most);
    g.info = up((int64_t)g.instances * g.stat_blocks * (int64_t)sizeof(Part), 256);
    int64_t head = g.info + up((int64_t)g.instances * INFO * 4, 256);
    g.part = 0;
    for (int i = 0; i < g.count; ++i)
        if (dims_of(g.mat[i].M, g.mat[i].N).np / BK > 40) g.part = head;
    if (g.part) head += SPLIT_BYTES;
    for (int i = 0; i < g.count; ++i) g.mat[i].ws += head;
    return head + bytes;
}

const char* check_mats(const wgs_matrix* mats, int count, int dtype, bool step, int steps) {
    if (dtype != WGS_F32 && dtype != WGS_BF16 && dtype != WGS_F16) return "unknown dtype";
    if (count < 0 || (count && !mats)) return "no matrices";
    if (steps < 1 || steps > MAX_STEPS) return "steps must be 1 .. 16";
    for (int i = 0; i < count; ++i) {
        const wgs_matrix& w = mats[i];
        if (w.rows < 1 || w.cols < 1 || w.batch < 0 || (int64_t)w.rows * up(w.cols, BK) >= (1LL << 29) || (int64_t)w.cols * up(w.rows, BK) >= (1LL << 29))
            return "bad sizes (rows, cols >= 1, fewer than 2^29 elements with the smaller side's padding to 32)";
        if (w.in_row_stride < w.cols || w.out_row_stride < w.cols || w.in_row_stride >= (1LL << 31) || w.out_row_stride >= (1LL << 31)) return "row strides must be at least cols";
        if (w.batch > 1 && (w.in_batch_stride < 0 || w.out_batch_stride < (int64_t)(w.rows - 1) * w.out_row_stride + w.cols)) return "batch strides overlap";
        if (w.joined < 0 || w.joined > MAX_STEPS || w.joined != mats[0].joined) return "joined must be 0 .. 16 and the same in all matrices of a call";
        if (w.batch > (1 << 20)) return "batch must be at most 2^20";
        if (w.batch && (!w.in || !w.out || (step && !w.momentum))) return "null pointer";
        const uintptr_t am = dtype == WGS_F32 ? 3 : 1;
        if ((((uintptr_t)w.in | (uintptr_t)w.out) & am) || ((uintptr_t)w.momentum & 3)) return "a matrix is not aligned to its type";
    }
    return nullptr;
}

int64_t workspace(const wgs_matrix* mats, int count, int dtype, bool step, int steps) {
    const Plan p = plan_of(dtype, step, steps, mats, count);
    Group g;
    g.dtype = dtype;
    int64_t need = 0;
    for (bool tiny : {true, false}) {
        Cursor c;
        while (const int64_t b = next_chunk(mats, count, p, tiny, c, g))
            if (b > need) need = b;
    }
    return need;
}

// the largest |a + b l + c l^2| on [0, top], and of l (a + b l + c l^2)^2
void poly_bounds(double a, double b, double c, double top, double* q, double* next) {
    auto f = [&](double l) { return a + l * (b + l * c); };
    double mq = fmax(fabs(f(0.0)), fabs(f(top))), mn = top * f(top) * f(top);
    if (c != 0.0) {
        const double v = -b / (2 * c);
        if (v > 0 && v < top) mq = fmax(mq, fabs(f(v)));
    }
    // d/dl l q^2 = q (a + 3 b l + 5 c l^2): where q = 0 the product is 0
    double r[2];
    int n = 0;
    if (c != 0.0) {
        const double disc = 9 * b * b - 20 * a * c;
        if (disc >= 0) { r[n++] = (-3 * b + sqrt(disc)) / (10 * c); r[n++] = (-3 * b - sqrt(disc)) / (10 * c); }
    } else if (b != 0.0) r[n++] = -a / (3 * b);
    for (int i = 0; i < n; ++i)
        if (r[i] > 0 && r[i] < top) mn = fmax(mn, r[i] * f(r[i]) * f(r[i]));
    *q = mq; *next = mn;
}
int ceil_log2(double v) { int e; const double f = frexp(v, &e); return f == 0.5 ? e - 1 : e; }

template <int NA, int NB, int BM, int WM, int WN, int NS, int E, bool SPLIT = false>
void launch_gemm(const Group& g, const Jobs& js, int total, hipStream_t st, int most = 1, int join = 0) {
    constexpr int stages = NS * (BM == 64 ? 2 : 1) * (NA + NB) * BM * ROW, blocks = WM * WN * E * (E + 4) * 4;
    constexpr int sm = stages > blocks ? stages : blocks;
    static_assert(sm <= 160 * 1024, "LDS of a CU");
    auto k = ortho_gemm_kernel<NA, NB, BM, WM, WN, NS, E, SPLIT>;
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, sm);
    const int per = (total + 7) / 8, run = (per + (per + 31) / 32 - 1) / ((per + 31) / 32);
    WGS_LAUNCH(k, dim3((unsigned)((per + run - 1) / run * run * 8)), dim3(64 * WM * WN), sm, st, js, total, run, most, join, g);
}
int tiles_of(const Group& g, const Jobs& js, int bm, int most = 1) {
    int64_t t = 0;
    for (int i = 0; i < g.count; ++i) {
        const Dims d = dims_of(g.mat[i].M, g.mat[i].N);
        const int64_t tm = (d.m + bm - 1) / bm, tn = (d.n + bm - 1) / bm;
        t += g.mat[i].batch * (js.sym ? tm * (tm + 1) / 2 : tm * tn) * parts_of_sum((js.kgram ? d.np : d.mp) / BK, most);
    }
    t *= js.count;
    return t < (1LL << 30) ? (int)t : 0;
}
template <int NA, int NB>
int gemm(const Group& g, const Jobs& js, hipStream_t st) {
    // Tile side.  Cost of a choice: rounds of tiles over the CUs (two workgroups a CU up to 128) times a tile's area; half of it by the mean,
    // since CUs that a last round leaves idle let the others clock higher (the products run at the card's power limit).
    int bm = 64;
    double best = 1e300;
    for (int s : {64, 128, 192, 256}) {
        const int t = tiles_of(g, js, s);
        if (t <= 0) continue;
        const double slots = s <= 128 ? 512 : 256, rounds = 0.5 * (ceil(t / slots) + t / slots);
        const double cost = rounds * s * s * (s == 64 ? 2 * 1.6 : s == 128 ? 2 * 1.1 : 1.0);
        if (cost < best) { best = cost; bm = s; }
    }
    const int total = tiles_of(g, js, bm);
    WGS_CHECK_ARG(total > 0, "orthogonalise: too many matrices for one launch");
    if (bm == 256) launch_gemm<NA, NB, 256, 2, 4, 2, 64>(g, js, total, st);
    else if (bm == 192) launch_gemm<NA, NB, 192, 2, 2, 3, 96>(g, js, total, st);
    else if (bm == 128) launch_gemm<NA, NB, 128, 2, 2, 2, 64>(g, js, total, st);
    else if (total <= 256) {
        // Parts where the tiles leave half the CUs idle, up to three workgroups a CU, and where they save over 40 chunks (some 0.24 us each) of the
        // longest sum for a second launch of some 8 us (512 x 4608 fp32: 403 -> 303 us; with 136 and 216 tiles: 402 -> 438, 738 -> 827).
        int most = 1, longest = 0;
        for (int i = 0; i < g.count; ++i) {
            const Dims d = dims_of(g.mat[i].M, g.mat[i].N);
            const int nk = (js.kgram ? d.np : d.mp) / BK;
            if (nk > longest) longest = nk;
        }
        if (g.part && js.count == 1 && total <= 128)
            for (int x = 2; x <= 16 && tiles_of(g, js, 64, x) <= 768; ++x) most = x;
        if (longest - longest / parts_of_sum(longest, most) > 40) {
            launch_gemm<NA, NB, 64, 2, 2, 2, 32, true>(g, js, tiles_of(g, js, 64, most), st, most);
            launch_gemm<NA, NB, 64, 2, 2, 2, 32, true>(g, js, total, st, most, 1);
        } else launch_gemm<NA, NB, 64, 2, 2, 4, 32>(g, js, total, st);
    }
    else launch_gemm<NA, NB, 64, 2, 2, 2, 32>(g, js, total, st);
    return WGS_OK;
}

template <int DT, bool STEP>
void launch_norm(const Group& g, const Momentum& mo, hipStream_t st) {
    WGS_LAUNCH((ortho_norm_kernel<DT, STEP>), dim3((unsigned)(g.instances * g.stat_blocks)), dim3(512), 0, st, g, mo);
}
template <int DT, bool STEP>
void launch_prepare(const Group& g, const Momentum& mo, const Bounds& bd, hipStream_t st) {
    launch_norm<DT, STEP>(g, mo, st);
    int64_t tiles = 0;
    for (int i = 0; i < g.count; ++i) tiles += (int64_t)g.mat[i].batch * ((up(g.mat[i].M, BK) + 63) / 64) * ((up(g.mat[i].N, BK) + 63) / 64);
    WGS_LAUNCH((ortho_split_kernel<DT, STEP>), dim3((unsigned)tiles), dim3(256), 0, st, g, mo, bd, (int)tiles);
}

bool all_small(const Group& g, const Plan& p, int steps) {
    // Single iterations: always.  Joined ones with m > 32 go on through the chain kernel, whose launches outweigh its work up to some 1000 phases / steps
    // columns (64 x 64 bf16 35 us here, 45 there, 64 x 256 48 / 47, 64 x 1000 113 / 51; fp16, two phases: 64 x 256 48 / 64, 64 x 576 80 / 67).
    const bool joined = p.phases < steps;
    for (int i = 0; i < g.count; ++i) {
        const Dims d = dims_of(g.mat[i].M, g.mat[i].N);
        if (!is_small(d) || (joined && d.m > 32 && d.n * steps > 1000 * p.phases)) return false;
    }
    return true;
}
void launch_small(const Group& g, const Momentum& mo, SmallArgs ar, hipStream_t st) {
    int m = 0, n = 0;
    ar.parts = 1;
    for (int i = 0; i < g.count; ++i) {
        const Dims d = dims_of(g.mat[i].M, g.mat[i].N);
        if (d.m > m) m = d.m;
        if (d.n > n) n = d.n;
        if (small_parts(d) > ar.parts) ar.parts = (int)small_parts(d);
    }
    // A step of its own launch costs some 9 us (m = 64) or 6 (m = 32) almost whatever n is, in one launch it grows with the blocks of a wave; but a workgroup
    // takes a CU.  One matrix in fp32: 64 x 384 (two blocks a wave) 62 against some 65 us, 64 x 576 80 / 67, 64 x 1000 113 / 69, 32 x 640 (three blocks) 43 / 42,
    // 32 x 1000 57 / 45, 32 x 2000 97 / 49; 64 of 64 x 1000 116 / 92.
    if (n <= 32 * SMALL_WAVES * (m > 32 ? 2 : 3) || (int64_t)g.instances * ar.parts > 256) {
        const dim3 gr((unsigned)g.instances), bl(64 * SMALL_WAVES);
        if (m <= 32) WGS_LAUNCH((ortho_small_kernel<1, true>), gr, bl, 0, st, g, mo, ar);
        else WGS_LAUNCH((ortho_small_kernel<2, true>), gr, bl, 0, st, g, mo, ar);
        return;
    }
    const bool step = g.step;
    if (g.dtype == WGS_F32) { if (step) launch_norm<WGS_F32, true>(g, mo, st); else launch_norm<WGS_F32, false>(g, mo, st); }
    else if (g.dtype == WGS_BF16) { if (step) launch_norm<WGS_BF16, true>(g, mo, st); else launch_norm<WGS_BF16, false>(g, mo, st); }
    else { if (step) launch_norm<WGS_F16, true>(g, mo, st); else launch_norm<WGS_F16, false>(g, mo, st); }
    const dim3 gr((unsigned)(g.instances * ar.parts)), bl(64 * SMALL_WAVES);
    for (ar.t = -1; ar.t < ar.bd.steps; ++ar.t) {
        if (m <= 32) WGS_LAUNCH((ortho_small_kernel<1, false>), gr, bl, 0, st, g, mo, ar);
        else WGS_LAUNCH((ortho_small_kernel<2, false>), gr, bl, 0, st, g, mo, ar);
    }
}

template <int DT>
void launch_tiny(const Group& g, const Momentum& mo, const TinyArgs& ar, hipStream_t st) {
    const dim3 gr((unsigned)g.instances), bl(64 * TINY_WAVES);
    if (g.step) WGS_LAUNCH((ortho_tiny_kernel<DT, true>), gr, bl, 0, st, g, mo, ar);
    else WGS_LAUNCH((ortho_tiny_kernel<DT, false>), gr, bl, 0, st, g, mo, ar);
}

int run(const char* who, const wgs_matrix* mats, int count, int dtype, bool step, const Momentum& mo, int steps, double a, double b, double c, float eps, void* ws,
        int64_t ws_bytes, hipStream_t st) {
    const char* bad = check_mats(mats, count, dtype, step, steps);
    WGS_CHECK_ARG(!bad, "%s: %s", who, bad);
    WGS_CHECK_ARG(eps >= 0.f && eps < 1e30f, "%s: eps must be a number >= 0", who);
    const int64_t need = workspace(mats, count, dtype, step, steps);
    if (!need) return WGS_OK;
    WGS_CHECK_ARG(ws && ws_bytes >= need && ((uintptr_t)ws & 255) == 0, "%s: workspace of %lld bytes needed, 256-byte aligned", who, (long long)need);
    // bounds of the iteration for these coefficients: Q_t = max |a + b l + c l^2|, cap = the largest eigenvalue of A_t
    Bounds bd;
    double q[MAX_STEPS], cap = 1.0, grow = 1.0;
    bd.eps = eps; bd.steps = steps;
    for (int t = 0; t <= steps; ++t) {
        bd.cap[t] = (float)(cap * 1.0001); bd.grow[t] = (float)grow;
        if (t == steps) break;
        double next;
        poly_bounds(a, b, c, cap * 1.0001, &q[t], &next);
        WGS_CHECK_ARG(next < 1e6 && q[t] < 1e6 && q[t] > 0, "%s: the iteration with these coefficients does not stay bounded", who);
        grow = fmin(grow * q[t] * q[t], 1e30); cap = next;
    }
    const Plan p = plan_of(dtype, step, steps, mats, count);
    Cursor cur, tiny;
    Group g;
    g.dtype = dtype; g.step = step; g.npx = p.npx; g.nt = p.nt; g.ns = p.ns; g.ws = (unsigned char*)ws;
    SmallArgs sm;
    sm.bd = bd; sm.a = (float)a; sm.b = (float)b; sm.c = (float)c;
    for (int t = 0; t < steps; ++t) sm.sb[t] = (float)ldexp(1.0, 14 - ceil_log2(q[t]));
    while (next_chunk(mats, count, p, true, tiny, g) > 0) {
        const TinyArgs ta = {a, b, c, eps, steps};
        if (dtype == WGS_F32) launch_tiny<WGS_F32>(g, mo, ta, st);
        else if (dtype == WGS_BF16) launch_tiny<WGS_BF16>(g, mo, ta, st);
        else launch_tiny<WGS_F16>(g, mo, ta, st);
    }
    while (next_chunk(mats, count, p, false, cur, g) > 0) {
        if (all_small(g, p, steps)) {
            launch_small(g, mo, sm, st);
            continue;
        }
        if (step) {
            if (dtype == WGS_F32) launch_prepare<WGS_F32, true>(g, mo, bd, st);
            else if (dtype == WGS_BF16) launch_prepare<WGS_BF16, true>(g, mo, bd, st);
            else launch_prepare<WGS_F16, true>(g, mo, bd, st);
        } else {
            if (dtype == WGS_F32) launch_prepare<WGS_F32, false>(g, mo, bd, st);
            else if (dtype == WGS_BF16) launch_prepare<WGS_BF16, false>(g, mo, bd, st);
            else launch_prepare<WGS_F16, false>(g, mo, bd, st);
        }
        int chained = 0;                     // the largest m
        for (int i = 0; i < g.count; ++i) { const int m = dims_of(g.mat[i].M, g.mat[i].N).m; if (m > chained) chained = m; }
        int t = 0;
        for (int ph = 0; ph < p.phases; ++ph) {
            const bool single = ph == 0 && p.planes == 1;
            const int A = BUF_S, B = BUF_S + 1, P = BUF_S + 2, T = BUF_T0 + (ph & 1), T2 = BUF_T0 + (~ph & 1);
            int Q = p.len[ph] > 1 ? BUF_S + 3 : B, Q2 = BUF_S + 4, rc;
            const int t0 = t;
            Jobs js = {};
            auto job = [&](int i, int kind, int op, int orr, int dst) -> Job& {
                Job& j = js.job[i];
                j = Job{};
                j.kind = kind; j.p = op; j.r = orr; j.dst = dst; j.t = t; j.first = ph == 0; j.mul = 1.f;
                return j;
            };
            js.count = 1; js.sym = 1; js.kgram = 1;
            job(0, GRAM, BUF_X, BUF_X, A);
            rc = single ? gemm<1, 1>(g, js, st) : gemm<2, 2>(g, js, st);
            if (rc) return rc;
            js.kgram = 0;
            double sq = 1.0;
            if (p.len[ph] > 1 && chained <= CHAIN_M) {
                ChainArgs ca = {};
                ca.t0 = t; ca.len = p.len[ph]; ca.src = A; ca.dst = Q; ca.a = (float)a; ca.b = (float)b; ca.c = (float)c;
                double bound = 1.0;
                for (int it = 0; it < p.len[ph]; ++it, ++t) {
                    const int em = ceil_log2(q[t]);
                    const double sb = ldexp(1.0, 14 - em);
                    bound *= q[t];
                    const double sq2 = it ? ldexp(1.0, 14 - ceil_log2(bound)) : sb;
                    ca.sb[it] = (float)sb; ca.grow[it] = (float)ldexp(1.0, em); ca.sq[it] = (float)(sq2 / (sq * sb));
                    sq = sq2;
                }
                if (chained <= 64) WGS_LAUNCH(ortho_chain_kernel<2>, dim3((unsigned)g.instances), dim3(512), 0, st, g, ca);
                else WGS_LAUNCH(ortho_chain_kernel<4>, dim3((unsigned)g.instances), dim3(512), 0, st, g, ca);
            } else
            for (int it = 0; it < p.len[ph]; ++it, ++t) {
                const int em = ceil_log2(q[t]);
                const double sb = ldexp(1.0, 14 - em);
                const int Bc = it == 0 ? Q : B;
                js.count = 1;
                Job& jp = job(0, POLY, A, A, Bc);
                jp.src = A; jp.a = (float)a; jp.b = (float)b; jp.c = (float)c; jp.mul = (float)sb;
                if ((rc = gemm<2, 2>(g, js, st))) return rc;
                const bool last = it + 1 == p.len[ph];
                int n = 0;
                if (!last) job(n++, PROD, Bc, A, P).mul = (float)(ldexp(1.0, -em) / sb);
                if (it > 0) {
                    double bound = 1.0;
                    for (int k = t0; k <= t; ++k) bound *= q[k];
                    const double sq2 = ldexp(1.0, 14 - ceil_log2(bound));
                    job(n++, PROD, Q, B, Q2).mul = (float)(sq2 / (sq * sb));
                    sq = sq2;
                    const int x = Q; Q = Q2; Q2 = x;
                } else sq = sb;
                if (n) { js.count = n; if ((rc = gemm<2, 2>(g, js, st))) return rc; }
                if (!last) {
                    js.count = 1;
                    Job& ja = job(0, PROD_A, P, Bc, A);
                    ja.t2 = t + 1; ja.mul = (float)(ldexp(1.0, em) / sb);
                    if ((rc = gemm<2, 2>(g, js, st))) return rc;
                }
            }
            js.count = 1; js.sym = 0;
            const bool out = ph + 1 == p.phases;
            Job& jx = job(0, out ? APPLY_OUT : APPLY_MID, Q, T, BUF_X);
            jx.dst2 = T2; jx.t = t0; jx.t2 = t; jx.mul = (float)(1.0 / sq);
            if ((rc = single ? gemm<2, 1>(g, js, st) : gemm<2, 2>(g, js, st))) return rc;
        }
    }
    WGS_CHECK_LAUNCH("ortho_gemm_kernel");
    return WGS_OK;
}

}  // namespace

extern "C" {

int64_t wgs_orthogonalise_ws_bytes(const wgs_matrix* mats, int count, int dtype, int steps) {
    return check_mats(mats, count, dtype, false, steps) ? 0 : workspace(mats, count, dtype, false, steps);
}
int wgs_orthogonalise(const wgs_matrix* mats, int count, int dtype, int steps, float a, float b, float c, float eps, void* ws, int64_t ws_bytes, wgs_stream_t stream) {
    return run("wgs_orthogonalise", mats, count, dtype, false, Momentum{0.f, 1.f, 0}, steps, a, b, c, eps, ws, ws_bytes, (hipStream_t)stream);
}
int64_t wgs_muon_step_ws_bytes(const wgs_matrix* mats, int count, int dtype, int steps) {
    return check_mats(mats, count, dtype, true, steps) ? 0 : workspace(mats, count, dtype, true, steps);
}
int wgs_muon_step(const wgs_matrix* mats, int count, int dtype, float momentum, int nesterov, float grad_scale, int steps, float a, float b, float c, float eps, void* ws,
                  int64_t ws_bytes, wgs_stream_t stream) {
    WGS_CHECK_ARG(momentum >= 0.f && momentum < 1.f, "wgs_muon_step: momentum must be in [0, 1)");
    return run("wgs_muon_step", mats, count, dtype, true, Momentum{momentum, grad_scale, nesterov}, steps, a, b, c, eps, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
