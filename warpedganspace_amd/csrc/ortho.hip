// Orthogonalised updates: the quintic Newton-Schulz iteration on matrices, alone or between a momentum and a weight update.
//
//   X_0 = X / (|X|_F + eps), on the wide side (m rows, n >= m columns);   A_t = X_t X_t^T,  B_t = a I + b A_t + c A_t^2,  X_{t+1} = B_t X_t
//
// Every A_t and B_t is a polynomial in A_0, so within a PHASE of k iterations only m x m matrices are needed:
//   A_{t+1} = B_t A_t B_t,  Q = B_{t+k-1} ... B_t,  X_{t+k} = Q X_t
// and all of them are symmetric: their products compute the tiles on and under the diagonal and write each twice.
//
// Arithmetic.  The iteration multiplies small singular values by a = 3.44 each time (A's eigenvalues by a^2), and the noise of the products with
// them, so the products keep fp32's precision: an operand is an fp16 pair hi + lo = value * 2^s (22 bits), a product lo*hi + hi*lo + hi*hi on
// the 16-bit matrix cores with fp32 accumulation — 3 / 2 500 of a TFLOP instead of 1 / 157 on the fp32 ones.  Exponents: X from its largest
// entry; A_t, X_t from bounds on their entries (|A_ij| <= max_i |x_i|^2, times the largest |a + b l + c l^2|^2 on the interval that the
// eigenvalues can reach, iteration by iteration); B, Q from the same polynomial's maximum.  16-bit inputs are their own hi part (one product in
// the first Gram matrix, two in its phase's Q X).  Norms are summed in fp64.
#include "wgs_common.h"
#include "../../include/wgs.h"
#include <math.h>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr int MAX_MATS = 24;             // matrices of one launch (they travel as kernel arguments)
constexpr int MAX_STEPS = 16;
constexpr int INFO = 64;                 // floats of an instance's scalars: f0, then sA[t], sX[t]
constexpr int I_SA = 4, I_SX = I_SA + MAX_STEPS + 1;
constexpr int STAT_BLOCKS = 256;         // partial norms of an instance
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
    Mat mat[MAX_MATS];
    unsigned char* ws;
    int count, instances;
    int npx, nt, ns;         // planes of X / X^T, buffers of X^T, m x m buffers
    int stat_blocks;
    int dtype, step;         // element type of in / out; a weight update rather than the bare factor
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
struct Plane { unsigned char* hi; int64_t step; int ld; int64_t bytes; };       // lo plane = hi + step
__device__ __forceinline__ Plane plane_of(const Group& g, const Mat& a, const Dims& d, int inst, int buf) {
    unsigned char* p = g.ws + a.ws + inst * instance_bytes(d, g.npx, g.nt, g.ns);
    Plane r;
    if (buf == BUF_X) { r = Plane{p, d.szx, d.np, (int64_t)d.m * d.np * 2}; }
    else if (buf < BUF_S) { r = Plane{p + g.npx * d.szx + (int64_t)(buf - 1) * g.npx * d.szt, d.szt, d.mp, (int64_t)d.n * d.mp * 2}; }
    else { r = Plane{p + g.npx * d.szx + (int64_t)g.nt * g.npx * d.szt + (int64_t)(buf - BUF_S) * 2 * d.szs, d.szs, d.mp, (int64_t)d.m * d.mp * 2}; }
    return r;
}
// header of the workspace: partial norms, then the scalars of every instance
struct Part { double ss; float amax; float pad; };
__host__ __device__ __forceinline__ int64_t header_bytes(int instances, int blocks) {
    return up((int64_t)instances * blocks * (int64_t)sizeof(Part), 256) + up((int64_t)instances * INFO * 4, 256);
}
__device__ __forceinline__ Part* parts_of(const Group& g, int inst) { return (Part*)g.ws + (int64_t)inst * g.stat_blocks; }
__device__ __forceinline__ float* info_of(const Group& g, int inst) {
    return (float*)(g.ws + up((int64_t)g.instances * g.stat_blocks * (int64_t)sizeof(Part), 256)) + (int64_t)inst * INFO;
}
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
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const Group g, const Momentum mo) {
    __shared__ double rs[4];
    __shared__ float rm[4];
    const int inst = blockIdx.x / (unsigned)g.stat_blocks, blk = blockIdx.x % (unsigned)g.stat_blocks;
    const Mat& a = g.mat[entry_of(g, inst)];
    const int b = inst - a.first;
    const int64_t total = (int64_t)a.M * a.N, off = b * a.in_bs, moff = b * total;
    const int64_t per = up((total + g.stat_blocks - 1) / g.stat_blocks, 1024);
    const int64_t e0 = blk * per, e1 = e0 + per < total ? e0 + per : total;
    double ss = 0.0;
    float amax = 0.f;
    for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
        const int64_t i = a.in_rs == a.N ? e : (e / a.N) * a.in_rs + e % a.N;
        const float v = update_of<DT, STEP>(a, off + i, moff + e, mo, true);
        ss += (double)v * v;
        amax = fmaxf(amax, fabsf(v));
    }
    ss = wave_sum_d(ss);
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) { rs[threadIdx.x >> 6] = ss; rm[threadIdx.x >> 6] = amax; }
    __syncthreads();
    if (threadIdx.x == 0) {
        Part* p = parts_of(g, inst) + blk;
        p->ss = rs[0] + rs[1] + rs[2] + rs[3];
        p->amax = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
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
    h = (_Float16)v;
    l = (_Float16)(v - (float)h);
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
    const bool finite = ss < 1e300;          // false for NaN and infinity
    const float mult = (finite && amax > 0.f) ? pow2_under(amax, 15, -120, 120) : 1.f;
    if (tt == 0 && t == 0) {
        float* info = info_of(g, inst);
        const double inv = ss > 0.0 ? 1.0 / (sqrt(ss) + (double)bd.eps) : 0.0;
        info[0] = finite ? (float)(inv / (double)mult) : NAN;
        const double top = (double)amax * inv;
        const double d0 = finite ? (double)d.n * top * top : 1.0;
        for (int k = 0; k <= bd.steps; ++k) {
            double v = d0 * (double)bd.grow[k];
            v = v < (double)bd.cap[k] ? v : (double)bd.cap[k];
            info[I_SA + k] = pow2_under((float)(v > 1e-30 ? v : 1e-30), 14, -60, 60);
            info[I_SX + k] = pow2_under((float)sqrt(v > 1e-70 ? v : 1e-70), 14, -60, 110);
        }
    }
    const int64_t off = b * a.in_bs, moff = (int64_t)b * a.M * a.N;
    for (int i = t; i < 64 * 64; i += 256) {
        const int r = r0 + (i >> 6), c = c0 + (i & 63);
        float v = 0.f;
        if (r < a.M && c < a.N) v = update_of<DT, STEP>(a, off + (int64_t)r * a.in_rs + c, moff + (int64_t)r * a.N + c, mo, false) * mult;
        tile[i >> 6][i & 63] = v;
    }
    __syncthreads();
    const bool wide = a.M <= a.N;
    const Plane nat = plane_of(g, a, d, b, wide ? BUF_X : BUF_T0), tra = plane_of(g, a, d, b, wide ? BUF_T0 : BUF_X);
    // natural: rows r < M, columns up to the padding; transposed: rows c < N, columns r up to the padding.  Two columns a thread.
    for (int i = t; i < 64 * 32; i += 256) {
        const int x = i >> 5, y = (i & 31) * 2;
        if (r0 + x < a.M && c0 + y < nat.ld) {
            _Float16 h0, l0, h1, l1;
            split_pair(tile[x][y], h0, l0); split_pair(tile[x][y + 1], h1, l1);
            const int64_t at = ((int64_t)(r0 + x) * nat.ld + c0 + y) * 2;
            _Float16* q = (_Float16*)(nat.hi + at);
            q[0] = h0; q[1] = h1;
            if (LO) { _Float16* w = (_Float16*)(nat.hi + nat.step + at); w[0] = l0; w[1] = l1; }
        }
        if (c0 + x < a.N && r0 + y < tra.ld) {
            _Float16 h0, l0, h1, l1;
            split_pair(tile[y][x], h0, l0); split_pair(tile[y + 1][x], h1, l1);
            const int64_t at = ((int64_t)(c0 + x) * tra.ld + r0 + y) * 2;
            _Float16* q = (_Float16*)(tra.hi + at);
            q[0] = h0; q[1] = h1;
            if (LO) { _Float16* w = (_Float16*)(tra.hi + tra.step + at); w[0] = l0; w[1] = l1; }
        }
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
struct Jobs { Job job[2]; int count; int sym; };

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

template <int NA, int NB, int BM, int WAVES_M, int WAVES_N, int NS>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 1) void ortho_gemm_kernel(const Group g, const Jobs js, int total) {
    constexpr int BN = BM, NW = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
    constexpr int A_BYTES = BM * ROW, B_BYTES = BN * ROW, STAGE = NA * A_BYTES + NB * B_BYTES;
    constexpr int AI = BM / 16 / NW, BI = BN / 16 / NW, NPIECE = NA * AI + NB * BI;
    static_assert(AI * 16 * NW == BM && BI * 16 * NW == BN && TM * 32 * WAVES_M == BM && TN * 32 * WAVES_N == BN, "tile / wave count mismatch");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;

    // workgroups go round the 8 XCDs: each gets a contiguous range of tiles
    const int per_xcd = (total + 7) >> 3;
    int tile = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || tile >= total) return;
    const int half = js.count == 2 ? total / 2 : total;
    const Job& J = js.job[tile >= half ? 1 : 0];
    if (tile >= half) tile -= half;
    int e = 0, tm = 0, tn = 0, per = 0;
    for (;; ++e) {
        const Dims q = dims_of(g.mat[e].M, g.mat[e].N);
        tm = (q.m + BM - 1) / BM; tn = (q.n + BN - 1) / BN;
        per = js.sym ? tm * (tm + 1) / 2 : tm * tn;
        const int c = g.mat[e].batch * per;
        if (tile < c || e + 1 == g.count) break;
        tile -= c;
    }
    const Mat& mat = g.mat[e];
    const Dims d = dims_of(mat.M, mat.N);
    const int b = tile / per, inst = mat.first + b;
    int ti, tj;
    if (js.sym) tile_lower(tile % per, tm, ti, tj);
    else tile_full(tile % per, tm, tn, ti, tj);
    const int i0 = ti * BM, j0 = tj * BN;
    const Plane P = plane_of(g, mat, d, b, J.p), R = plane_of(g, mat, d, b, J.r);
    const int nk = P.ld / BK;

    const __amdgpu_buffer_rsrc_t rp0 = __builtin_amdgcn_make_buffer_rsrc(P.hi, 0, (unsigned)P.bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rp1 = __builtin_amdgcn_make_buffer_rsrc(P.hi + (NA > 1 ? P.step : 0), 0, (unsigned)P.bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rr0 = __builtin_amdgcn_make_buffer_rsrc(R.hi, 0, (unsigned)R.bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rr1 = __builtin_amdgcn_make_buffer_rsrc(R.hi + (NB > 1 ? R.step : 0), 0, (unsigned)R.bytes, 0x00020000);
    // An LDS load writes wave base + lane * 16: one instruction fills 16 rows of 64 bytes.  The four 16-byte slots of a row are permuted by
    // (row >> 2) & 3, on the address that is fetched and on the one that is read, so that the rows of a fragment read spread over the banks.
    const int lrow = lane >> 2, slot = lane & 3;
    int a_off[AI], b_off[BI];
#pragma unroll
    for (int j = 0; j < AI; ++j) {
        const int row = (wave * AI + j) * 16 + lrow, lc = slot ^ ((row >> 2) & 3);
        a_off[j] = i0 + row < d.m ? (int)(((int64_t)(i0 + row) * P.ld + lc * 8) * 2) : OOB;
    }
    const int rows_r = J.kind >= APPLY_MID ? d.n : d.m;
#pragma unroll
    for (int j = 0; j < BI; ++j) {
        const int row = (wave * BI + j) * 16 + lrow, lc = slot ^ ((row >> 2) & 3);
        b_off[j] = j0 + row < rows_r ? (int)(((int64_t)(j0 + row) * R.ld + lc * 8) * 2) : OOB;
    }
    int nC = 0;
    auto issue = [&](int buf) {
        const bool past = nC >= nk;
        const int adv = past ? 0 : nC * ROW;
        ++nC;
#pragma unroll
        for (int idx = 0; idx < NPIECE; ++idx) {
            lds_byte* st = (lds_byte*)(smem + buf * STAGE);
            if (idx < NA * AI) {
                const int j = idx / NA, pl = idx % NA;
                const int off = past ? OOB : (int)((unsigned)a_off[j] + (unsigned)adv);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(pl ? rp1 : rp0, st + (wave * AI + j) * 16 * ROW + pl * A_BYTES, 16, off, 0, 0, 0);
            } else {
                const int j = (idx - NA * AI) / NB, pl = (idx - NA * AI) % NB;
                const int off = past ? OOB : (int)((unsigned)b_off[j] + (unsigned)adv);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(pl ? rr1 : rr0, st + NA * A_BYTES + (wave * BI + j) * 16 * ROW + pl * B_BYTES, 16, off, 0, 0, 0);
            }
        }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int l31 = lane & 31, lh = lane >> 5, swz = (l31 >> 2) & 3;
    const int a_rd = (wm * WM + l31) * ROW, b_rd = NA * A_BYTES + (wn * WN + l31) * ROW;

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue(s);
    int cur = 0, nxt = NS - 1;
    for (int kt = 0; kt < nk; ++kt) {
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NS - 2) * NPIECE) : "memory");      // this wave's pieces of chunk kt have landed
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();                                                   // ... and everybody's; stage nxt is no longer read
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        issue(nxt);
        const unsigned char* base = smem + cur * STAGE;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int kc = ((2 * ks + lh) ^ swz) * 16;
            half8 af[TM][NA], bf[TN][NB];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int pl = 0; pl < NA; ++pl) af[i][pl] = *reinterpret_cast<const half8*>(base + a_rd + pl * A_BYTES + i * 32 * ROW + kc);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int pl = 0; pl < NB; ++pl) bf[j][pl] = *reinterpret_cast<const half8*>(base + b_rd + pl * B_BYTES + j * 32 * ROW + kc);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    if (NA > 1) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i][NA - 1], bf[j][0], acc[i][j], 0, 0, 0);
                    if (NB > 1) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i][0], bf[j][NB - 1], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i][0], bf[j][0], acc[i][j], 0, 0, 0);
                }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        cur = cur + 1 == NS ? 0 : cur + 1;
        nxt = nxt + 1 == NS ? 0 : nxt + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the zero loads past the last chunk

    // ---- epilogue: a lane holds column j = lane & 31 and rows 8 q + 4 (lane >> 5) + 0..3 of every 32 x 32 block
    const float* info = info_of(g, inst);
    const float fx = J.first ? info[0] : 1.f / info[I_SX + J.t];
    float mult = J.mul;
    if (J.kind == GRAM) mult = fx * fx * info[I_SA + J.t];
    else if (J.kind == POLY) mult = 1.f / (info[I_SA + J.t] * info[I_SA + J.t]);
    else if (J.kind == PROD_A) mult = J.mul * (info[I_SA + J.t2] / info[I_SA + J.t]);
    else if (J.kind == APPLY_MID) mult = J.mul * fx * info[I_SX + J.t2];
    else if (J.kind == APPLY_OUT) mult = J.mul * fx;
    if (J.kind == APPLY_OUT) {
        const bool wide = mat.M <= mat.N;
        const int64_t ob = b * mat.out_bs;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int c = j0 + wn * WN + j * 32 + l31;
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int r = i0 + wm * WM + i * 32 + 8 * (q >> 2) + 4 * lh + (q & 3);
                    if (r < d.m && c < d.n) {
                        const int64_t at = ob + (wide ? (int64_t)r * mat.out_rs + c : (int64_t)c * mat.out_rs + r);
                        float v = acc[i][j][q] * mult;
                        if (g.step) v = mat.decay * load_as(g.dtype, mat.out, at) - mat.step * v;
                        store_as(g.dtype, mat.out, at, v);
                    }
                }
            }
        return;
    }
    const bool mid = J.kind == APPLY_MID;
    const Plane D = plane_of(g, mat, d, b, J.dst);                              // [i][j]
    const Plane T = mid ? plane_of(g, mat, d, b, J.dst2) : D;                   // [j][i]
    const Plane S = J.kind == POLY ? plane_of(g, mat, d, b, J.src) : D;
    const float isa = J.kind == POLY ? 1.f / info[I_SA + J.t] : 0.f;
    const int nc = mid ? d.n : d.m;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int c = j0 + wn * WN + j * 32 + l31, rb = i0 + wm * WM + i * 32, cb = j0 + wn * WN + j * 32;
            // A tile on the diagonal computes both triangles, whose roundings differ where the factors do not quite commute: the strict upper
            // one is dropped, else the iteration amplifies the antisymmetric part (measured: ten times the error on spiked spectra).
            if (!mid && rb < cb) continue;
            const bool half = !mid && rb == cb;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = i0 + wm * WM + i * 32 + 8 * q + 4 * lh;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = acc[i][j][4 * q + k] * mult;
                if (J.kind == POLY) {
                    if (c < d.m && r < d.mp) {
                        const half4 sh = *reinterpret_cast<const half4*>(S.hi + ((int64_t)c * S.ld + r) * 2);
                        const half4 sl = *reinterpret_cast<const half4*>(S.hi + S.step + ((int64_t)c * S.ld + r) * 2);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float A = ((float)sh[k] + (float)sl[k]) * isa;
                            v[k] = ((r + k == c ? J.a : 0.f) + (J.b * A + J.c * v[k])) * J.mul;
                        }
                    }
                }
                half4 h, l;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (r + k >= d.m || c >= nc) v[k] = 0.f;                  // the padding of both planes
                    _Float16 hh, ll;
                    split_pair(v[k], hh, ll);
                    h[k] = hh; l[k] = ll;
                }
                if (half) {                                   // both writes, only from the triangle r >= c
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r + k >= c && c < d.m && r + k < D.ld) {
                            _Float16* x = reinterpret_cast<_Float16*>(D.hi + ((int64_t)c * D.ld + r + k) * 2);
                            x[0] = h[k];
                            *reinterpret_cast<_Float16*>(reinterpret_cast<unsigned char*>(x) + D.step) = l[k];
                            if (r + k < d.m) {
                                _Float16* y = reinterpret_cast<_Float16*>(D.hi + ((int64_t)(r + k) * D.ld + c) * 2);
                                y[0] = h[k];
                                *reinterpret_cast<_Float16*>(reinterpret_cast<unsigned char*>(y) + D.step) = l[k];
                            }
                        }
                    continue;
                }
                if (c < nc && r < T.ld) {
                    *reinterpret_cast<half4*>(T.hi + ((int64_t)c * T.ld + r) * 2) = h;
                    *reinterpret_cast<half4*>(T.hi + T.step + ((int64_t)c * T.ld + r) * 2) = l;
                }
                if (c < D.ld) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r + k < d.m) {
                            *reinterpret_cast<_Float16*>(D.hi + ((int64_t)(r + k) * D.ld + c) * 2) = h[k];
                            *reinterpret_cast<_Float16*>(D.hi + D.step + ((int64_t)(r + k) * D.ld + c) * 2) = l[k];
                        }
                }
            }
        }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
struct Plan { int phases, len[MAX_STEPS]; int planes, npx, nt, ns; };
// Iterations of a phase.  Longer phases leave out products with the n columns, but A_t then carries its own rounding through a^2 a step instead
// of being formed anew from X_t: measured on spectra from flat to a single spike, one phase of five is within 4e-4 of the exact factor, (3, 2)
// within 3e-5, single iterations within the 32-bit iteration's own 2e-5 (1e-6 .. 1e-5 for noise-dominated matrices).  So: what the result's
// type can hold.
Plan plan_of(int dtype, bool step, int steps) {
    Plan p;
    const int most = dtype == WGS_BF16 ? 5 : dtype == WGS_F16 ? 3 : 1;
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

// The matrices in runs of at most MAX_MATS entries and CHUNK_BYTES (or one matrix); batches are cut where they have to be.
struct Cursor { int entry = 0, done = 0; };
int64_t next_chunk(const wgs_matrix* mats, int count, const Plan& p, Cursor& c, Group& g) {
    int64_t bytes = 0;
    g.count = 0; g.instances = 0;
    int64_t most = 0;
    while (c.entry < count && g.count < MAX_MATS) {
        const wgs_matrix& w = mats[c.entry];
        const int left = w.batch - c.done;
        if (left <= 0) { ++c.entry; c.done = 0; continue; }
        const int64_t one = instance_bytes(dims_of(w.rows, w.cols), p.npx, p.nt, p.ns);
        int64_t fit = (CHUNK_BYTES - bytes) / one;
        if (fit < 1) { if (g.count) break; fit = 1; }
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
        if ((int64_t)w.rows * w.cols > most) most = (int64_t)w.rows * w.cols;
        c.done += take;
        if (c.done == w.batch) { ++c.entry; c.done = 0; }
        if (take < left) break;
    }
    if (!g.count) return 0;
    int64_t sb = most / 16384;                    // 64 elements a thread where the matrix is large
    g.stat_blocks = sb < 1 ? 1 : (sb > STAT_BLOCKS ? STAT_BLOCKS : (int)sb);
    const int64_t head = header_bytes(g.instances, g.stat_blocks);
    for (int i = 0; i < g.count; ++i) g.mat[i].ws += head;
    return head + bytes;
}

const char* check_mats(const wgs_matrix* mats, int count, int dtype, bool step, int steps) {
    if (dtype != WGS_F32 && dtype != WGS_BF16 && dtype != WGS_F16) return "unknown dtype";
    if (count < 0 || (count && !mats)) return "no matrices";
    if (steps < 1 || steps > MAX_STEPS) return "steps must be 1 .. 16";
    for (int i = 0; i < count; ++i) {
        const wgs_matrix& w = mats[i];
        if (w.rows < 1 || w.cols < 1 || w.batch < 0 || (int64_t)w.rows * up(w.cols, BK) >= (1LL << 30) || (int64_t)w.cols * up(w.rows, BK) >= (1LL << 30))
            return "bad sizes (rows, cols >= 1, fewer than 2^30 elements with the smaller side's padding to 32)";
        if (w.in_row_stride < w.cols || w.out_row_stride < w.cols || w.in_row_stride >= (1LL << 31) || w.out_row_stride >= (1LL << 31)) return "row strides must be at least cols";
        if (w.batch > 1 && (w.in_batch_stride < 0 || w.out_batch_stride < (int64_t)(w.rows - 1) * w.out_row_stride + w.cols)) return "batch strides overlap";
        if (w.batch > (1 << 20)) return "batch must be at most 2^20";
        if (w.batch && (!w.in || !w.out || (step && !w.momentum))) return "null pointer";
        const uintptr_t am = dtype == WGS_F32 ? 3 : 1;
        if ((((uintptr_t)w.in | (uintptr_t)w.out) & am) || ((uintptr_t)w.momentum & 3)) return "a matrix is not aligned to its type";
    }
    return nullptr;
}

int64_t workspace(const wgs_matrix* mats, int count, int dtype, bool step, int steps) {
    const Plan p = plan_of(dtype, step, steps);
    Cursor c;
    Group g;
    g.dtype = dtype;
    int64_t need = 0;
    for (;;) {
        const int64_t b = next_chunk(mats, count, p, c, g);
        if (!b) return need;
        if (b > need) need = b;
    }
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

template <int NA, int NB, int BM, int WM, int WN, int NS>
void launch_gemm(const Group& g, const Jobs& js, int total, hipStream_t st) {
    constexpr int sm = NS * (NA + NB) * BM * ROW;
    auto k = ortho_gemm_kernel<NA, NB, BM, WM, WN, NS>;
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, sm);
    WGS_LAUNCH(k, dim3((unsigned)((total + 7) / 8 * 8)), dim3(64 * WM * WN), sm, st, g, js, total);
}
int tiles_of(const Group& g, const Jobs& js, int bm) {
    int64_t t = 0;
    for (int i = 0; i < g.count; ++i) {
        const Dims d = dims_of(g.mat[i].M, g.mat[i].N);
        const int64_t tm = (d.m + bm - 1) / bm, tn = (d.n + bm - 1) / bm;
        t += g.mat[i].batch * (js.sym ? tm * (tm + 1) / 2 : tm * tn);
    }
    t *= js.count;
    return t < (1LL << 30) ? (int)t : 0;
}
template <int NA, int NB>
int gemm(const Group& g, const Jobs& js, hipStream_t st) {
    int bm = 64;
    if (tiles_of(g, js, 256) >= 200) bm = 256;
    else if (tiles_of(g, js, 128) >= 200) bm = 128;
    const int total = tiles_of(g, js, bm);
    WGS_CHECK_ARG(total > 0, "orthogonalise: too many matrices for one launch");
    if (bm == 256) launch_gemm<NA, NB, 256, 2, 4, 2>(g, js, total, st);
    else if (bm == 128) launch_gemm<NA, NB, 128, 2, 2, 2>(g, js, total, st);
    else launch_gemm<NA, NB, 64, 2, 2, 4>(g, js, total, st);
    return WGS_OK;
}

template <int DT, bool STEP>
void launch_prepare(const Group& g, const Momentum& mo, const Bounds& bd, hipStream_t st) {
    WGS_LAUNCH((ortho_norm_kernel<DT, STEP>), dim3((unsigned)(g.instances * g.stat_blocks)), dim3(256), 0, st, g, mo);
    int64_t tiles = 0;
    for (int i = 0; i < g.count; ++i) tiles += (int64_t)g.mat[i].batch * ((up(g.mat[i].M, BK) + 63) / 64) * ((up(g.mat[i].N, BK) + 63) / 64);
    WGS_LAUNCH((ortho_split_kernel<DT, STEP>), dim3((unsigned)tiles), dim3(256), 0, st, g, mo, bd, (int)tiles);
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
    const Plan p = plan_of(dtype, step, steps);
    Cursor cur;
    Group g;
    g.dtype = dtype; g.step = step; g.npx = p.npx; g.nt = p.nt; g.ns = p.ns; g.ws = (unsigned char*)ws;
    while (next_chunk(mats, count, p, cur, g) > 0) {
        if (step) {
            if (dtype == WGS_F32) launch_prepare<WGS_F32, true>(g, mo, bd, st);
            else if (dtype == WGS_BF16) launch_prepare<WGS_BF16, true>(g, mo, bd, st);
            else launch_prepare<WGS_F16, true>(g, mo, bd, st);
        } else {
            if (dtype == WGS_F32) launch_prepare<WGS_F32, false>(g, mo, bd, st);
            else if (dtype == WGS_BF16) launch_prepare<WGS_BF16, false>(g, mo, bd, st);
            else launch_prepare<WGS_F16, false>(g, mo, bd, st);
        }
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
            js.count = 1; js.sym = 1;
            job(0, GRAM, BUF_X, BUF_X, A);
            rc = single ? gemm<1, 1>(g, js, st) : gemm<2, 2>(g, js, st);
            if (rc) return rc;
            double sq = 1.0;
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
