// Log-probabilities of given labels with the entropy of the scores and the `top` most likely alternatives, and their gradient.
//
//   l = a row of V scores, m = max l, s = sum exp(l - m), u = sum exp(l - m) (l - m)
//   logp = (l_t - m) - log s,      H = -sum p log p = log s - u / s,      p = exp(l - m) / s
//   dl_v = g ([v = t] - p_v) - h p_v (log p_v + H) + sum_j q_j ([v = i_j] - p_v)        for upstream (g, h, q) of (logp, H, top_logp)
//
// Both directions are HBM-bound: the forward reads the scores once (m, s, u are carried online per lane, rescaled when the lane's maximum
// rises), the backward reads them once more and writes the gradient.  All statistics are fp32; s and u have at most V / 256 terms a lane
// (V / 64 up to 2048 scores) before the tree.  Scores are taken relative to m before the exponential, so far-from-zero rows lose nothing.
//
// Alternatives: a score's key = (order-preserving bits << 32 | ~index), so keys are distinct and equal scores sort by the lower index.  Every
// wave keeps its own sorted list of 64 keys, one a lane, and the key of the `top`-th: a vector of scores costs one comparison of its maximum
// with that threshold, and only candidates over it are collected (in LDS), sorted and merged, 64 at a time.  The first vectors set the
// threshold: the `top`-th largest of the 64 lanes' maxima has at least `top` scores at or over it.
#include "wgs_common.h"
#include "../../include/wgs.h"

namespace {

typedef unsigned long long u64;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr float L2E = 1.4426950408889634f;
constexpr float LOWEST = -3.402823466e38f;
constexpr int UNROLL = 4;               // 16-byte vectors in flight a lane
constexpr int TOP_MAX = 64;             // one key a lane
constexpr int MAX_SPLIT = 64;           // parts of a row: one a lane in the joining launch

template <int DT> struct Vec;
template <> struct Vec<WGS_F32> {
    static constexpr int N = 4;
    typedef float elem;
    static __device__ __forceinline__ float get(elem v) { return v; }
    static __device__ __forceinline__ elem put(float v) { return v; }
    static __device__ __forceinline__ void unpack(uint4 q, float (&f)[N]) {
        f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[N]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Vec<WGS_BF16> {
    static constexpr int N = 8;
    typedef __bf16 elem;
    static __device__ __forceinline__ float get(elem v) { return (float)v; }
    static __device__ __forceinline__ elem put(float v) { return (__bf16)v; }
    static __device__ __forceinline__ void unpack(uint4 q, float (&f)[N]) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[N]) {
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        b8 v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (__bf16)f[i];
        return __builtin_bit_cast(uint4, v);
    }
};
template <> struct Vec<WGS_F16> {
    static constexpr int N = 8;
    typedef _Float16 elem;
    static __device__ __forceinline__ float get(elem v) { return (float)v; }
    static __device__ __forceinline__ elem put(float v) { return (_Float16)v; }
    static __device__ __forceinline__ void unpack(uint4 q, float (&f)[N]) {
        const half8 v = __builtin_bit_cast(half8, q);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = (float)v[i];
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[N]) {
        half8 v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (_Float16)f[i];
        return __builtin_bit_cast(uint4, v);
    }
};

// ---- keys ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned order_bits(float f) {      // order-preserving; -0 as +0
    const unsigned b = __float_as_uint(f + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) { return __uint_as_float(o ^ ((unsigned)~((int)o >> 31) | 0x80000000u)); }
__device__ __forceinline__ u64 make_key(float f, int index) { return (u64)order_bits(f) << 32 | (unsigned)~index; }
__device__ __forceinline__ u64 shfl_xor64(u64 v, int mask) {
    const unsigned lo = __shfl_xor((unsigned)v, mask, 64), hi = __shfl_xor((unsigned)(v >> 32), mask, 64);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl64(u64 v, int lane) {
    const unsigned lo = __shfl((unsigned)v, lane, 64), hi = __shfl((unsigned)(v >> 32), lane, 64);
    return (u64)hi << 32 | lo;
}
// one compare-exchange step of a bitonic network over the wave
__device__ __forceinline__ u64 exchange(u64 v, int mask, bool keep_max) {
    const u64 o = shfl_xor64(v, mask);
    return ((v > o) == keep_max) ? v : o;
}
__device__ __forceinline__ u64 sort_ascending(u64 v, int lane) {
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int mask = size >> 1; mask > 0; mask >>= 1) {
            const bool up = size == 64 || !(lane & size);       // this block ends ascending
            v = exchange(v, mask, up == (bool)(lane & mask));
        }
    return v;
}
// `list` descending, `batch` ascending: the 64 largest of both, descending
__device__ __forceinline__ u64 merge_descending(u64 list, u64 batch, int lane) {
    u64 v = list > batch ? list : batch;
#pragma unroll
    for (int mask = 32; mask > 0; mask >>= 1) v = exchange(v, mask, !(lane & mask));
    return v;
}
// the k-th largest (k in 1 .. 64) of one float a lane
__device__ __forceinline__ float kth_largest(float f, int k, int lane) {
    unsigned v = order_bits(f);
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int mask = size >> 1; mask > 0; mask >>= 1) {
            const bool up = size == 64 || !(lane & size);
            const unsigned o = __shfl_xor(v, mask, 64);
            v = ((v > o) == (up == (bool)(lane & mask))) ? v : o;
        }
    return order_value(__shfl(v, 64 - k, 64));
}

// One wave's running list.  buf: 128 keys of LDS of its own.
struct TopList {
    u64 list, threshold;      // keys over `threshold` are candidates
    float value;              // its score and index: the test on a whole vector
    int index, count, k;
    u64* buf;
    int lane;
    __device__ __forceinline__ void init(int k_, u64* b, int l) { list = 0; threshold = 0; value = -INFINITY; index = 0x7fffffff; count = 0; k = k_; buf = b; lane = l; }
    __device__ __forceinline__ void raise(u64 key) {
        if (key > threshold) { threshold = key; value = order_value((unsigned)(key >> 32)); index = (int)~(unsigned)key; }
    }
    // at least k scores are at or over f
    __device__ __forceinline__ void at_least(float f) {
        const u64 key = ((u64)order_bits(f) << 32) - 1;
        if (key > threshold) { threshold = key; value = f; index = 0x7fffffff; }
    }
    __device__ __forceinline__ void flush() {
        __builtin_amdgcn_wave_barrier();
        const u64 batch = sort_ascending(lane < count ? buf[lane] : 0, lane);
        const int rest = count - 64;
        u64 moved = 0;
        if (lane < rest) moved = buf[64 + lane];
        __builtin_amdgcn_wave_barrier();
        if (lane < rest) buf[lane] = moved;
        __builtin_amdgcn_wave_barrier();
        count = rest > 0 ? rest : 0;
        list = merge_descending(list, batch, lane);
        raise(shfl64(list, k - 1));
    }
    __device__ __forceinline__ void offer(u64 key, bool have) {      // called by the whole wave
        const bool cand = have && key > threshold;
        const u64 mask = __ballot(cand);
        if (!mask) return;
        if (cand) buf[count + __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0))] = key;
        count += __popcll(mask);
        if (count >= 64) flush();
    }
    __device__ __forceinline__ void finish() { while (count > 0) flush(); }
};

// ---- running statistics of a lane / wave / row ------------------------------------------------------------------------------------
struct Stat { float m, s, u; };
// w d for a weight w = (something) exp(d): exactly 0 once exp(d) is (below -104), whatever d is, minus infinity too; a NaN stays in w
__device__ __forceinline__ float weigh(float w, float d) { return w * fmaxf(d, -200.f); }
__device__ __forceinline__ void add_scores(Stat& a, float cm, const float* f, int n) {
    const float mn = fmaxf(a.m, cm);
    const float shift = a.m - mn, scale = __builtin_amdgcn_exp2f(shift * L2E);
    float s = a.s * scale, u = scale * (a.u + weigh(a.s, shift));
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const float d = f[i] - mn, e = __builtin_amdgcn_exp2f(d * L2E);
        s += e;
        u += weigh(e, d);
    }
    a.m = mn; a.s = s; a.u = u;
}
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m - m, db = b.m - m;
    const float ea = __builtin_amdgcn_exp2f(da * L2E), eb = __builtin_amdgcn_exp2f(db * L2E);
    Stat r;
    r.m = m;
    r.s = a.s * ea + b.s * eb;
    r.u = ea * (a.u + weigh(a.s, da)) + eb * (b.u + weigh(b.s, db));
    return r;
}
__device__ __forceinline__ Stat wave_join(Stat a) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        Stat b;
        b.m = __shfl_xor(a.m, off, 64); b.s = __shfl_xor(a.s, off, 64); b.u = __shfl_xor(a.u, off, 64);
        a = join(a, b);
    }
    return a;
}

struct FwdArgs {
    const void* logits;
    const int64_t* labels;
    float *logp, *entropy, *stat, *top_logp;
    int64_t* top_index;
    float* part_stat;         // [rows][split][4]
    u64* part_key;            // [rows][split][top]
    int64_t rows, stride, ignore;
    int V, top, split;
};

// outputs of one row from its statistics; called by lane 0
template <int DT>
__device__ __forceinline__ void write_row(const FwdArgs& a, int64_t row, const Stat& t) {
    const int64_t label = a.labels[row];
    const float ls = logf(t.s);
    const bool empty = t.s == 0.f;              // every score is minus infinity: no distribution, entropy 0
    float lp = 0.f;
    if (label >= 0 && label < a.V) {
        const float x = Vec<DT>::get(((const typename Vec<DT>::elem*)a.logits)[row * a.stride + label]);
        lp = empty ? -INFINITY : (x - t.m) - ls;
    } else if (label != a.ignore) {
        lp = NAN;                               // neither a class nor the ignored label
    }
    a.logp[row] = (label == a.ignore) ? 0.f : lp;
    a.entropy[row] = empty ? 0.f : ls - t.u / t.s;
    a.stat[2 * row] = t.m;
    a.stat[2 * row + 1] = ls;                   // minus infinity marks an empty row
}
__device__ __forceinline__ void write_top(const FwdArgs& a, int64_t row, const Stat& t, u64 list, int lane) {
    if (lane >= a.top) return;
    const float x = order_value((unsigned)(list >> 32));
    const bool none = t.s != t.s;               // NaN or +inf among the scores
    a.top_logp[row * a.top + lane] = none ? NAN : (t.s == 0.f ? -INFINITY : (x - t.m) - logf(t.s));
    a.top_index[row * a.top + lane] = none ? -1 : (int64_t)(int)~(unsigned)list;
}

// WPR waves a row part.  WPR = 1: a wave a row, four rows a workgroup (short rows: no barrier, no join).
// WPR = 4: a workgroup a row, or one of `split` parts of a row where the rows alone do not fill the chip.
template <int DT, int WPR, bool TOP>
__global__ __launch_bounds__(256) void logprob_fwd_kernel(const FwdArgs a) {
    typedef Vec<DT> X;
    constexpr int N = X::N, T = 64 * WPR;
    __shared__ u64 keys[TOP ? 4 * 128 : 1];
    __shared__ float red[4][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = WPR == 1 ? lane : (int)threadIdx.x;
    int64_t row;
    int part = 0;
    if (WPR == 1) row = (int64_t)blockIdx.x * 4 + wave;
    else { row = blockIdx.x / (unsigned)a.split; part = blockIdx.x % (unsigned)a.split; }
    if (WPR == 1 && row >= a.rows) return;
    const typename X::elem* p = (const typename X::elem*)a.logits + row * a.stride;
    // 16-byte vectors of the row, the scores before the first and behind the last one
    const int head0 = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(typename X::elem);
    const int head = head0 < a.V ? head0 : a.V;
    const int nvec = (a.V - head) / N, tail = a.V - head - nvec * N;
    const int per = (nvec + a.split - 1) / a.split;
    const int v0 = part * per < nvec ? part * per : nvec, v1 = v0 + per < nvec ? v0 + per : nvec;
    const uint4* pv = (const uint4*)(p + head);

    Stat st = {LOWEST, 0.f, 0.f};
    TopList top;
    if (TOP) top.init(a.top, keys + wave * 128, lane);
    bool first = true;
    for (int v = v0; v < v1; v += UNROLL * T) {
        float f[UNROLL][N], vm[UNROLL];
        uint4 q[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int at = v + i * T + t;
            if (at < v1) q[i] = pv[at];
        }
        float cm = -INFINITY;
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            X::unpack(q[i], f[i]);
            if (v + i * T + t >= v1) {
#pragma unroll
                for (int j = 0; j < N; ++j) f[i][j] = -INFINITY;
            }
            float x = f[i][0];
#pragma unroll
            for (int j = 1; j < N; ++j) x = fmaxf(x, f[i][j]);
            vm[i] = x;
            cm = fmaxf(cm, x);
        }
        add_scores(st, cm, &f[0][0], UNROLL * N);
        if (TOP) {
            if (first) { top.at_least(kth_largest(cm, a.top, lane)); first = false; }
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                const int at = v + i * T + t, base = head + at * N;
                const bool have = at < v1;
                if (!__any(have && (vm[i] > top.value || (vm[i] == top.value && base < top.index)))) continue;
#pragma unroll
                for (int j = 0; j < N; ++j) top.offer(make_key(f[i][j], base + j), have);
            }
        }
    }
    {   // the ends: at most 7 + 7 scores
        const int h = part == 0 ? head : 0, e = part == a.split - 1 ? tail : 0;
        if (h + e > 0 && (WPR == 1 || wave == 0)) {
            const bool have = lane < h + e;
            const int at = lane < h ? lane : a.V - tail + (lane - h);
            float x[1] = {-INFINITY};
            if (have) x[0] = X::get(p[at]);
            add_scores(st, x[0], x, 1);
            if (TOP) top.offer(make_key(x[0], at), have);
        }
    }
    st = wave_join(st);
    if (TOP) top.finish();
    if (WPR == 1) {
        if (lane == 0) write_row<DT>(a, row, st);
        if (TOP) write_top(a, row, st, top.list, lane);
        return;
    }
    if (lane == 0) { red[wave][0] = st.m; red[wave][1] = st.s; red[wave][2] = st.u; }
    if (TOP) keys[wave * 128 + lane] = top.list;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) st = join(st, Stat{red[w][0], red[w][1], red[w][2]});
    u64 list = 0;
    if (TOP) {
        list = top.list;
#pragma unroll
        for (int w = 1; w < 4; ++w) list = merge_descending(list, keys[w * 128 + 63 - lane], lane);
    }
    if (a.split == 1) {
        if (lane == 0) write_row<DT>(a, row, st);
        if (TOP) write_top(a, row, st, list, lane);
        return;
    }
    const int64_t at = row * a.split + part;
    if (lane == 0) { float* o = a.part_stat + at * 4; o[0] = st.m; o[1] = st.s; o[2] = st.u; }
    if (TOP && lane < a.top) a.part_key[at * a.top + lane] = list;
}

// Joins the parts of a row: one wave a row, one part a lane.
template <int DT, bool TOP>
__global__ __launch_bounds__(64) void logprob_join_kernel(const FwdArgs a) {
    __shared__ u64 keys[TOP ? 128 : 1];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const bool have = lane < a.split;
    Stat st = {LOWEST, 0.f, 0.f};
    if (have) { const float* q = a.part_stat + (row * a.split + lane) * 4; st = Stat{q[0], q[1], q[2]}; }
    st = wave_join(st);
    if (lane == 0) write_row<DT>(a, row, st);
    if (!TOP) return;
    const u64* pk = a.part_key + (row * a.split + lane) * a.top;
    TopList top;
    top.init(a.top, keys, lane);
    // the lists are sorted: the top-th largest of their first keys is a threshold where there are that many, and a list ends the search
    // once its next key is under the threshold
    u64 key = have ? pk[0] : 0;
    if (a.top <= a.split) {
        const u64 order = sort_ascending(key, lane);
        const u64 kth = shfl64(order, 64 - a.top);
        if (kth) top.raise(kth - 1);
    }
    for (int j = 0; j < a.top; ++j) {
        const bool live = have && key > top.threshold;
        if (!__any(live)) break;
        top.offer(key, live);
        key = have && j + 1 < a.top ? pk[j + 1] : 0;
    }
    top.finish();
    write_top(a, row, st, top.list, lane);
}

struct BwdArgs {
    const void* logits;
    void* grad;
    const int64_t *labels, *top_index;
    const float *stat, *entropy, *g_logp, *g_entropy, *g_top;
    int64_t rows, stride, grad_stride, ignore;
    int V, top, parts, per;       // a workgroup handles `per` vectors of a row
};

// A workgroup a part of a row; the label's and the alternatives' own terms are added by the workgroup that holds them, from the scores and
// in 32 bits, after its part is written.  grad and logits are read / written 16 bytes at a time where a row starts at the same place of a
// 16-byte block in both (always so for the gradients that ops.label_logprobs allocates), else one score at a time.
template <int DT>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(const BwdArgs a) {
    typedef Vec<DT> X;
    typedef typename X::elem elem;
    constexpr int N = X::N;
    const int64_t row = blockIdx.x / (unsigned)a.parts;
    const int part = blockIdx.x % (unsigned)a.parts, t = threadIdx.x;
    const elem* p = (const elem*)a.logits + row * a.stride;
    elem* o = (elem*)a.grad + row * a.grad_stride;
    const float m = a.stat[2 * row], ls = a.stat[2 * row + 1], H = a.entropy[row];
    const bool empty = ls == -INFINITY;
    const int64_t label = a.labels[row];
    const bool ignored = label == a.ignore;
    const bool given = !ignored && label >= 0 && label < a.V;
    float g = (a.g_logp && !ignored) ? a.g_logp[row] : 0.f;
    if (!ignored && !given) g = NAN;
    const float h = a.g_entropy ? a.g_entropy[row] : 0.f;
    float total = g;
    if (a.g_top)
        for (int j = 0; j < a.top; ++j) total += a.g_top[row * a.top + j];
    // -p (total + h (log p + H)) = -exp(d - ls) (c + h d), d = l - m
    const float c = total + h * (H - ls);
    auto value = [&](float x) {
        const float d = x - m, e = __builtin_amdgcn_exp2f((d - ls) * L2E);
        return empty ? 0.f : -e * (c + weigh(h, d));
    };
    const int head0 = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(elem);
    const int head = head0 < a.V ? head0 : a.V;
    const int nvec = (a.V - head) / N, tail0 = head + nvec * N;
    // (a row that begins off a 16-byte block can have fewer vectors than V / N: the last part is then the scores behind them)
    const int v0 = part * a.per < nvec ? part * a.per : nvec, v1 = v0 + a.per < nvec ? v0 + a.per : nvec;
    const int from = part == 0 ? 0 : head + v0 * N, to = part == a.parts - 1 ? a.V : head + v1 * N;      // scores of this workgroup
    if ((((uintptr_t)p ^ (uintptr_t)o) & 15) == 0) {
        const uint4* pv = (const uint4*)(p + head);
        uint4* ov = (uint4*)(o + head);
        for (int v = v0; v < v1; v += UNROLL * 256) {
            uint4 q[UNROLL];
#pragma unroll
            for (int i = 0; i < UNROLL; ++i)
                if (v + i * 256 + t < v1) q[i] = pv[v + i * 256 + t];
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                if (v + i * 256 + t >= v1) continue;
                float f[N];
                X::unpack(q[i], f);
#pragma unroll
                for (int j = 0; j < N; ++j) f[j] = value(f[j]);
                ov[v + i * 256 + t] = X::pack(f);
            }
        }
        if (part == 0 && t < head) o[t] = X::put(value(X::get(p[t])));
        if (part == a.parts - 1 && tail0 + t < a.V) o[tail0 + t] = X::put(value(X::get(p[tail0 + t])));
    } else {
        for (int v = from + t; v < to; v += 256) o[v] = X::put(value(X::get(p[v])));
    }
    __syncthreads();      // the part is written (the same addresses are overwritten below by other threads of this workgroup)
    if (empty) return;
    if (t <= a.top) {     // thread 0: the label, thread 1 + j: alternative j
        int64_t v = t == 0 ? (given ? label : -1) : (a.g_top ? a.top_index[row * a.top + t - 1] : -1);
        if (v >= from && v < to) {
            float add = given && v == label ? g : 0.f;
            if (a.g_top)
                for (int j = 0; j < a.top; ++j)
                    if (a.top_index[row * a.top + j] == v) add += a.g_top[row * a.top + j];
            o[v] = X::put(value(X::get(p[v])) + add);      // (written twice with one value where an alternative is the label)
        }
    }
}

int split_of(int64_t rows, int64_t V) {
    // Parts of a row: enough workgroups to cover the 256 CUs four times, at least 4096 scores each; never for rows that one wave handles.
    if (V <= 2048 || rows >= 512) return 1;
    int64_t s = 1024 / rows, most = V / 4096;
    if (s > most) s = most;
    if (s > MAX_SPLIT) s = MAX_SPLIT;
    return s < 1 ? 1 : (int)s;
}

template <int DT>
void launch_fwd(const FwdArgs& a, hipStream_t st) {
    if (a.V <= 2048) {
        const dim3 g((unsigned)wgs_cdiv(a.rows, 4));
        if (a.top) WGS_LAUNCH((logprob_fwd_kernel<DT, 1, true>), g, dim3(256), 0, st, a);
        else WGS_LAUNCH((logprob_fwd_kernel<DT, 1, false>), g, dim3(256), 0, st, a);
        return;
    }
    const dim3 g((unsigned)(a.rows * a.split));
    if (a.top) WGS_LAUNCH((logprob_fwd_kernel<DT, 4, true>), g, dim3(256), 0, st, a);
    else WGS_LAUNCH((logprob_fwd_kernel<DT, 4, false>), g, dim3(256), 0, st, a);
    if (a.split > 1) {
        if (a.top) WGS_LAUNCH((logprob_join_kernel<DT, true>), dim3((unsigned)a.rows), dim3(64), 0, st, a);
        else WGS_LAUNCH((logprob_join_kernel<DT, false>), dim3((unsigned)a.rows), dim3(64), 0, st, a);
    }
}

}  // namespace

extern "C" {

int64_t wgs_label_logprobs_ws_bytes(int64_t rows, int64_t V, int top) {
    if (rows <= 0 || V <= 0 || V >= (1LL << 31) || top < 0) return 0;
    const int s = split_of(rows, V);
    return s > 1 ? rows * s * (16 + 8 * (int64_t)top) : 0;
}

int wgs_label_logprobs_fwd(const void* logits, int dtype, int64_t rows, int64_t V, int64_t row_stride, const int64_t* labels, int64_t ignore_index, int top,
                           float* logp, float* entropy, float* stat, float* top_logp, int64_t* top_index, void* ws, int64_t ws_bytes, wgs_stream_t stream) {
    WGS_CHECK_ARG(dtype == WGS_F32 || dtype == WGS_BF16 || dtype == WGS_F16, "wgs_label_logprobs_fwd: unknown dtype %d", dtype);
    WGS_CHECK_ARG(rows >= 0 && rows < (1LL << 24) && V > 0 && V < (1LL << 30) && row_stride >= V, "wgs_label_logprobs_fwd: bad sizes (rows < 2^24, 0 < V < 2^30, row stride >= V)");
    WGS_CHECK_ARG(top >= 0 && top <= TOP_MAX && top <= V, "wgs_label_logprobs_fwd: top must be at most %d and at most V, got %d", TOP_MAX, top);
    if (rows == 0) return WGS_OK;
    WGS_CHECK_ARG(logits && labels && logp && entropy && stat && (top == 0 || (top_logp && top_index)), "wgs_label_logprobs_fwd: null pointer");
    WGS_CHECK_ARG(((uintptr_t)logits & (dtype == WGS_F32 ? 3 : 1)) == 0, "wgs_label_logprobs_fwd: logits are not aligned to their type");
    const int64_t need = wgs_label_logprobs_ws_bytes(rows, V, top);
    WGS_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), "wgs_label_logprobs_fwd: workspace of %lld bytes needed, 16-byte aligned", (long long)need);
    FwdArgs a;
    a.logits = logits; a.labels = labels; a.logp = logp; a.entropy = entropy; a.stat = stat; a.top_logp = top_logp; a.top_index = top_index;
    a.rows = rows; a.stride = row_stride; a.ignore = ignore_index; a.V = (int)V; a.top = top; a.split = split_of(rows, V);
    a.part_stat = (float*)ws;
    a.part_key = (u64*)((char*)ws + rows * a.split * 16);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WGS_F32) launch_fwd<WGS_F32>(a, st);
    else if (dtype == WGS_BF16) launch_fwd<WGS_BF16>(a, st);
    else launch_fwd<WGS_F16>(a, st);
    WGS_CHECK_LAUNCH("logprob_fwd_kernel");
    return WGS_OK;
}

int wgs_label_logprobs_bwd(const void* logits, int dtype, int64_t rows, int64_t V, int64_t row_stride, const int64_t* labels, int64_t ignore_index,
                           const float* stat, const float* entropy, int top, const int64_t* top_index, const float* g_logp, const float* g_entropy,
                           const float* g_top, void* grad, int64_t grad_row_stride, wgs_stream_t stream) {
    WGS_CHECK_ARG(dtype == WGS_F32 || dtype == WGS_BF16 || dtype == WGS_F16, "wgs_label_logprobs_bwd: unknown dtype %d", dtype);
    WGS_CHECK_ARG(rows >= 0 && rows < (1LL << 24) && V > 0 && V < (1LL << 30) && row_stride >= V && grad_row_stride >= V,
                  "wgs_label_logprobs_bwd: bad sizes (rows < 2^24, 0 < V < 2^30, row strides >= V)");
    WGS_CHECK_ARG(top >= 0 && top <= TOP_MAX && top <= V, "wgs_label_logprobs_bwd: top must be at most %d and at most V, got %d", TOP_MAX, top);
    if (rows == 0) return WGS_OK;
    WGS_CHECK_ARG(logits && labels && stat && entropy && grad && (top == 0 || !g_top || top_index), "wgs_label_logprobs_bwd: null pointer");
    const uintptr_t am = dtype == WGS_F32 ? 3 : 1;
    WGS_CHECK_ARG((((uintptr_t)logits | (uintptr_t)grad) & am) == 0, "wgs_label_logprobs_bwd: a tensor is not aligned to its type");
    BwdArgs a;
    a.logits = logits; a.grad = grad; a.labels = labels; a.top_index = top_index; a.stat = stat; a.entropy = entropy;
    a.g_logp = g_logp; a.g_entropy = g_entropy; a.g_top = top ? g_top : nullptr;
    a.rows = rows; a.stride = row_stride; a.grad_stride = grad_row_stride; a.ignore = ignore_index; a.V = (int)V; a.top = top;
    const int nv = wgs_cdiv(V, dtype == WGS_F32 ? 4 : 8);
    a.per = UNROLL * 256;
    a.parts = wgs_cdiv(nv, a.per);
    WGS_CHECK_ARG(rows * a.parts < (1LL << 24), "wgs_label_logprobs_bwd: too many scores for one launch");      // (a grid has fewer than 2^32 threads)
    hipStream_t st = (hipStream_t)stream;
    const dim3 gr((unsigned)(rows * a.parts));
    if (dtype == WGS_F32) WGS_LAUNCH(logprob_bwd_kernel<WGS_F32>, gr, dim3(256), 0, st, a);
    else if (dtype == WGS_BF16) WGS_LAUNCH(logprob_bwd_kernel<WGS_BF16>, gr, dim3(256), 0, st, a);
    else WGS_LAUNCH(logprob_bwd_kernel<WGS_F16>, gr, dim3(256), 0, st, a);
    WGS_CHECK_LAUNCH("logprob_bwd_kernel");
    return WGS_OK;
}

}  // extern "C"
