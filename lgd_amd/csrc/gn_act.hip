// GroupNorm(G groups, per-channel affine) + activation over a list of CHANNELS-LAST maps (B, H_l, W_l, C in memory), fp32 / bf16 / fp16, forward and
// backward: one module shared by all maps, as gn_group.hip does for NCHW fp32 + ReLU.
//   n = HW * C/G values per (map, sample, group):   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) r,  z = gamma_c xh + beta_c,
//   y = act(z), act in {identity, ReLU, SiLU};      g = dy act'(z);  dbeta_c = sum g;  dgamma_c = sum g xh  (over maps, samples, pixels)
//   m1 = mean_grp(gamma g), m2 = mean_grp(gamma g xh);   dx = r (gamma g - m1 - xh m2)
// Memory bound: forward reads x twice and writes y, backward reads x and dy twice and writes dx (the second read can come out of the caches).
//
// Layout.  A sample is HW * C contiguous elements.  A thread owns ONE 16-byte vector column of a "super-row" of P = lcm(C, V) elements (V elements
// per 16 bytes; P = C when V divides C): stepping by whole super-rows its V channels never change, so per-channel constants and sums live in
// registers, all loads are full dwordx4 for any C, and a wave's addresses are contiguous.  Samples whose size is not a multiple of 16 bytes start
// unaligned: the vector type below carries the element's alignment and gfx950 runs global memory in unaligned access mode.
//
// Precision.  Sums of x and x^2 are fp64 (gfx950 runs fp64 FMA at the rate of unpacked fp32), the statistics stay fp64, and z = x (r gamma) +
// (beta - mu r gamma) is ONE fp64 FMA per element: the sign a ReLU's gradient hangs on is decided in 64 bits.  Sums of the backward begin in fp32: at
// most kGaTerms rows of a thread, which then join a 64-bit sum (a thread has 160 rows at 340 MB, tens of thousands at the largest sizes); from there on
// they are fp64 but for the words that pass between threads, workgroups and kernels, each one rounding to fp32.  Outputs are rounded once
// (fp32 -> 16 bits).
#include "gn_act.h"

#include <type_traits>

namespace lgd {

// Workgroups of a streaming call, about: two for every CU, in step.  8 x 320 x 256 x 256 bf16, forward / backward us: 512 168 / 290 (6.0 and
// 5.8 TB/s of the 3 and 5 times a map's bytes that they move), 768 197 / 345 (three on some CUs, four on others), 1024 177 / 299
constexpr int kGaWorkgroups = 512;
constexpr int kGaU = 4, kGaUB = 2;     // vectors (of x; of x and dy each) of a thread in flight
constexpr int kGaTerms = 256;          // terms that the backward adds in fp32 before they join a 64-bit sum
constexpr int kGaRecordsU = 8;         // records of a thread in flight
constexpr int kGaThreads = 256;        // of the kernels in between
constexpr int kGaMax = 320;            // of the streaming kernels: 192, 256 or 320, whichever has a vector for most of its threads
constexpr int kGaFusedG = 512;         // groups of a fused call at most (its statistics lie in LDS) ...
constexpr int kGaFusedRecords = 8192;  // ... and records x groups of a sample (64 - 128 KB that every workgroup of the apply kernel reads from the L2)

constexpr int kGaParamC = 16;          // channels of a workgroup that makes dgamma and dbeta

struct GaArgs {
    const void* x[LGD_MAX_LEVELS];
    const void* dy[LGD_MAX_LEVELS];
    void* out[LGD_MAX_LEVELS];       // fwd: y ; bwd: dx
    int E[LGD_MAX_LEVELS];           // elements per sample, HW * C
    int HW[LGD_MAX_LEVELS];
    int K[LGD_MAX_LEVELS];           // workgroups (chunks) per sample
    int wg0[LGD_MAX_LEVELS + 1];     // first workgroup of the map: B * K per map
    int L, B, C, G, cg;
    int P, PV;                       // super-row: elements, vectors
    int NT;                          // threads of a workgroup
    int cols, R, nCB;                // vectors of a column block, super-rows a workgroup covers at once, column blocks
    int mixed;                       // several column blocks that cut groups or rows: each leaves records of its own, of all groups and channels
    double eps;
    const void* gamma;               // [C] or null
    const void* beta;
    int ptype;                       // LGD_F32 / LGD_BF16 / LGD_F16
    double* partd;                   // forward [record][G][2], a record per chunk (mixed: and column block)
    float* partf;                    // backward [record][C][2]
    float* partg;                    // backward, fused: [record][G][2], the channel sums with gamma, by group
    int fused;                       // the apply kernels reduce the records themselves (no kernel in between)
    int nparam;                      // fused backward: workgroups in front of the apply kernel's own that make dgamma and dbeta
    double* stats;                   // [L*B*G][2] mean, rstd
    float* bstats;                   // [L*B*G][2] m1, m2
    double* csum;                    // [L*B][C][2] sum g, sum g xh
    void* dgamma;
    void* dbeta;
};

// a 16-byte vector at the element's own alignment
template <int ALIGN> struct GaU;
template <> struct GaU<2> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct GaU<4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };
template <typename T> __device__ __forceinline__ lgd_u32x4 ga_load(const T* p) { return *reinterpret_cast<const typename GaU<sizeof(T)>::type*>(p); }
template <typename T> __device__ __forceinline__ lgd_u32x4 ga_stream(const T* p) { return __builtin_nontemporal_load(reinterpret_cast<const typename GaU<sizeof(T)>::type*>(p)); }
template <typename T> __device__ __forceinline__ void ga_store(T* p, const lgd_u32x4& u) {
    __builtin_nontemporal_store((typename GaU<sizeof(T)>::type)u, reinterpret_cast<typename GaU<sizeof(T)>::type*>(p));
}

// The channels and groups that a column block's record holds: its own where blocks are whole groups, otherwise (one block, or mixed) all.  Position o of
// the block (element p0 + o of the super-row) is channel (p0 + o) % C: first(c) is the first position of channel c, the others follow in steps of C
struct GaBlock {
    int c0, nc, g0, ng, np, shift, C;
    __device__ __forceinline__ int first(int c) const { const int o = c - shift; return o < 0 ? o + C : o; }
};
template <int V> __device__ __forceinline__ GaBlock ga_block(const GaArgs& a) {
    const int p0 = blockIdx.y * a.cols * V;
    GaBlock q = {0, a.C, 0, a.G, min(a.cols * V, a.P - p0), p0 % a.C, a.C};
    if (a.nCB > 1 && !a.mixed) {
        q.c0 = p0; q.nc = q.np;
        q.g0 = q.c0 / a.cg; q.ng = q.nc / a.cg;
    }
    return q;
}
__device__ __forceinline__ int ga_per_chunk(const GaArgs& a) { return a.mixed ? a.nCB : 1; }   // records of a chunk
__device__ __forceinline__ size_t ga_record(const GaArgs& a) { return a.mixed ? (size_t)blockIdx.x * a.nCB + blockIdx.y : blockIdx.x; }

struct GaWhere { int l, b, k; };
__device__ __forceinline__ GaWhere ga_locate(const GaArgs& a, int w) {
    int l = 0;
    #pragma unroll
    for (int i = 1; i < LGD_MAX_LEVELS; ++i) l += (i < a.L && w >= a.wg0[i]) ? 1 : 0;
    const int local = w - a.wg0[l];
    GaWhere q;
    q.l = l; q.b = local / a.K[l]; q.k = local % a.K[l];
    return q;
}

// what a thread owns: vector column v of the super-row, super-rows r, r + R, ... of the blocks of U * R super-rows k, k + K, ... of its sample (the
// sample's workgroups sweep it side by side: a contiguous run for each reads 10 % slower)
struct GaThread { int v, r, on, send; };   // send: super-rows in which the thread's vector is whole
template <int V>
__device__ __forceinline__ GaThread ga_thread(const GaArgs& a, int E) {
    GaThread t;
    t.r = threadIdx.x / a.cols;
    t.v = blockIdx.y * a.cols + (threadIdx.x - t.r * a.cols);
    t.on = t.r < a.R && t.v < a.PV;
    const int room = E - (t.v + 1) * V;   // the vector of super-row s is whole iff s * P <= room
    t.send = !t.on || room < 0 ? 0 : room / a.P + 1;
    return t;
}

// A thread's way through its vectors, U in flight: begin() issues the first block's loads (kernels that have something to compute first call it in
// front of that), run() consumes them and goes on.  load(e): a whole vector's registers; use(regs, e, count); part(e, count): the one vector that the
// sample's end cuts, zero filled, comes last; turn(): behind every U vectors
template <int V, int U, typename Regs> struct GaWalk {
    int s, K, block, step, send;
    unsigned e;   // element offset of super-row s (wraps only behind the last one, where it is not used)
    Regs v[U];
    template <typename Load> __device__ __forceinline__ void loads(const GaArgs& a, Load load) {
        #pragma unroll
        for (int u = 0; u < U; ++u) if (s + u * a.R < send) v[u] = load(e + u * step);
    }
    template <typename Load> __device__ __forceinline__ void begin(const GaArgs& a, const GaWhere& q, const GaThread& t, Load load) {
        K = a.K[q.l]; block = U * a.R; step = a.R * a.P; send = t.send;
        s = q.k * block + t.r;
        e = (unsigned)s * a.P + t.v * V;
        loads(a, load);
    }
    template <typename Load, typename Part, typename Use, typename Turn>
    __device__ __forceinline__ void run(const GaArgs& a, const GaWhere& q, const GaThread& t, int E, Load load, Part part, Use use, Turn turn) {
        while (s < send) {
            #pragma unroll
            for (int u = 0; u < U; ++u) if (s + u * a.R < send) use(v[u], e + u * step, V);
            s += K * block; e += (unsigned)(K * U) * step;
            loads(a, load);
            turn();
        }
        if (a.P == a.C || !t.on) return;   // samples are whole vectors
        const unsigned cut = (unsigned)send * a.P + t.v * V;
        if (cut < (unsigned)E && send / block % K == q.k && send % a.R == t.r) use(part(cut, E - cut), cut, E - cut);
    }
    template <typename Load, typename Part, typename Use>
    __device__ __forceinline__ void run(const GaArgs& a, const GaWhere& q, const GaThread& t, int E, Load load, Part part, Use use) {
        run(a, q, t, E, load, part, use, [] {});
    }
};

// the channels of the thread's V lanes and their groups, f(lane, channel, group) (one division for all of them)
template <int V, typename F>
__device__ __forceinline__ void ga_lanes(const GaArgs& a, const GaThread& t, F f) {
    int c = t.on ? t.v * V % a.C : 0, g = c / a.cg, m = c - g * a.cg;
    #pragma unroll
    for (int i = 0; i < V; ++i) {
        f(i, c, g);
        ++c; ++m;
        if (m == a.cg) { m = 0; ++g; }
        if (c == a.C) { c = 0; g = 0; }
    }
}

template <typename T> struct GaX { lgd_u32x4 x; };
template <typename T> struct GaXD { lgd_u32x4 x, d; };

// count (1 .. V - 1) elements, the rest zero: all loads at once, those behind the end from the last element (branches around them wait for each other, 5 us)
template <typename T> __device__ __forceinline__ lgd_u32x4 ga_load_part(const T* p, int count) {
    T tmp[Vec16<T>::V];
    #pragma unroll
    for (int i = 0; i < Vec16<T>::V; ++i) tmp[i] = p[i < count ? i : count - 1];
    #pragma unroll
    for (int i = 0; i < Vec16<T>::V; ++i) tmp[i] = i < count ? tmp[i] : (T)0.f;
    lgd_u32x4 u;
    __builtin_memcpy(&u, tmp, 16);
    return u;
}
template <typename T> __device__ __forceinline__ void ga_store_n(T* p, const lgd_u32x4& u, int count) {
    if (count == Vec16<T>::V) { ga_store(p, u); return; }
    T tmp[Vec16<T>::V];
    __builtin_memcpy(tmp, &u, 16);
    #pragma unroll
    for (int i = 0; i < Vec16<T>::V; ++i) if (i < count) p[i] = tmp[i];
}

// Pieces.  W = gcd(cg, V) consecutive lanes of a vector lie in one group (groups, rows and vectors all end at multiples of W), so a thread holds
// S = V / W pieces: V = 8: one for groups of 8, 16, ... channels, two for 20, four for 30, eight for odd ones.

// ---- sums of a workgroup: pairs that the threads left in LDS, n bins of rows x per terms each; term(bin, r, c) -> the pair, put(bin, s0, s1).  Few bins
// are split over the threads, neighbours taking neighbouring terms, and joined eight at a time in a fixed order.  Barriers inside, none in front
template <typename Term, typename Put>
__device__ __forceinline__ void ga_bins(int nt, int n, int rows, int per, Term term, Put put) {
    __shared__ double2 tmp[kGaMax];
    const int terms = rows * per;
    int m = 1;   // threads of a bin
    while (2 * m * n <= nt && m < terms) m <<= 1;
    if (m == 1) {
        for (int j = threadIdx.x; j < n; j += nt) {
            double s0 = 0.0, s1 = 0.0;
            for (int r = 0; r < rows; ++r)
                for (int c = 0; c < per; ++c) { const auto v = term(j, r, c); s0 += (double)v.x; s1 += (double)v.y; }
            put(j, s0, s1);
        }
        return;
    }
    const int j = threadIdx.x / m, first = threadIdx.x & (m - 1);
    double s0 = 0.0, s1 = 0.0;
    if (j < n) {
        const int dr = m / per, dc = m - dr * per;
        for (int r = first / per, c = first - r * per; r < rows;) {
            const auto v = term(j, r, c);
            s0 += (double)v.x; s1 += (double)v.y;
            r += dr; c += dc;
            if (c >= per) { c -= per; ++r; }
        }
    }
    __syncthreads();   // (tmp may be in use by an earlier call)
    tmp[threadIdx.x] = make_double2(s0, s1);
    for (;;) {
        __syncthreads();
        const int next = m > 8 ? m >> 3 : 1, step = m / next;
        const bool on = (int)threadIdx.x < n * next;
        const int bin = threadIdx.x / next, k = threadIdx.x - bin * next;
        if (on) {
            s0 = s1 = 0.0;
            for (int i = 0; i < step; ++i) { const double2 v = tmp[bin * m + k + i * next]; s0 += v.x; s1 += v.y; }
        }
        if (next == 1) {
            if (on) put(bin, s0, s1);
            return;
        }
        __syncthreads();
        if (on) tmp[threadIdx.x] = make_double2(s0, s1);
        m = next;
    }
}

constexpr int kGaPad = kGaMax + 1;   // pairs between the pieces of a thread: neighbouring threads and neighbouring pieces lie on different banks

// the groups' sums of a column block out of the threads' pieces sh[piece][thread]
template <int V, int S, typename P2, typename Put>
__device__ __forceinline__ void ga_piece_groups(const GaArgs& a, const GaBlock& blk, const P2* sh, Put put) {
    constexpr int W = V / S;
    const int per = a.cg / W, Cp = a.C / W, np = blk.np / W, shift = blk.shift / W;
    ga_bins(a.NT, blk.ng, a.R, per, [&](int g, int r, int c) {
        int o = (blk.g0 + g) * per + c - shift;
        if (o < 0) o += Cp;
        P2 s = {};
        for (; o < np; o += Cp) { const P2 v = sh[(o & (S - 1)) * kGaPad + r * a.cols + o / S]; s.x += v.x; s.y += v.y; }
        return s;
    }, put);
}

template <typename T, int S>
__global__ __launch_bounds__(kGaMax) void ga_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V, W = V / S;
    __shared__ double2 sh[S * kGaPad];
    const GaWhere q = ga_locate(a, blockIdx.x);
    const int E = a.E[q.l];
    const GaThread t = ga_thread<V>(a, E);
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const auto load = [&](unsigned e) { return GaX<T>{ga_load(px + e)}; };
    GaWalk<V, kGaU, GaX<T>> walk;
    walk.begin(a, q, t, load);
    double s0[S], s1[S];
    #pragma unroll
    for (int i = 0; i < S; ++i) s0[i] = s1[i] = 0.0;
    walk.run(a, q, t, E, load,
        [&](unsigned e, int n) { return GaX<T>{ga_load_part(px + e, n)}; },
        [&](const GaX<T>& v, unsigned, int) {
            float f[V];
            Vec16<T>::unpack(v.x, f);
            #pragma unroll
            for (int i = 0; i < V; ++i) { const double d = f[i]; s0[i / W] += d; s1[i / W] = fma(d, d, s1[i / W]); }
        });
    double2* part = reinterpret_cast<double2*>(a.partd) + ga_record(a) * a.G;
    const GaBlock blk = ga_block<V>(a);
    #pragma unroll
    for (int i = 0; i < S; ++i) sh[i * kGaPad + threadIdx.x] = make_double2(s0[i], s1[i]);
    __syncthreads();
    ga_piece_groups<V, S>(a, blk, sh, [&](int g, double g0, double g1) { part[blk.g0 + g] = make_double2(g0, g1); });
}

// mean and 1 / sqrt(var + eps) of a group of n values with sums s0, s1
__device__ __forceinline__ void ga_moments(double s0, double s1, double n, double eps, double& mean, double& rstd) {
    mean = s0 / n;
    double var = s1 / n - mean * mean;
    var = var < 0.0 ? 0.0 : var;   // (NaN stays)
    rstd = 1.0 / sqrt(var + eps);
}

// one workgroup per (map, sample, group): its statistics from the chunks' records
__global__ __launch_bounds__(kGaThreads) void ga_finalize_kernel(GaArgs a) {
    __shared__ double sh[4][2];
    const int seg = blockIdx.x, g = seg % a.G, lb = seg / a.G, l = lb / a.B, b = lb % a.B;
    const int n = a.K[l] * ga_per_chunk(a);
    const double2* p = reinterpret_cast<const double2*>(a.partd) + (size_t)(a.wg0[l] + b * a.K[l]) * ga_per_chunk(a) * a.G + g;
    double s0 = 0.0, s1 = 0.0;
    for (int i = threadIdx.x; i < n; i += kGaThreads) { const double2 v = p[(size_t)i * a.G]; s0 += v.x; s1 += v.y; }
    s0 = wave_sum(s0); s1 = wave_sum(s1);
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6][0] = s0; sh[threadIdx.x >> 6][1] = s1; }
    __syncthreads();
    if (threadIdx.x == 0)
        ga_moments((sh[0][0] + sh[1][0]) + (sh[2][0] + sh[3][0]), (sh[0][1] + sh[1][1]) + (sh[2][1] + sh[3][1]), (double)a.HW[l] * a.cg, a.eps,
                   a.stats[2 * (size_t)seg], a.stats[2 * (size_t)seg + 1]);
}

// sums of the K records of G pairs of one sample, by every workgroup that needs them: put(g, s0, s1).  Threads = groups x slices of the records; the
// slices meet in LDS, in a fixed order.  P2: pair of the records.  Barriers inside
template <typename P2, typename Put>
__device__ __forceinline__ void ga_records(int nt, const P2* __restrict__ p, int K, int G, const GaBlock& blk, Put put) {
    __shared__ double2 tmp[kGaMax];
    int sub = 1;
    while (sub < blk.ng && 2 * sub <= nt) sub <<= 1;
    const int slices = nt / sub, sl = threadIdx.x / sub;
    const int gend = blk.g0 + blk.ng;
    for (int g0 = blk.g0; g0 < gend; g0 += sub) {
        const int g = g0 + (threadIdx.x & (sub - 1));
        double s0 = 0.0, s1 = 0.0;
        if (g < gend && sl < slices) {
            for (int k = sl; k < K; k += kGaRecordsU * slices) {
                P2 v[kGaRecordsU];
                #pragma unroll
                for (int u = 0; u < kGaRecordsU; ++u) { v[u] = P2{}; if (k + u * slices < K) v[u] = p[(size_t)(k + u * slices) * G + g]; }
                #pragma unroll
                for (int u = 0; u < kGaRecordsU; ++u) { s0 += (double)v[u].x; s1 += (double)v[u].y; }
            }
        }
        if (slices > 1) tmp[threadIdx.x] = make_double2(s0, s1);
        for (int m = slices; m > 1;) {   // eight at a time
            const int next = (m + 7) >> 3;
            __syncthreads();
            if (sl < next) {
                s0 = s1 = 0.0;
                for (int i = sl; i < m; i += next) { const double2 v = tmp[threadIdx.x + (i - sl) * sub]; s0 += v.x; s1 += v.y; }
            }
            m = next;
            __syncthreads();
            if (m > 1 && sl < m) tmp[threadIdx.x] = make_double2(s0, s1);
        }
        if (sl == 0 && g < gend) put(g, s0, s1);
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(kGaMax) void ga_apply_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    const GaWhere q = ga_locate(a, blockIdx.x);
    const int E = a.E[q.l];
    const GaThread t = ga_thread<V>(a, E);
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    T* __restrict__ po = static_cast<T*>(a.out[q.l]) + (size_t)q.b * E;
    const auto load = [&](unsigned e) { return GaX<T>{ga_stream(px + e)}; };
    GaWalk<V, kGaU, GaX<T>> walk;
    walk.begin(a, q, t, load);
    int c[V], g[V];
    ga_lanes<V>(a, t, [&](int i, int ci, int gi) { c[i] = ci; g[i] = gi; });
    uint32_t wga[V] = {}, wbe[V] = {};   // (asked for in front of the barriers)
    ga_param_words<V>(a.gamma, a.ptype, c, wga);
    ga_param_words<V>(a.beta, a.ptype, c, wbe);
    double A[V], Bc[V];
    double* gst = a.stats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
    const double* st = gst;
    if (a.fused) {   // the statistics from the chunks' records; the sample's first workgroup leaves them for the backward
        __shared__ double sst[2 * kGaFusedG];
        const double n = (double)a.HW[q.l] * a.cg;
        const int rec = ga_per_chunk(a);
        ga_records(a.NT, reinterpret_cast<const double2*>(a.partd) + (size_t)(a.wg0[q.l] + q.b * a.K[q.l]) * rec * a.G, a.K[q.l] * rec, a.G, ga_block<V>(a), [&](int g, double s0, double s1) {
            double m, r;
            ga_moments(s0, s1, n, a.eps, m, r);
            sst[2 * g] = m; sst[2 * g + 1] = r;
            if (q.k == 0 && (!a.mixed || blockIdx.y == 0)) { gst[2 * g] = m; gst[2 * g + 1] = r; }
        });
        __syncthreads();
        st = sst;
    }
    {
        float ga[V], be[V];
        ga_param_values<V>(a.gamma, a.ptype, wga, 1.f, ga);
        ga_param_values<V>(a.beta, a.ptype, wbe, 0.f, be);
        #pragma unroll
        for (int i = 0; i < V; ++i) { A[i] = st[2 * g[i] + 1] * (double)ga[i]; Bc[i] = fma(-st[2 * g[i]], A[i], (double)be[i]); }
    }
    walk.run(a, q, t, E, load, [&](unsigned e, int n) { return GaX<T>{ga_load_part(px + e, n)}; },
        [&](const GaX<T>& v, unsigned e, int n) {
            float f[V];
            Vec16<T>::unpack(v.x, f);
            #pragma unroll
            for (int i = 0; i < V; ++i) f[i] = ga_act<ACT>(ga_single(fma((double)f[i], A[i], Bc[i])));
            ga_store_n(po + e, Vec16<T>::pack(f), n);
        });
}

// constants of a thread's V lanes in S pieces
template <int V, int S> struct GaCoef {
    static constexpr int W = V / S;
    GaGroup grp[S];
    float ga[V], be[V];
    __device__ __forceinline__ void fill(const GaArgs& a, const GaWhere& q, const GaThread& t) {
        const double2* st = reinterpret_cast<const double2*>(a.stats) + (size_t)(q.l * a.B + q.b) * a.G;
        int c[V];
        double2 m[S];
        ga_lanes<V>(a, t, [&](int i, int ci, int gi) {
            c[i] = ci;
            if (i % W == 0) m[i / W] = st[gi];
        });
        uint32_t wga[V] = {}, wbe[V] = {};
        ga_param_words<V>(a.gamma, a.ptype, c, wga);
        ga_param_words<V>(a.beta, a.ptype, c, wbe);
        ga_param_values<V>(a.gamma, a.ptype, wga, 1.f, ga);
        ga_param_values<V>(a.beta, a.ptype, wbe, 0.f, be);
        #pragma unroll
        for (int i = 0; i < S; ++i) grp[i] = ga_group(m[i].x, m[i].y);
    }
    __device__ __forceinline__ const GaGroup& at(int i) const { return grp[i / W]; }
};

template <typename T, int ACT, int S>
__global__ __launch_bounds__(kGaMax) void ga_bwd_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V, W = V / S;
    // 64-bit sums of the blocks of kGaTerms terms before the last (written by long chunks only: in registers they cost 16-bit types a wave per SIMD, 12 - 17 %
    // on odd channels); then the threads' sums and, with gamma, the groups' pieces
    __shared__ double2 acc[V * kGaPad];
    float2* sh = reinterpret_cast<float2*>(acc);
    float2* shg = sh + V * kGaPad;
    const GaWhere q = ga_locate(a, blockIdx.x);
    const int E = a.E[q.l];
    const GaThread t = ga_thread<V>(a, E);
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const T* __restrict__ pd = static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * E;
    const auto load = [&](unsigned e) { return GaXD<T>{ga_load(px + e), ga_load(pd + e)}; };
    GaWalk<V, kGaUB, GaXD<T>> walk;
    walk.begin(a, q, t, load);
    GaCoef<V, S> k;
    k.fill(a, q, t);
    float s0[V], s1[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.f;
    int turns = 0, blocks = 0;
    walk.run(a, q, t, E, load,
        [&](unsigned e, int n) { return GaXD<T>{ga_load_part(px + e, n), ga_load_part(pd + e, n)}; },
        [&](const GaXD<T>& v, unsigned, int) {
            float x[V], d[V];
            Vec16<T>::unpack(v.x, x); Vec16<T>::unpack(v.d, d);   // behind a cut vector's end dy = 0: no contribution
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = ga_xhat(x[i], k.at(i)), g = ga_grad<ACT>(d[i], x[i], xh, k.at(i), k.ga[i], k.be[i]);
                s0[i] += g; s1[i] = __builtin_fmaf(g, xh, s1[i]);
            }
        },
        [&] {
            if (++turns < kGaTerms / kGaUB) return;
            turns = 0;
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                double2& t = acc[i * kGaPad + threadIdx.x];
                const double2 before = blocks ? t : make_double2(0.0, 0.0);
                t = make_double2(before.x + (double)s0[i], before.y + (double)s1[i]);
                s0[i] = s1[i] = 0.f;
            }
            ++blocks;
        });
    // (the same for the whole workgroup: no thread of a shorter chunk has got that far)
    if (E / a.P + 1 > (kGaTerms - kGaUB) * a.R * a.K[q.l]) {
        if (blocks) {
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const double2 t = acc[i * kGaPad + threadIdx.x];
                s0[i] = (float)(t.x + (double)s0[i]); s1[i] = (float)(t.y + (double)s1[i]);
            }
        }
        __syncthreads();
    }
    #pragma unroll
    for (int i = 0; i < V; ++i) sh[i * kGaPad + threadIdx.x] = make_float2(s0[i], s1[i]);
    if (a.fused) {   // with gamma, for the groups
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            float g0 = 0.f, g1 = 0.f;
            #pragma unroll
            for (int m = 0; m < W; ++m) { g0 = __builtin_fmaf(k.ga[i * W + m], s0[i * W + m], g0); g1 = __builtin_fmaf(k.ga[i * W + m], s1[i * W + m], g1); }
            shg[i * kGaPad + threadIdx.x] = make_float2(g0, g1);
        }
    }
    __syncthreads();
    float2* part = reinterpret_cast<float2*>(a.partf) + ga_record(a) * a.C;
    const GaBlock blk = ga_block<V>(a);
    ga_bins(a.NT, blk.nc, a.R, 1, [&](int c, int r, int) {   // positions -> channels
        float2 s = {};
        for (int o = blk.first(blk.c0 + c); o < blk.np; o += a.C) { const float2 v = sh[(o & (V - 1)) * kGaPad + r * a.cols + o / V]; s.x += v.x; s.y += v.y; }
        return s;
    }, [&](int c, double c0, double c1) { part[blk.c0 + c] = make_float2((float)c0, (float)c1); });
    if (a.fused) {
        float2* gp = reinterpret_cast<float2*>(a.partg) + ga_record(a) * a.G;
        ga_piece_groups<V, S>(a, blk, shg, [&](int g, double g0, double g1) { gp[blk.g0 + g] = make_float2((float)g0, (float)g1); });
    }
}

// one workgroup per (map, sample, group): channel sums over the chunks (kept for dgamma / dbeta) and the group's two means.  Threads = `sub` channels x
// 256 / sub slices of the chunks (sub a power of two); the slices meet in a tree, in a fixed order.  (One wave per group left 33 - 47 us of load
// latency in this kernel.)
__global__ __launch_bounds__(256) void ga_bwd_finalize_kernel(GaArgs a) {
    __shared__ double sh[256][2];
    const int seg = blockIdx.x, g = seg % a.G, lb = seg / a.G, l = lb / a.B, b = lb % a.B, tid = threadIdx.x;
    const int n = a.K[l] * ga_per_chunk(a);
    const float2* p = reinterpret_cast<const float2*>(a.partf) + (size_t)(a.wg0[l] + b * a.K[l]) * ga_per_chunk(a) * a.C;
    int sub = 1;
    while (sub < a.cg && sub < 256) sub <<= 1;
    double m1 = 0.0, m2 = 0.0;
    for (int c0 = 0; c0 < a.cg; c0 += sub) {
        const int j = c0 + (tid & (sub - 1)), c = g * a.cg + j, slices = 256 / sub;
        double s0 = 0.0, s1 = 0.0;
        if (j < a.cg) {
            auto at = [&](int i) { return p[(size_t)i * a.C + c]; };
            int i = tid / sub;
            for (; i + 3 * slices < n; i += 4 * slices) {
                float2 v[4];
                #pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = at(i + u * slices);
                #pragma unroll
                for (int u = 0; u < 4; ++u) { s0 += (double)v[u].x; s1 += (double)v[u].y; }
            }
            for (; i < n; i += slices) { const float2 v = at(i); s0 += (double)v.x; s1 += (double)v.y; }
        }
        sh[tid][0] = s0; sh[tid][1] = s1;
        __syncthreads();
        for (int o = 128; o >= sub; o >>= 1) {
            if (tid < o) { sh[tid][0] += sh[tid + o][0]; sh[tid][1] += sh[tid + o][1]; }
            __syncthreads();
        }
        if (tid < sub && j < a.cg) {
            s0 = sh[tid][0]; s1 = sh[tid][1];
            a.csum[2 * ((size_t)lb * a.C + c)] = s0;
            a.csum[2 * ((size_t)lb * a.C + c) + 1] = s1;
            const double ga = (double)ga_param(a.gamma, a.ptype, c, 1.f);
            m1 = fma(ga, s0, m1); m2 = fma(ga, s1, m2);
        }
        __syncthreads();
    }
    m1 = wave_sum(m1); m2 = wave_sum(m2);
    if ((tid & 63) == 0) { sh[tid >> 6][0] = m1; sh[tid >> 6][1] = m2; }
    __syncthreads();
    if (tid == 0) {
        const double cnt = (double)a.HW[l] * a.cg;
        a.bstats[2 * (size_t)seg] = (float)(((sh[0][0] + sh[1][0]) + (sh[2][0] + sh[3][0])) / cnt);
        a.bstats[2 * (size_t)seg + 1] = (float)(((sh[0][1] + sh[1][1]) + (sh[2][1] + sh[3][1])) / cnt);
    }
}

// dgamma, dbeta: the channel sums over every (map, sample); 64 channels x 4 slices per workgroup
__global__ __launch_bounds__(256) void ga_param_kernel(GaArgs a) {
    __shared__ double sh[4][64][2];
    const int j = threadIdx.x & 63, sl = threadIdx.x >> 6, c = blockIdx.x * 64 + j;
    double s0 = 0.0, s1 = 0.0;
    if (c < a.C)
        for (int i = sl; i < a.L * a.B; i += 4) { const double* v = a.csum + 2 * ((size_t)i * a.C + c); s0 += v[0]; s1 += v[1]; }
    sh[sl][j][0] = s0; sh[sl][j][1] = s1;
    __syncthreads();
    if (sl == 0 && c < a.C) {
        s0 = (sh[0][j][0] + sh[1][j][0]) + (sh[2][j][0] + sh[3][j][0]);
        s1 = (sh[0][j][1] + sh[1][j][1]) + (sh[2][j][1] + sh[3][j][1]);
        if (a.dbeta) ga_param_store(a.dbeta, a.ptype, c, (float)s0);
        if (a.dgamma) ga_param_store(a.dgamma, a.ptype, c, (float)s1);
    }
}

// dgamma, dbeta of 16 channels: the channel sums of every chunk of every (map, sample); 16 channels x NT / 16 slices of the records
__device__ __forceinline__ void ga_params(const GaArgs& a) {
    __shared__ double sh[kGaMax][2];
    const int c = blockIdx.x * kGaParamC + (threadIdx.x & 15), sl = threadIdx.x >> 4, slices = a.NT >> 4, n = a.wg0[LGD_MAX_LEVELS] * ga_per_chunk(a);
    const float2* __restrict__ p = reinterpret_cast<const float2*>(a.partf);
    double s0 = 0.0, s1 = 0.0;
    if (c < a.C) {
        int i = sl;
        for (; i + 7 * slices < n; i += 8 * slices) {
            float2 v[8];
            #pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p[(size_t)(i + u * slices) * a.C + c];
            #pragma unroll
            for (int u = 0; u < 8; ++u) { s0 += (double)v[u].x; s1 += (double)v[u].y; }
        }
        for (; i < n; i += slices) { const float2 v = p[(size_t)i * a.C + c]; s0 += (double)v.x; s1 += (double)v.y; }
    }
    sh[threadIdx.x][0] = s0; sh[threadIdx.x][1] = s1;
    __syncthreads();
    if (sl == 0 && c < a.C) {
        for (int i = 1; i < slices; ++i) { s0 += sh[threadIdx.x + 16 * i][0]; s1 += sh[threadIdx.x + 16 * i][1]; }
        if (a.dbeta) ga_param_store(a.dbeta, a.ptype, c, (float)s0);
        if (a.dgamma) ga_param_store(a.dgamma, a.ptype, c, (float)s1);
    }
}
__global__ __launch_bounds__(kGaMax) void ga_params_kernel(GaArgs a) { ga_params(a); }

template <typename T, int ACT, int S>
__global__ __launch_bounds__(kGaMax) void ga_bwd_apply_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V, W = V / S;
    if ((int)blockIdx.x < a.nparam) {   // the first workgroups of a fused call: dgamma, dbeta out of all the chunks' channel sums
        if (blockIdx.y == 0) ga_params(a);
        return;
    }
    const GaWhere q = ga_locate(a, blockIdx.x - a.nparam);
    const int E = a.E[q.l];
    const GaThread t = ga_thread<V>(a, E);
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const T* __restrict__ pd = static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * E;
    T* __restrict__ po = static_cast<T*>(a.out[q.l]) + (size_t)q.b * E;
    const auto load = [&](unsigned e) { return GaXD<T>{ga_stream(px + e), ga_stream(pd + e)}; };
    GaWalk<V, kGaUB, GaXD<T>> walk;
    walk.begin(a, q, t, load);
    GaCoef<V, S> k;
    k.fill(a, q, t);
    const float* bs = a.bstats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
    if (a.fused) {   // the two means from the chunks' records
        __shared__ float sbs[2 * kGaFusedG];
        const double n = (double)a.HW[q.l] * a.cg;
        const int rec = ga_per_chunk(a);
        ga_records(a.NT, reinterpret_cast<const float2*>(a.partg) + (size_t)(a.wg0[q.l] + q.b * a.K[q.l]) * rec * a.G, a.K[q.l] * rec, a.G, ga_block<V>(a),
                   [&](int g, double s0, double s1) { sbs[2 * g] = (float)(s0 / n); sbs[2 * g + 1] = (float)(s1 / n); });
        __syncthreads();
        bs = sbs;
    }
    float c2[S], c3[S];
    ga_lanes<V>(a, t, [&](int i, int, int g) {
        if (i % W == 0) { c2[i / W] = -k.at(i).r * bs[2 * g + 1]; c3[i / W] = -k.at(i).r * bs[2 * g]; }
    });
    walk.run(a, q, t, E, load,
        [&](unsigned e, int n) { return GaXD<T>{ga_load_part(px + e, n), ga_load_part(pd + e, n)}; },
        [&](const GaXD<T>& v, unsigned e, int n) {
            float x[V], d[V];
            Vec16<T>::unpack(v.x, x); Vec16<T>::unpack(v.d, d);
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = ga_xhat(x[i], k.at(i)), g = ga_grad<ACT>(d[i], x[i], xh, k.at(i), k.ga[i], k.be[i]);
                d[i] = __builtin_fmaf(k.at(i).r * k.ga[i], g, __builtin_fmaf(c2[i / W], xh, c3[i / W]));
            }
            ga_store_n(po + e, Vec16<T>::pack(d), n);
        });
}

static int ga_gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// the split of a call: super-rows, column blocks and chunks
static int ga_plan(GaArgs& a, const int32_t* hw, int L, int B, int C, int G, int dtype) {
    if (!hw || L < 1 || L > LGD_MAX_LEVELS || B < 1 || C < 1 || G < 1 || C % G || (dtype != LGD_F32 && dtype != LGD_BF16 && dtype != LGD_F16)) return LGD_EINVAL;
    const int size = dtype == LGD_F32 ? 4 : 2, V = 16 / size;
    a = GaArgs{};
    a.L = L; a.B = B; a.C = C; a.G = G; a.cg = C / G;
    if (C > (1 << 26)) return LGD_EINVAL;
    a.P = C / ga_gcd(C, V) * V; a.PV = a.P / V;
    a.nCB = (a.PV + kGaMax - 1) / kGaMax;
    a.cols = (a.PV + a.nCB - 1) / a.nCB;
    a.mixed = a.nCB > 1;
    const int unit = a.cg / ga_gcd(a.cg, V);   // vectors of lcm(cg, V) channels: column blocks of whole groups, where one fits
    if (a.mixed && a.P == C && unit <= kGaMax) {
        a.cols = (a.cols + unit - 1) / unit * unit;
        if (a.cols > kGaMax) a.cols = kGaMax / unit * unit;
        a.nCB = (a.PV + a.cols - 1) / a.cols;
        a.mixed = 0;
    }
    // threads: 256, or where that leaves more than a tenth without a vector, the width of which most have one (160 vectors a row: two rows for 320; 16 x 1280
    // x 32 x 32 bf16 backward 49 us against 54).  240 of 256 stay: 320 took 4 % longer on 8 x 320 x 256 x 256
    a.NT = kGaThreads;
    for (int nt = 192; nt <= kGaMax && a.NT / a.cols * a.cols * 10 < a.NT * 9; nt += 64)
        if (nt >= a.cols && nt / a.cols * a.cols * a.NT > a.NT / a.cols * a.cols * nt) a.NT = nt;
    a.R = a.NT / a.cols;
    long long total = 0;
    for (int l = 0; l < L; ++l) {
        if (hw[2 * l] < 1 || hw[2 * l + 1] < 1) return LGD_EINVAL;
        const long long n = (long long)hw[2 * l] * hw[2 * l + 1], e = n > (1LL << 31) ? n : n * C;
        if (e + 8LL * a.R * a.P >= (1LL << 31)) return LGD_EINVAL;   // in-sample offsets are 32 bits
        a.E[l] = (int)e; a.HW[l] = (int)n;
        total += e * B * size;
    }
    // a chunk is `bytes` of a sample for each of its nCB workgroups, and a block of U super-rows a thread at least: more chunks than that hold nothing, and
    // leave records of zeros (2 x 2047 x 30 x 30 fp32, 7 column blocks: forward 45 -> 20 us, both directions 178 -> 53; 4 x 2048 x 40 x 40, 2 blocks of
    // whole groups: 84 -> 79)
    const long long bytes = (total / kGaWorkgroups < 16384 ? 16384 : total / kGaWorkgroups) * a.nCB;
    const long long block = (long long)kGaU * a.R * a.P * size;
    const int rec = a.mixed ? a.nCB : 1;
    const long long cap = kGaFusedRecords / ((long long)G * rec);
    long long w = 0, wf = 0;
    for (int l = 0; l < L; ++l) {
        const long long sample = (long long)a.E[l] * size, want = (sample + bytes - 1) / bytes, most = (sample + block - 1) / block;
        const long long k = want < most ? want : most;
        a.K[l] = (int)k;
        w += B * k;
        wf += B * (k < cap ? k : cap);
    }
    // one kernel less where the records are few enough without leaving the chip short of workgroups
    a.fused = G <= kGaFusedG && cap >= 1 && (wf == w || wf * a.nCB >= 384);
    if ((w + C / kGaParamC + 1) * a.NT > 0xffffffffLL || w * a.nCB > 0x3fffffffLL || (!a.fused && (long long)L * B * G * kGaThreads > 0xffffffffLL) ||
        (long long)L * B * G > 0x3fffffffLL)
        return LGD_EINVAL;   // (threads of a launch; 32-bit numbers of records and statistics)
    w = 0;
    for (int l = 0; l < L; ++l) {
        if (a.fused && a.K[l] > cap) a.K[l] = (int)cap;
        a.wg0[l] = (int)w;
        w += (long long)B * a.K[l];
    }
    for (int l = L; l <= LGD_MAX_LEVELS; ++l) a.wg0[l] = (int)w;
    return LGD_OK;
}

static size_t ga_round(size_t n) { return (n + 255) & ~(size_t)255; }
static size_t ga_chunks(const GaArgs& a) { return (size_t)a.wg0[LGD_MAX_LEVELS]; }
static size_t ga_rows(const GaArgs& a) { return ga_chunks(a) * (size_t)(a.mixed ? a.nCB : 1); }   // records of a call

template <typename T, int S>
static int ga_fwd_s(GaArgs& a, int act, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    LGD_LAUNCH("gn_act_stats_kernel", (ga_stats_kernel<T, S>), grid, dim3((unsigned)a.NT), 0, s, a);
    if (!a.fused) LGD_LAUNCH("gn_act_finalize_kernel", ga_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(kGaThreads), 0, s, a);
    if (act == kActNone) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActNone>), grid, dim3((unsigned)a.NT), 0, s, a);
    else if (act == kActRelu) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActRelu>), grid, dim3((unsigned)a.NT), 0, s, a);
    else LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActSilu>), grid, dim3((unsigned)a.NT), 0, s, a);
    return check_launch();
}

// f(pieces of a vector)
template <typename T, typename F>
static int ga_pieces(const GaArgs& a, F f) {
    constexpr int V = Vec16<T>::V;
    const int S = V / ga_gcd(a.cg, V);
    if (S == 1) return f(std::integral_constant<int, 1>());
    if (S == 2) return f(std::integral_constant<int, 2>());
    if constexpr (V == 8) if (S == 4) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, V>());
}
template <typename T>
static int ga_fwd(GaArgs& a, int act, hipStream_t s) {
    return ga_pieces<T>(a, [&](auto S) { return ga_fwd_s<T, decltype(S)::value>(a, act, s); });
}

template <typename T, int ACT, int S>
static int ga_bwd(GaArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    LGD_LAUNCH("gn_act_bwd_stats_kernel", (ga_bwd_stats_kernel<T, ACT, S>), grid, dim3((unsigned)a.NT), 0, s, a);
    const bool params = a.dgamma || a.dbeta;
    if (a.fused) {
        const unsigned np = params ? (unsigned)((a.C + kGaParamC - 1) / kGaParamC) : 0u;
        a.nparam = (int)np;
        if (a.out[0]) LGD_LAUNCH("gn_act_bwd_apply_kernel", (ga_bwd_apply_kernel<T, ACT, S>), dim3(grid.x + np, grid.y), dim3((unsigned)a.NT), 0, s, a);
        else if (params) LGD_LAUNCH("gn_act_bwd_param_kernel", ga_params_kernel, dim3(np), dim3((unsigned)a.NT), 0, s, a);
        return check_launch();
    }
    LGD_LAUNCH("gn_act_bwd_finalize_kernel", ga_bwd_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(256), 0, s, a);
    if (params) LGD_LAUNCH("gn_act_bwd_param_kernel", ga_param_kernel, dim3((unsigned)((a.C + 63) / 64)), dim3(256), 0, s, a);
    if (a.out[0]) LGD_LAUNCH("gn_act_bwd_apply_kernel", (ga_bwd_apply_kernel<T, ACT, S>), grid, dim3((unsigned)a.NT), 0, s, a);
    return check_launch();
}
template <typename T>
static int ga_bwd_any(GaArgs& a, int act, hipStream_t s) {
    return ga_pieces<T>(a, [&](auto S) {
        if (act == kActNone) return ga_bwd<T, kActNone, decltype(S)::value>(a, s);
        if (act == kActRelu) return ga_bwd<T, kActRelu, decltype(S)::value>(a, s);
        return ga_bwd<T, kActSilu, decltype(S)::value>(a, s);
    });
}

}  // namespace lgd

extern "C" {

size_t lgd_gn_act_ws_bytes(const int32_t* level_hw_host, int L, int B, int C, int G, int dtype, int backward) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK) return (size_t)-1;
    const size_t rows = lgd::ga_rows(a);
    if (lgd::ga_slab_takes(level_hw_host, L, B, C, G, dtype)) return backward && L * B > 1 ? lgd::ga_round((size_t)L * B * C * 2 * sizeof(double)) : 0;
    if (!backward) return lgd::ga_round(rows * G * 2 * sizeof(double));
    return lgd::ga_round(rows * C * 2 * sizeof(float)) + lgd::ga_round((size_t)L * B * C * 2 * sizeof(double)) +
           lgd::ga_round((size_t)L * B * G * 2 * sizeof(float)) + (a.fused ? lgd::ga_round(rows * G * 2 * sizeof(float)) : 0);
}

int lgd_gn_act_fwd(const void* const* x_host, const int32_t* level_hw_host, int L, int B, int C, int G, int dtype, const void* gamma,
                   const void* beta, int param_dtype, double eps, int act, void* ws, double* stats, void* const* y_host, void* stream) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK || !x_host || !y_host || !stats || act < 0 || act > 2 ||
        param_dtype < 0 || param_dtype > 2 || !(eps >= 0.0))
        return LGD_EINVAL;
    for (int l = 0; l < L; ++l) {
        if (!x_host[l] || !y_host[l]) return LGD_EINVAL;
        a.x[l] = x_host[l]; a.out[l] = y_host[l];
    }
    a.gamma = gamma; a.beta = beta; a.ptype = param_dtype; a.eps = eps;
    a.partd = static_cast<double*>(ws); a.stats = stats;
    hipStream_t s = (hipStream_t)stream;
    const lgd::GaCall c = {x_host, nullptr, y_host, level_hw_host, L, B, C, G, dtype, act, param_dtype, eps, gamma, beta, stats, nullptr, nullptr, nullptr};
    if (lgd::ga_slab_fwd(c, s)) return lgd::check_launch();
    if (!ws) return LGD_EINVAL;
    if (dtype == LGD_F32) return lgd::ga_fwd<float>(a, act, s);
    if (dtype == LGD_BF16) return lgd::ga_fwd<__bf16>(a, act, s);
    return lgd::ga_fwd<_Float16>(a, act, s);
}

int lgd_gn_act_bwd(const void* const* x_host, const void* const* dy_host, const int32_t* level_hw_host, int L, int B, int C, int G, int dtype,
                   const void* gamma, const void* beta, int param_dtype, int act, const double* stats, void* ws, void* const* dx_host,
                   void* dgamma, void* dbeta, void* stream) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK || !x_host || !dy_host || !stats || act < 0 || act > 2 || param_dtype < 0 ||
        param_dtype > 2)
        return LGD_EINVAL;
    for (int l = 0; l < L; ++l) {
        if (!x_host[l] || !dy_host[l] || (dx_host && !dx_host[l])) return LGD_EINVAL;
        a.x[l] = x_host[l]; a.dy[l] = dy_host[l]; a.out[l] = dx_host ? dx_host[l] : nullptr;
    }
    a.gamma = gamma; a.beta = beta; a.ptype = param_dtype; a.stats = const_cast<double*>(stats); a.dgamma = dgamma; a.dbeta = dbeta;
    hipStream_t s = (hipStream_t)stream;
    char* w = static_cast<char*>(ws);
    if (!w && !(lgd::ga_slab_takes(level_hw_host, L, B, C, G, dtype) && L * B == 1)) return LGD_EINVAL;
    a.csum = reinterpret_cast<double*>(w);
    const lgd::GaCall c = {x_host, dy_host, dx_host, level_hw_host, L, B, C, G, dtype, act, param_dtype, 0.0, gamma, beta, a.stats, a.csum, dgamma, dbeta};
    if (lgd::ga_slab_bwd(c, s)) {
        if (L * B > 1 && (dgamma || dbeta))
            LGD_LAUNCH("gn_act_bwd_param_kernel", lgd::ga_param_kernel, dim3((unsigned)((C + 63) / 64)), dim3(256), 0, s, a);
        return lgd::check_launch();
    }
    w += lgd::ga_round((size_t)L * B * C * 2 * sizeof(double));
    a.partf = reinterpret_cast<float*>(w);
    w += lgd::ga_round(lgd::ga_rows(a) * (size_t)C * 2 * sizeof(float));
    a.bstats = reinterpret_cast<float*>(w);
    w += lgd::ga_round((size_t)L * B * G * 2 * sizeof(float));
    a.partg = reinterpret_cast<float*>(w);
    if (dtype == LGD_F32) return lgd::ga_bwd_any<float>(a, act, s);
    if (dtype == LGD_BF16) return lgd::ga_bwd_any<__bf16>(a, act, s);
    return lgd::ga_bwd_any<_Float16>(a, act, s);
}

}  // extern "C"
