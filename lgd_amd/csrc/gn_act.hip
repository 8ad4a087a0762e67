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
// (beta - mu r gamma) is ONE fp64 FMA per element: the sign a ReLU's gradient hangs on is decided in 64 bits.  Sums of the backward are fp32 over one
// thread's rows of a chunk (<= a few hundred terms) and its workgroup, fp64 from there on.  Outputs are rounded once (fp32 -> 16 bits).
#include "gn_act.h"

namespace lgd {

// Workgroups of a streaming call, about: two for every CU, in step.  8 x 320 x 256 x 256 bf16, forward / backward us: 512 168 / 291, 768 197 / 345 (three on
// some CUs, four on others), 1024 177 / 299
constexpr int kGaWorkgroups = 512;
constexpr int kGaU = 4, kGaUB = 2;     // vectors (of x; of x and dy each) of a thread in flight
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
// sample's end cuts, zero filled, comes last
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
    template <typename Load, typename Part, typename Use>
    __device__ __forceinline__ void run(const GaArgs& a, const GaWhere& q, const GaThread& t, int E, Load load, Part part, Use use) {
        while (s < send) {
            #pragma unroll
            for (int u = 0; u < U; ++u) if (s + u * a.R < send) use(v[u], e + u * step, V);
            s += K * block; e += (unsigned)(K * U) * step;
            loads(a, load);
        }
        if (a.P == a.C || !t.on) return;   // samples are whole vectors
        const unsigned cut = (unsigned)send * a.P + t.v * V;
        if (cut < (unsigned)E && send / block % K == q.k && send % a.R == t.r) use(part(cut, E - cut), cut, E - cut);
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

template <typename T> __device__ __forceinline__ lgd_u32x4 ga_load_part(const T* p, int count) {   // count < V elements, the rest zero
    T tmp[Vec16<T>::V];
    #pragma unroll
    for (int i = 0; i < Vec16<T>::V; ++i) tmp[i] = i < count ? p[i] : (T)0.f;
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

// ---- sums of a workgroup: every thread brings V pairs (one per position of the super-row); fixed-order tree over the R super-rows, result in
// sh[position][2] for the positions of this column block.  sh holds kGaMax * V pairs.
template <int V, typename A>
__device__ __forceinline__ void ga_block_positions(const GaArgs& a, const GaThread& t, A (&s0)[V], A (&s1)[V], A* sh) {
    const int r = t.r, col = threadIdx.x - r * a.cols;
    int half = 1;
    while (half < a.R) half <<= 1;
    for (half >>= 1; half >= 1; half >>= 1) {
        if (t.on && r >= half && r < 2 * half) {
            A* p = sh + (long)((r - half) * a.cols + col) * V * 2;
            #pragma unroll
            for (int i = 0; i < V; ++i) { p[2 * i] = s0[i]; p[2 * i + 1] = s1[i]; }
        }
        __syncthreads();
        if (t.on && r < half && r + half < a.R) {
            const A* p = sh + (long)(r * a.cols + col) * V * 2;
            #pragma unroll
            for (int i = 0; i < V; ++i) { s0[i] += p[2 * i]; s1[i] += p[2 * i + 1]; }
        }
        __syncthreads();
    }
    if (t.on && r == 0) {
        A* p = sh + (long)col * V * 2;
        #pragma unroll
        for (int i = 0; i < V; ++i) { p[2 * i] = s0[i]; p[2 * i + 1] = s1[i]; }
    }
    __syncthreads();
}

// sums over the n terms of each of ng groups: value(g, i, k) of term i, k in {0, 1}; put(2 g + k, sum).  Few groups are split over the workgroup (a
// thread walking a whole group alone took 12 us at 512 channels), the parts meet in a tree.  Barriers inside
template <typename Value, typename Put>
__device__ __forceinline__ void ga_block_groups(int nt, int ng, int n, Value value, Put put) {
    __shared__ double tmp[kGaMax];
    const int outs = 2 * ng;
    if (outs > nt / 2) {
        for (int j = threadIdx.x; j < outs; j += nt) {
            double s = 0.0;
            for (int i = 0; i < n; ++i) s += value(j >> 1, i, j & 1);
            put(j, s);
        }
        return;
    }
    int slices = 1;
    while (2 * slices * outs <= nt) slices <<= 1;
    const int sl = threadIdx.x / outs, j = threadIdx.x - sl * outs;
    double s = 0.0;
    if (sl < slices) for (int i = sl; i < n; i += slices) s += value(j >> 1, i, j & 1);
    for (slices >>= 1; slices >= 1; slices >>= 1) {
        if (sl >= slices && sl < 2 * slices) tmp[threadIdx.x - slices * outs] = s;
        __syncthreads();
        if (sl < slices) s += tmp[threadIdx.x];
        __syncthreads();
    }
    if (sl == 0) put(j, s);
}

template <typename T, bool UG>
__global__ __launch_bounds__(kGaMax) void ga_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V, S = UG ? 1 : V;
    __shared__ double sh[kGaMax * S * 2];
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
            for (int i = 0; i < V; ++i) { const double d = f[i]; s0[UG ? 0 : i] += d; s1[UG ? 0 : i] = fma(d, d, s1[UG ? 0 : i]); }
        });
    double* part = a.partd + ga_record(a) * a.G * 2;
    const GaBlock blk = ga_block<V>(a);
    if constexpr (UG) {   // (not mixed) a thread's vectors lie in one group: its pair is all that the others need of it
        sh[2 * threadIdx.x] = s0[0]; sh[2 * threadIdx.x + 1] = s1[0];
        __syncthreads();
        const int per = a.cg / V;
        ga_block_groups(a.NT, blk.ng, a.R * per, [&](int g, int i, int k) {
            const int r = i / per;
            return sh[2 * (r * a.cols + g * per + i - r * per) + k];
        }, [&](int j, double s) { part[2 * blk.g0 + j] = s; });
    } else {
        ga_block_positions<V, double>(a, t, s0, s1, sh);
        ga_block_groups(a.NT, blk.ng, a.cg, [&](int g, int i, int k) {   // positions -> groups
            double s = 0.0;
            for (int o = blk.first((blk.g0 + g) * a.cg + i); o < blk.np; o += a.C) s += sh[2 * o + k];
            return s;
        }, [&](int j, double s) { part[2 * blk.g0 + j] = s; });
    }
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
    __shared__ double tmp[kGaMax][2];
    int sub = 1;
    while (sub < blk.ng && 2 * sub <= nt) sub <<= 1;
    const int slices = nt / sub, sl = threadIdx.x / sub;
    const int gend = blk.g0 + blk.ng;
    for (int g0 = blk.g0; g0 < gend; g0 += sub) {
        const int g = g0 + (threadIdx.x & (sub - 1));
        double s0 = 0.0, s1 = 0.0;
        if (g < gend && sl < slices) {
            int k = sl;
            for (; k + 3 * slices < K; k += 4 * slices) {
                P2 v[4];
                #pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = p[(size_t)(k + u * slices) * G + g];
                #pragma unroll
                for (int u = 0; u < 4; ++u) { s0 += (double)v[u].x; s1 += (double)v[u].y; }
            }
            for (; k < K; k += slices) { const P2 v = p[(size_t)k * G + g]; s0 += (double)v.x; s1 += (double)v.y; }
        }
        if (slices > 1) {
            tmp[threadIdx.x][0] = s0; tmp[threadIdx.x][1] = s1;
            __syncthreads();
            if (sl == 0) for (int i = 1; i < slices; ++i) { s0 += tmp[threadIdx.x + i * sub][0]; s1 += tmp[threadIdx.x + i * sub][1]; }
        }
        if (sl == 0 && g < gend) put(g, s0, s1);
        if (slices > 1) __syncthreads();
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
    ga_lanes<V>(a, t, [&](int i, int c, int g) {
        A[i] = st[2 * g + 1] * (double)ga_param(a.gamma, a.ptype, c, 1.f);
        Bc[i] = fma(-st[2 * g], A[i], (double)ga_param(a.beta, a.ptype, c, 0.f));
    });
    walk.run(a, q, t, E, load, [&](unsigned e, int n) { return GaX<T>{ga_load_part(px + e, n)}; },
        [&](const GaX<T>& v, unsigned e, int n) {
            float f[V];
            Vec16<T>::unpack(v.x, f);
            #pragma unroll
            for (int i = 0; i < V; ++i) f[i] = ga_act<ACT>(ga_single(fma((double)f[i], A[i], Bc[i])));
            ga_store_n(po + e, Vec16<T>::pack(f), n);
        });
}

// constants of a thread's V lanes; UG: V divides the channels of a group, so that a vector lies in one group
template <int V, bool UG> struct GaCoef {
    GaGroup grp[UG ? 1 : V];
    float ga[V], be[V];
    __device__ __forceinline__ void fill(const GaArgs& a, const GaWhere& q, const GaThread& t) {
        const double* st = a.stats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
        ga_lanes<V>(a, t, [&](int i, int c, int g) {
            if (!UG || i == 0) grp[UG ? 0 : i] = ga_group(st, g);
            ga[i] = ga_param(a.gamma, a.ptype, c, 1.f); be[i] = ga_param(a.beta, a.ptype, c, 0.f);
        });
    }
    __device__ __forceinline__ const GaGroup& at(int i) const { return grp[UG ? 0 : i]; }
};

template <typename T, int ACT, bool UG>
__global__ __launch_bounds__(kGaMax) void ga_bwd_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    __shared__ float sh[kGaMax * V * 2];
    const GaWhere q = ga_locate(a, blockIdx.x);
    const int E = a.E[q.l];
    const GaThread t = ga_thread<V>(a, E);
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const T* __restrict__ pd = static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * E;
    const auto load = [&](unsigned e) { return GaXD<T>{ga_load(px + e), ga_load(pd + e)}; };
    GaWalk<V, kGaUB, GaXD<T>> walk;
    walk.begin(a, q, t, load);
    GaCoef<V, UG> k;
    k.fill(a, q, t);
    float s0[V], s1[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.f;
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
        });
    ga_block_positions<V, float>(a, t, s0, s1, sh);
    float* part = a.partf + ga_record(a) * a.C * 2;
    const GaBlock blk = ga_block<V>(a);
    for (int j = threadIdx.x; j < 2 * blk.nc; j += a.NT) {   // positions -> channels, and with gamma -> groups
        const int c = blk.c0 + (j >> 1), k = j & 1, o0 = blk.first(c);
        float s = 0.f;
        for (int o = o0; o < blk.np; o += a.C) s += sh[2 * o + k];
        part[2 * blk.c0 + j] = s;
        if (o0 < blk.np) sh[2 * o0 + k] = s * ga_param(a.gamma, a.ptype, c, 1.f);   // (a channel's positions are read and written by this thread only)
    }
    if (a.fused) {
        float* gp = a.partg + ga_record(a) * a.G * 2;
        __syncthreads();
        ga_block_groups(a.NT, blk.ng, a.cg, [&](int g, int i, int k) {
            const int o = blk.first((blk.g0 + g) * a.cg + i);
            return o < blk.np ? (double)sh[2 * o + k] : 0.0;
        }, [&](int j, double s) { gp[2 * blk.g0 + j] = (float)s; });
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

template <typename T, int ACT, bool UG>
__global__ __launch_bounds__(kGaMax) void ga_bwd_apply_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
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
    GaCoef<V, UG> k;
    k.fill(a, q, t);
    float c2[UG ? 1 : V], c3[UG ? 1 : V];
    ga_lanes<V>(a, t, [&](int i, int, int g) {
        if (!UG || i == 0) { c2[UG ? 0 : i] = -k.at(i).r * bs[2 * g + 1]; c3[UG ? 0 : i] = -k.at(i).r * bs[2 * g]; }
    });
    walk.run(a, q, t, E, load,
        [&](unsigned e, int n) { return GaXD<T>{ga_load_part(px + e, n), ga_load_part(pd + e, n)}; },
        [&](const GaXD<T>& v, unsigned e, int n) {
            float x[V], d[V];
            Vec16<T>::unpack(v.x, x); Vec16<T>::unpack(v.d, d);
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = ga_xhat(x[i], k.at(i)), g = ga_grad<ACT>(d[i], x[i], xh, k.at(i), k.ga[i], k.be[i]);
                d[i] = __builtin_fmaf(k.at(i).r * k.ga[i], g, __builtin_fmaf(c2[UG ? 0 : i], xh, c3[UG ? 0 : i]));
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
    const long long bytes = total / kGaWorkgroups < 16384 ? 16384 : total / kGaWorkgroups;
    const long long block = 16LL * kGaU * a.R * a.cols;   // (U vectors a thread)
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
    a.fused = G <= kGaFusedG && cap >= 1 && (wf == w || wf >= 384);
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

template <typename T>
static int ga_fwd(GaArgs& a, int act, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    if (!a.mixed && a.cg % Vec16<T>::V == 0) LGD_LAUNCH("gn_act_stats_kernel", (ga_stats_kernel<T, true>), grid, dim3((unsigned)a.NT), 0, s, a);
    else LGD_LAUNCH("gn_act_stats_kernel", (ga_stats_kernel<T, false>), grid, dim3((unsigned)a.NT), 0, s, a);
    if (!a.fused) LGD_LAUNCH("gn_act_finalize_kernel", ga_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(kGaThreads), 0, s, a);
    if (act == kActNone) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActNone>), grid, dim3((unsigned)a.NT), 0, s, a);
    else if (act == kActRelu) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActRelu>), grid, dim3((unsigned)a.NT), 0, s, a);
    else LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActSilu>), grid, dim3((unsigned)a.NT), 0, s, a);
    return check_launch();
}

template <typename T, int ACT, bool UG>
static int ga_bwd(GaArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    LGD_LAUNCH("gn_act_bwd_stats_kernel", (ga_bwd_stats_kernel<T, ACT, UG>), grid, dim3((unsigned)a.NT), 0, s, a);
    const bool params = a.dgamma || a.dbeta;
    if (a.fused) {
        const unsigned np = params ? (unsigned)((a.C + kGaParamC - 1) / kGaParamC) : 0u;
        a.nparam = (int)np;
        if (a.out[0]) LGD_LAUNCH("gn_act_bwd_apply_kernel", (ga_bwd_apply_kernel<T, ACT, UG>), dim3(grid.x + np, grid.y), dim3((unsigned)a.NT), 0, s, a);
        else if (params) LGD_LAUNCH("gn_act_bwd_param_kernel", ga_params_kernel, dim3(np), dim3((unsigned)a.NT), 0, s, a);
        return check_launch();
    }
    LGD_LAUNCH("gn_act_bwd_finalize_kernel", ga_bwd_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(256), 0, s, a);
    if (params) LGD_LAUNCH("gn_act_bwd_param_kernel", ga_param_kernel, dim3((unsigned)((a.C + 63) / 64)), dim3(256), 0, s, a);
    if (a.out[0]) LGD_LAUNCH("gn_act_bwd_apply_kernel", (ga_bwd_apply_kernel<T, ACT, UG>), grid, dim3((unsigned)a.NT), 0, s, a);
    return check_launch();
}
template <typename T, bool UG>
static int ga_bwd_act(GaArgs& a, int act, hipStream_t s) {
    if (act == kActNone) return ga_bwd<T, kActNone, UG>(a, s);
    if (act == kActRelu) return ga_bwd<T, kActRelu, UG>(a, s);
    return ga_bwd<T, kActSilu, UG>(a, s);
}
template <typename T>
static int ga_bwd_ug(GaArgs& a, int act, hipStream_t s) { return a.cg % Vec16<T>::V ? ga_bwd_act<T, false>(a, act, s) : ga_bwd_act<T, true>(a, act, s); }

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
    if (dtype == LGD_F32) return lgd::ga_bwd_ug<float>(a, act, s);
    if (dtype == LGD_BF16) return lgd::ga_bwd_ug<__bf16>(a, act, s);
    return lgd::ga_bwd_ug<_Float16>(a, act, s);
}

}  // extern "C"
