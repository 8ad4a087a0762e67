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
#include "vec16.h"

namespace lgd {

constexpr int kGaThreads = 256;

enum GaAct { kActNone = 0, kActRelu = 1, kActSilu = 2 };

struct GaArgs {
    const void* x[LGD_MAX_LEVELS];
    const void* dy[LGD_MAX_LEVELS];
    void* out[LGD_MAX_LEVELS];       // fwd: y ; bwd: dx
    int E[LGD_MAX_LEVELS];           // elements per sample, HW * C
    int HW[LGD_MAX_LEVELS];
    int spc[LGD_MAX_LEVELS];         // super-rows per chunk
    int K[LGD_MAX_LEVELS];           // chunks per sample
    int wg0[LGD_MAX_LEVELS + 1];     // first workgroup of the map: B * K per map
    int L, B, C, G, cg;
    int P, PV;                       // super-row: elements, vectors
    int cols, R, nCB;                // vectors of a column block, super-rows a workgroup covers at once, column blocks
    int W;                           // width of a chunk's record in `part`: G (forward, one column block), C (backward, one column block) or P
    double eps;
    const void* gamma;               // [C] or null
    const void* beta;
    int ptype;                       // LGD_F32 / LGD_BF16 / LGD_F16
    double* partd;                   // forward [chunk][W][2]
    float* partf;                    // backward [chunk][W][2]
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
template <typename T> __device__ __forceinline__ void ga_store(T* p, const lgd_u32x4& u) { *reinterpret_cast<typename GaU<sizeof(T)>::type*>(p) = u; }

// gamma / beta in any of the three types; null: the neutral value
__device__ __forceinline__ float ga_param(const void* p, int type, int c, float none) {
    if (!p) return none;
    if (type == LGD_F32) return static_cast<const float*>(p)[c];
    if (type == LGD_BF16) return (float)static_cast<const __bf16*>(p)[c];
    return (float)static_cast<const _Float16*>(p)[c];
}
__device__ __forceinline__ void ga_param_store(void* p, int type, int c, float v) {
    if (type == LGD_F32) static_cast<float*>(p)[c] = v;
    else if (type == LGD_BF16) static_cast<__bf16*>(p)[c] = (__bf16)v;
    else static_cast<_Float16*>(p)[c] = (_Float16)v;
}

// sigmoid: v_exp_f32 and v_rcp_f32 (one ulp each); z = -inf gives 0, +inf gives 1
__device__ __forceinline__ float ga_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z)); }

template <int ACT> __device__ __forceinline__ float ga_act(float z) {
    if (ACT == kActRelu) return z <= 0.f ? 0.f : z;   // NaN passes, as torch.relu
    if (ACT == kActSilu) return z * ga_sigmoid(z);
    return z;
}

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

// what a thread owns: vector column v of the super-row, super-rows s0 + r, s0 + r + R, ... of the chunk [s0, s1)
struct GaThread { int v, s, s1, slim, on; };
template <int V>
__device__ __forceinline__ GaThread ga_thread(const GaArgs& a, const GaWhere& q) {
    GaThread t;
    const int r = threadIdx.x / a.cols, col = threadIdx.x % a.cols;
    t.v = blockIdx.y * a.cols + col;
    t.on = r < a.R && t.v < a.PV;
    t.s = q.k * a.spc[q.l] + r;
    const int NS = (a.E[q.l] + a.P - 1) / a.P;
    t.s1 = min(NS, (q.k + 1) * a.spc[q.l]);
    if (!t.on) t.s1 = 0;
    const int room = a.E[q.l] - (t.v + 1) * V;   // the vector of super-row s is whole iff s * P <= room
    t.slim = room < 0 ? 0 : room / a.P + 1;
    return t;
}

// every vector of the thread in order, U loads in flight; the (at most one) vector that the sample's end cuts comes last, zero filled.
// load(e) starts a vector's loads into a register struct, use(regs, e, count) consumes it
template <int V, int U, typename Regs, typename Load, typename Part, typename Use>
__device__ __forceinline__ void ga_walk(const GaArgs& a, const GaThread& t, int E, Load load, Part part, Use use) {
    const int send = min(t.s1, t.slim), step = a.R * a.P;
    int s = t.s;
    long e = (long)s * a.P + (long)t.v * V;
    for (; s + (U - 1) * a.R < send; s += U * a.R, e += (long)U * step) {
        Regs q[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) q[u] = load(e + (long)u * step);
        #pragma unroll
        for (int u = 0; u < U; ++u) use(q[u], e + (long)u * step, V);
    }
    for (; s < send; s += a.R, e += step) use(load(e), e, V);
    if (s < t.s1 && e < E) use(part(e, (int)(E - e)), e, (int)(E - e));
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
// sh[position][2] for the positions of this column block.  sh holds kGaThreads * V pairs.
template <int V, typename A>
__device__ __forceinline__ void ga_block_positions(const GaArgs& a, const GaThread& t, A (&s0)[V], A (&s1)[V], A* sh) {
    const int r = threadIdx.x / a.cols, col = threadIdx.x % a.cols;
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

template <typename T>
__global__ __launch_bounds__(kGaThreads) void ga_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    __shared__ double sh[kGaThreads * V * 2];
    const GaWhere q = ga_locate(a, blockIdx.x);
    const GaThread t = ga_thread<V>(a, q);
    const int E = a.E[q.l];
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    double s0[V], s1[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.0;
    ga_walk<V, 4, GaX<T>>(a, t, E, [&](long e) { return GaX<T>{ga_load(px + e)}; }, [&](long e, int n) { return GaX<T>{ga_load_part(px + e, n)}; },
        [&](const GaX<T>& v, long, int) {
            float f[V];
            Vec16<T>::unpack(v.x, f);
            #pragma unroll
            for (int i = 0; i < V; ++i) { const double d = f[i]; s0[i] += d; s1[i] = fma(d, d, s1[i]); }
        });
    ga_block_positions<V, double>(a, t, s0, s1, sh);
    double* part = a.partd + (size_t)blockIdx.x * a.W * 2;
    if (a.nCB == 1) {   // positions -> groups
        const int wraps = a.P / a.C;
        for (int j = threadIdx.x; j < 2 * a.G; j += kGaThreads) {
            const int g = j >> 1, k = j & 1;
            double s = 0.0;
            for (int w = 0; w < wraps; ++w)
                for (int c = 0; c < a.cg; ++c) s += sh[2 * (w * a.C + g * a.cg + c) + k];
            part[j] = s;
        }
    } else {
        const int p0 = blockIdx.y * a.cols * V, np = min(a.cols * V, a.P - p0);
        for (int j = threadIdx.x; j < 2 * np; j += kGaThreads) part[2 * (size_t)p0 + j] = sh[j];
    }
}

// one wave per (map, sample, group): mean and 1 / sqrt(var + eps) from the chunks' records
__global__ __launch_bounds__(64) void ga_finalize_kernel(GaArgs a) {
    const int seg = blockIdx.x, g = seg % a.G, lb = seg / a.G, l = lb / a.B, b = lb % a.B, lane = threadIdx.x;
    const int K = a.K[l], per = a.nCB == 1 ? 1 : a.cg, wraps = a.nCB == 1 ? 1 : a.W / a.C;
    const double* p = a.partd + (size_t)(a.wg0[l] + b * K) * a.W * 2;
    double s0 = 0.0, s1 = 0.0;
    const int n = K * per * wraps;
    for (int i = lane; i < n; i += 64) {
        const int k = i / (per * wraps), j = i % (per * wraps);
        const double* v = p + 2 * ((size_t)k * a.W + (j / per) * a.C + g * per + j % per);
        s0 += v[0]; s1 += v[1];
    }
    s0 = wave_sum(s0); s1 = wave_sum(s1);
    if (lane == 0) {
        const double cnt = (double)a.HW[l] * a.cg, m = s0 / cnt;
        double var = s1 / cnt - m * m;
        var = var < 0.0 ? 0.0 : var;   // (NaN stays)
        a.stats[2 * (size_t)seg] = m;
        a.stats[2 * (size_t)seg + 1] = 1.0 / sqrt(var + a.eps);
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(kGaThreads) void ga_apply_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    const GaWhere q = ga_locate(a, blockIdx.x);
    const GaThread t = ga_thread<V>(a, q);
    const int E = a.E[q.l];
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    T* __restrict__ po = static_cast<T*>(a.out[q.l]) + (size_t)q.b * E;
    double A[V], Bc[V];
    const double* st = a.stats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
    #pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = t.on ? (t.v * V + i) % a.C : 0, g = c / a.cg;
        A[i] = st[2 * g + 1] * (double)ga_param(a.gamma, a.ptype, c, 1.f);
        Bc[i] = fma(-st[2 * g], A[i], (double)ga_param(a.beta, a.ptype, c, 0.f));
    }
    ga_walk<V, 4, GaX<T>>(a, t, E, [&](long e) { return GaX<T>{ga_load(px + e)}; }, [&](long e, int n) { return GaX<T>{ga_load_part(px + e, n)}; },
        [&](const GaX<T>& v, long e, int n) {
            float f[V];
            Vec16<T>::unpack(v.x, f);
            #pragma unroll
            for (int i = 0; i < V; ++i) f[i] = ga_act<ACT>((float)fma((double)f[i], A[i], Bc[i]));
            ga_store_n(po + e, Vec16<T>::pack(f), n);
        });
}

// g = dy act'(z) and xh of one element.  ReLU: the sign of z in fp64 (A, Bc as the forward's); SiLU: z in fp32 from xh
template <int ACT> __device__ __forceinline__ float ga_grad(float dy, float x, float xh, double A, double Bc, float ga, float be) {
    if (ACT == kActRelu) return fma((double)x, A, Bc) <= 0.0 ? 0.f : dy;
    if (ACT == kActSilu) {
        const float z = __builtin_fmaf(xh, ga, be), s = ga_sigmoid(z);
        return dy * __builtin_fmaf(z * s, 1.f - s, s);
    }
    return dy;
}

// per-channel constants of the backward
template <int ACT, int V> struct GaCoef {
    double r[V], nmr[V];     // xh = x r - mu r
    double A[V], Bc[V];      // ReLU only
    float ga[V], be[V];
    __device__ __forceinline__ void fill(const GaArgs& a, const GaWhere& q, const GaThread& t) {
        const double* st = a.stats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t.on ? (t.v * V + i) % a.C : 0, g = c / a.cg;
            r[i] = st[2 * g + 1]; nmr[i] = -st[2 * g] * r[i];
            ga[i] = ga_param(a.gamma, a.ptype, c, 1.f); be[i] = ga_param(a.beta, a.ptype, c, 0.f);
            if (ACT == kActRelu) { A[i] = r[i] * (double)ga[i]; Bc[i] = fma(-st[2 * g], A[i], (double)be[i]); }
        }
    }
};

template <typename T, int ACT>
__global__ __launch_bounds__(kGaThreads) void ga_bwd_stats_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    __shared__ float sh[kGaThreads * V * 2];
    const GaWhere q = ga_locate(a, blockIdx.x);
    const GaThread t = ga_thread<V>(a, q);
    const int E = a.E[q.l];
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const T* __restrict__ pd = static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * E;
    GaCoef<ACT, V> k;
    k.fill(a, q, t);
    float s0[V], s1[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.f;
    ga_walk<V, 2, GaXD<T>>(a, t, E, [&](long e) { return GaXD<T>{ga_load(px + e), ga_load(pd + e)}; },
        [&](long e, int n) { return GaXD<T>{ga_load_part(px + e, n), ga_load_part(pd + e, n)}; },
        [&](const GaXD<T>& v, long, int) {
            float x[V], d[V];
            Vec16<T>::unpack(v.x, x); Vec16<T>::unpack(v.d, d);   // behind a cut vector's end dy = 0: no contribution
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (float)fma((double)x[i], k.r[i], k.nmr[i]);
                const float g = ga_grad<ACT>(d[i], x[i], xh, k.A[i], k.Bc[i], k.ga[i], k.be[i]);
                s0[i] += g; s1[i] = __builtin_fmaf(g, xh, s1[i]);
            }
        });
    ga_block_positions<V, float>(a, t, s0, s1, sh);
    float* part = a.partf + (size_t)blockIdx.x * a.W * 2;
    if (a.nCB == 1) {   // positions -> channels
        const int wraps = a.P / a.C;
        for (int j = threadIdx.x; j < 2 * a.C; j += kGaThreads) {
            float s = 0.f;
            for (int w = 0; w < wraps; ++w) s += sh[2 * w * a.C + j];
            part[j] = s;
        }
    } else {
        const int p0 = blockIdx.y * a.cols * V, np = min(a.cols * V, a.P - p0);
        for (int j = threadIdx.x; j < 2 * np; j += kGaThreads) part[2 * (size_t)p0 + j] = sh[j];
    }
}

// one wave per (map, sample, group): channel sums over the chunks (kept for dgamma / dbeta) and the group's two means.  Lanes = `sub` channels x
// 64 / sub chunk slices (sub a power of two); slices meet by an xor butterfly, in a fixed order
__global__ __launch_bounds__(64) void ga_bwd_finalize_kernel(GaArgs a) {
    const int seg = blockIdx.x, g = seg % a.G, lb = seg / a.G, l = lb / a.B, b = lb % a.B, lane = threadIdx.x;
    const int K = a.K[l], wraps = a.W / a.C;
    const float* p = a.partf + (size_t)(a.wg0[l] + b * K) * a.W * 2;
    int sub = 1;
    while (sub < a.cg && sub < 64) sub <<= 1;
    double m1 = 0.0, m2 = 0.0;
    for (int c0 = 0; c0 < a.cg; c0 += sub) {
        const int j = c0 + (lane & (sub - 1)), c = g * a.cg + j;
        double s0 = 0.0, s1 = 0.0;
        if (j < a.cg)
            for (int i = lane / sub; i < K * wraps; i += 64 / sub) {
                const float* v = p + 2 * ((size_t)(i / wraps) * a.W + (i % wraps) * a.C + c);
                s0 += (double)v[0]; s1 += (double)v[1];
            }
        for (int o = sub; o < 64; o <<= 1) { s0 += __shfl_xor(s0, o); s1 += __shfl_xor(s1, o); }
        if (j < a.cg && lane < sub) {
            a.csum[2 * ((size_t)lb * a.C + c)] = s0;
            a.csum[2 * ((size_t)lb * a.C + c) + 1] = s1;
            const double ga = (double)ga_param(a.gamma, a.ptype, c, 1.f);
            m1 = fma(ga, s0, m1); m2 = fma(ga, s1, m2);
        }
    }
    m1 = wave_sum(m1); m2 = wave_sum(m2);
    if (lane == 0) {
        const double cnt = (double)a.HW[l] * a.cg;
        a.bstats[2 * (size_t)seg] = (float)(m1 / cnt);
        a.bstats[2 * (size_t)seg + 1] = (float)(m2 / cnt);
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

template <typename T, int ACT>
__global__ __launch_bounds__(kGaThreads) void ga_bwd_apply_kernel(GaArgs a) {
    constexpr int V = Vec16<T>::V;
    const GaWhere q = ga_locate(a, blockIdx.x);
    const GaThread t = ga_thread<V>(a, q);
    const int E = a.E[q.l];
    const T* __restrict__ px = static_cast<const T*>(a.x[q.l]) + (size_t)q.b * E;
    const T* __restrict__ pd = static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * E;
    T* __restrict__ po = static_cast<T*>(a.out[q.l]) + (size_t)q.b * E;
    GaCoef<ACT, V> k;
    k.fill(a, q, t);
    float c1[V], c2[V], c3[V];
    const float* bs = a.bstats + 2 * (size_t)(q.l * a.B + q.b) * a.G;
    #pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = t.on ? (t.v * V + i) % a.C : 0, g = c / a.cg;
        c1[i] = (float)(k.r[i] * (double)k.ga[i]);
        c2[i] = (float)(-k.r[i] * (double)bs[2 * g + 1]);
        c3[i] = (float)(-k.r[i] * (double)bs[2 * g]);
    }
    ga_walk<V, 2, GaXD<T>>(a, t, E, [&](long e) { return GaXD<T>{ga_load(px + e), ga_load(pd + e)}; },
        [&](long e, int n) { return GaXD<T>{ga_load_part(px + e, n), ga_load_part(pd + e, n)}; },
        [&](const GaXD<T>& v, long e, int n) {
            float x[V], d[V];
            Vec16<T>::unpack(v.x, x); Vec16<T>::unpack(v.d, d);
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (float)fma((double)x[i], k.r[i], k.nmr[i]);
                const float g = ga_grad<ACT>(d[i], x[i], xh, k.A[i], k.Bc[i], k.ga[i], k.be[i]);
                d[i] = __builtin_fmaf(c1[i], g, __builtin_fmaf(c2[i], xh, c3[i]));
            }
            ga_store_n(po + e, Vec16<T>::pack(d), n);
        });
}

static int ga_gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// the split of a call: super-rows, column blocks and chunks.  Chunks are about total / 2048 (eight workgroups of 256 threads per CU), 16 KB at least.
static int ga_plan(GaArgs& a, const int32_t* hw, int L, int B, int C, int G, int dtype) {
    if (!hw || L < 1 || L > LGD_MAX_LEVELS || B < 1 || C < 1 || G < 1 || C % G || (dtype != LGD_F32 && dtype != LGD_BF16 && dtype != LGD_F16)) return LGD_EINVAL;
    const int size = dtype == LGD_F32 ? 4 : 2, V = 16 / size;
    a = GaArgs{};
    a.L = L; a.B = B; a.C = C; a.G = G; a.cg = C / G;
    if (C > (1 << 26)) return LGD_EINVAL;
    a.P = C / ga_gcd(C, V) * V; a.PV = a.P / V;
    a.nCB = (a.PV + kGaThreads - 1) / kGaThreads;
    a.cols = (a.PV + a.nCB - 1) / a.nCB;
    a.R = kGaThreads / a.cols;
    long long total = 0;
    for (int l = 0; l < L; ++l) {
        if (hw[2 * l] < 1 || hw[2 * l + 1] < 1) return LGD_EINVAL;
        const long long n = (long long)hw[2 * l] * hw[2 * l + 1], e = n > (1LL << 31) ? n : n * C;
        if (e + 4LL * kGaThreads * a.P >= (1LL << 31)) return LGD_EINVAL;   // in-sample offsets are 32 bits
        a.E[l] = (int)e; a.HW[l] = (int)n;
        total += e * B * size;
    }
    long long bytes = total / 2048;
    if (bytes < 16384) bytes = 16384;
    long long w = 0;
    for (int l = 0; l < L; ++l) {
        const int NS = (a.E[l] + a.P - 1) / a.P;
        long long spc = (bytes + (long long)a.P * size - 1) / ((long long)a.P * size);
        spc = (spc + a.R - 1) / a.R * a.R;
        a.spc[l] = (int)(spc < NS ? spc : NS);
        a.K[l] = (NS + a.spc[l] - 1) / a.spc[l];
        a.wg0[l] = (int)w;
        w += (long long)B * a.K[l];
        if (w > 0x7fffffffLL) return LGD_EINVAL;
    }
    for (int l = L; l <= LGD_MAX_LEVELS; ++l) a.wg0[l] = (int)w;
    if ((long long)L * B * G > 0x7fffffffLL) return LGD_EINVAL;
    return LGD_OK;
}

static size_t ga_round(size_t n) { return (n + 255) & ~(size_t)255; }
static size_t ga_chunks(const GaArgs& a) { return (size_t)a.wg0[LGD_MAX_LEVELS]; }

template <typename T>
static int ga_fwd(GaArgs& a, int act, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    LGD_LAUNCH("gn_act_stats_kernel", ga_stats_kernel<T>, grid, dim3(kGaThreads), 0, s, a);
    LGD_LAUNCH("gn_act_finalize_kernel", ga_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(64), 0, s, a);
    if (act == kActNone) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActNone>), grid, dim3(kGaThreads), 0, s, a);
    else if (act == kActRelu) LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActRelu>), grid, dim3(kGaThreads), 0, s, a);
    else LGD_LAUNCH("gn_act_apply_kernel", (ga_apply_kernel<T, kActSilu>), grid, dim3(kGaThreads), 0, s, a);
    return check_launch();
}

template <typename T, int ACT>
static int ga_bwd(GaArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)ga_chunks(a), (unsigned)a.nCB);
    LGD_LAUNCH("gn_act_bwd_stats_kernel", (ga_bwd_stats_kernel<T, ACT>), grid, dim3(kGaThreads), 0, s, a);
    LGD_LAUNCH("gn_act_bwd_finalize_kernel", ga_bwd_finalize_kernel, dim3((unsigned)(a.L * a.B * a.G)), dim3(64), 0, s, a);
    if (a.dgamma || a.dbeta) LGD_LAUNCH("gn_act_bwd_param_kernel", ga_param_kernel, dim3((unsigned)((a.C + 63) / 64)), dim3(256), 0, s, a);
    if (a.out[0]) LGD_LAUNCH("gn_act_bwd_apply_kernel", (ga_bwd_apply_kernel<T, ACT>), grid, dim3(kGaThreads), 0, s, a);
    return check_launch();
}
template <typename T>
static int ga_bwd_act(GaArgs& a, int act, hipStream_t s) {
    if (act == kActNone) return ga_bwd<T, kActNone>(a, s);
    if (act == kActRelu) return ga_bwd<T, kActRelu>(a, s);
    return ga_bwd<T, kActSilu>(a, s);
}

}  // namespace lgd

extern "C" {

size_t lgd_gn_act_ws_bytes(const int32_t* level_hw_host, int L, int B, int C, int G, int dtype, int backward) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK) return 0;
    const size_t chunks = lgd::ga_chunks(a);
    if (!backward) return lgd::ga_round(chunks * (size_t)(a.nCB == 1 ? G : a.P) * 2 * sizeof(double));
    return lgd::ga_round(chunks * (size_t)(a.nCB == 1 ? C : a.P) * 2 * sizeof(float)) + lgd::ga_round((size_t)L * B * C * 2 * sizeof(double)) +
           lgd::ga_round((size_t)L * B * G * 2 * sizeof(float));
}

int lgd_gn_act_fwd(const void* const* x_host, const int32_t* level_hw_host, int L, int B, int C, int G, int dtype, const void* gamma,
                   const void* beta, int param_dtype, double eps, int act, void* ws, double* stats, void* const* y_host, void* stream) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK || !x_host || !y_host || !ws || !stats || act < 0 || act > 2 ||
        param_dtype < 0 || param_dtype > 2 || !(eps >= 0.0))
        return LGD_EINVAL;
    for (int l = 0; l < L; ++l) {
        if (!x_host[l] || !y_host[l]) return LGD_EINVAL;
        a.x[l] = x_host[l]; a.out[l] = y_host[l];
    }
    a.gamma = gamma; a.beta = beta; a.ptype = param_dtype; a.eps = eps;
    a.W = a.nCB == 1 ? G : a.P;
    a.partd = static_cast<double*>(ws); a.stats = stats;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == LGD_F32) return lgd::ga_fwd<float>(a, act, s);
    if (dtype == LGD_BF16) return lgd::ga_fwd<__bf16>(a, act, s);
    return lgd::ga_fwd<_Float16>(a, act, s);
}

int lgd_gn_act_bwd(const void* const* x_host, const void* const* dy_host, const int32_t* level_hw_host, int L, int B, int C, int G, int dtype,
                   const void* gamma, const void* beta, int param_dtype, int act, const double* stats, void* ws, void* const* dx_host,
                   void* dgamma, void* dbeta, void* stream) {
    lgd::GaArgs a;
    if (lgd::ga_plan(a, level_hw_host, L, B, C, G, dtype) != LGD_OK || !x_host || !dy_host || !ws || !stats || act < 0 || act > 2 ||
        param_dtype < 0 || param_dtype > 2)
        return LGD_EINVAL;
    for (int l = 0; l < L; ++l) {
        if (!x_host[l] || !dy_host[l] || (dx_host && !dx_host[l])) return LGD_EINVAL;
        a.x[l] = x_host[l]; a.dy[l] = dy_host[l]; a.out[l] = dx_host ? dx_host[l] : nullptr;
    }
    a.gamma = gamma; a.beta = beta; a.ptype = param_dtype; a.stats = const_cast<double*>(stats);
    a.W = a.nCB == 1 ? C : a.P;
    char* w = static_cast<char*>(ws);
    a.partf = reinterpret_cast<float*>(w);
    w += lgd::ga_round(lgd::ga_chunks(a) * (size_t)a.W * 2 * sizeof(float));
    a.csum = reinterpret_cast<double*>(w);
    w += lgd::ga_round((size_t)L * B * C * 2 * sizeof(double));
    a.bstats = reinterpret_cast<float*>(w);
    a.dgamma = dgamma; a.dbeta = dbeta;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == LGD_F32) return lgd::ga_bwd_act<float>(a, act, s);
    if (dtype == LGD_BF16) return lgd::ga_bwd_act<__bf16>(a, act, s);
    return lgd::ga_bwd_act<_Float16>(a, act, s);
}

}  // extern "C"
