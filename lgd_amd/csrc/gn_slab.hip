// Channels-last GroupNorm + activation in ONE pass: a workgroup owns a slab -- all pixels of one (map, sample) x one group (or a few narrow ones) -- and
// keeps it in registers between the statistics and the output: x (and dy) are read once, y (dx) is written once, one launch forward.
//   bytes moved: the floor (2 N forward, 3 N backward, against 3 N and 5 N of the streaming kernels); no partial sums through memory.
// What it costs: a row of a slab is only C/G * ng elements long, so a 128-byte line is shared by several workgroups.  They are neighbours in blockIdx
// order AFTER the XCD swizzle (workgroup i runs on XCD i % 8: each XCD gets a contiguous eighth of a map's slabs), so that the line is fetched once
// into their common L2 and its pieces are merged there on the way out.
// Atoms: a thread's memory accesses are VW dwords (4, 2 or 1, what divides the slab's row); thread t owns atom column t % VR of rows t / VR, + rows, ...
#include "gn_act.h"

namespace lgd {

constexpr int kSlabThreads = 1024;
constexpr int kSlabCh = 1024;     // channels of a slab at most
constexpr int kSlabSmall = 16, kSlabLarge = 24;   // dwords of a tensor that a thread holds, two instances

struct SlabArgs {
    const void* x[LGD_MAX_LEVELS];
    const void* dy[LGD_MAX_LEVELS];
    void* out[LGD_MAX_LEVELS];
    int HW[LGD_MAX_LEVELS];
    int wg0[LGD_MAX_LEVELS + 1];     // first workgroup of the map, a multiple of 8
    int cnt;                         // slabs per map: B * G / ng
    int L, B, C, G, cg, ng;          // ng: groups of a slab
    int VR, rows;                    // atoms of a slab's row; rows a workgroup covers at once
    int act, ptype;
    double eps;
    const void* gamma;
    const void* beta;
    double* stats;
    double* csum;                    // for the parameter kernel; null when one (map, sample) is all there is
    void* dgamma;                    // set when one (map, sample) is all there is: written here
    void* dbeta;
};

template <int VW, int ALIGN> struct SlabU;
template <> struct SlabU<1, 2> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct SlabU<1, 4> { typedef uint32_t type; };
template <> struct SlabU<2, 2> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct SlabU<2, 4> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct SlabU<4, 2> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct SlabU<4, 4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };
template <int VW> struct SlabReg { uint32_t w[VW]; };

template <typename T, int VW> __device__ __forceinline__ SlabReg<VW> slab_load(const char* p) {
    SlabReg<VW> r;
    const auto v = *reinterpret_cast<const typename SlabU<VW, sizeof(T)>::type*>(p);
    if constexpr (VW == 1) r.w[0] = v;
    else {
        #pragma unroll
        for (int i = 0; i < VW; ++i) r.w[i] = v[i];
    }
    return r;
}
template <typename T, int VW> __device__ __forceinline__ void slab_store(char* p, const SlabReg<VW>& r) {
    typename SlabU<VW, sizeof(T)>::type v;
    if constexpr (VW == 1) v = r.w[0];
    else {
        #pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = r.w[i];
    }
    *reinterpret_cast<typename SlabU<VW, sizeof(T)>::type*>(p) = v;
}
// element i of an atom and back
template <typename T> __device__ __forceinline__ float slab_get(const uint32_t* w, int i) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
    else if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, (i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else { const lgd_f16x2 h = __builtin_bit_cast(lgd_f16x2, w[i >> 1]); return (i & 1) ? (float)h.y : (float)h.x; }
}
template <typename T, int E> __device__ __forceinline__ void slab_pack(const float* f, uint32_t* w) {
    if constexpr (sizeof(T) == 4) {
        #pragma unroll
        for (int i = 0; i < E; ++i) w[i] = __builtin_bit_cast(uint32_t, f[i]);
    } else {
        #pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            if constexpr (__is_same(T, __bf16)) w[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
            else { const lgd_f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]}; w[i] = __builtin_bit_cast(uint32_t, h); }
        }
    }
}

// makes the values unknown to the compiler (no instruction): what the first pass unpacked is unpacked again in the second, instead of staying in registers
template <int VW, int N> __device__ __forceinline__ void slab_forget(SlabReg<VW> (&x)[N]) {
    #pragma unroll
    for (int u = 0; u < N; ++u) {
        #pragma unroll
        for (int i = 0; i < VW; ++i) asm volatile("" : "+v"(x[u].w[i]));
    }
}

struct SlabWhere { int l, b, sl; bool on; };
__device__ __forceinline__ SlabWhere slab_locate(const SlabArgs& a) {
    SlabWhere q;
    int l = 0;
    #pragma unroll
    for (int i = 1; i < LGD_MAX_LEVELS; ++i) l += (i < a.L && (int)blockIdx.x >= a.wg0[i]) ? 1 : 0;
    const int loc = (int)blockIdx.x - a.wg0[l], n8 = (a.wg0[l + 1] - a.wg0[l]) >> 3;
    const int idx = (loc & 7) * n8 + (loc >> 3), per = a.G / a.ng;
    q.l = l; q.on = idx < a.cnt;
    q.b = idx / per; q.sl = idx - q.b * per;
    return q;
}

// threads that a map's slabs need: the waves behind them end at once (a barrier does not wait for ended waves), so that the workgroups of a call's small
// maps leave room for one another (12 x 64 channels on five maps from 27 x 45, 32 groups, forward 18.3 -> 10.6 us)
__device__ __forceinline__ int slab_threads(const SlabArgs& a, int HW) { return HW < a.rows ? (HW * a.VR + 63) & ~63 : (int)blockDim.x; }

// two sums over the workgroup's nt threads, in every thread (fixed order; sh: 32 words).  Barriers inside
__device__ __forceinline__ void slab_sum(int nt, double& v0, double& v1, double* sh) {
    v0 = wave_sum(v0); v1 = wave_sum(v1);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { sh[2 * (threadIdx.x >> 6)] = v0; sh[2 * (threadIdx.x >> 6) + 1] = v1; }
    __syncthreads();
    const int nw = nt >> 6;
    v0 = sh[0]; v1 = sh[1];
    for (int i = 1; i < nw; ++i) { v0 += sh[2 * i]; v1 += sh[2 * i + 1]; }
}

// the groups of a thread's E lanes: one for all of them when the slab is one group
template <int E, bool MULTI> struct SlabLanes {
    GaGroup grp[MULTI ? E : 1];
    int lg[MULTI ? E : 1];
    float ga[E], be[E];
    __device__ __forceinline__ const GaGroup& at(int i) const { return grp[MULTI ? i : 0]; }
};

template <typename T, int VW, int NW, bool MULTI>
__global__ __launch_bounds__(kSlabThreads) void slab_fwd_kernel(SlabArgs a) {
    constexpr int E = VW * 4 / (int)sizeof(T), N = NW / VW;
    __shared__ double sh[32];
    const SlabWhere q = slab_locate(a);
    if (!q.on) return;
    const int HW = a.HW[q.l], t = threadIdx.x, nt = slab_threads(a, HW), row0 = t / a.VR, col = t - row0 * a.VR;
    if (t >= nt) return;
    const int c0 = q.sl * a.ng * a.cg + col * E;
    // a uniform base and 32-bit byte offsets
    const char* px = reinterpret_cast<const char*>(static_cast<const T*>(a.x[q.l]) + (size_t)q.b * HW * a.C);
    char* po = reinterpret_cast<char*>(static_cast<T*>(a.out[q.l]) + (size_t)q.b * HW * a.C);
    // atoms u <= full of all threads are rows of the slab but for the last one's tail
    const unsigned step = (unsigned)a.rows * (unsigned)a.C * (unsigned)sizeof(T);
    const int full = HW / a.rows, mine = row0 >= a.rows ? 0 : row0 < HW - full * a.rows ? full + 1 : full;
    SlabReg<VW> x[N];
    {
        unsigned e = ((unsigned)row0 * a.C + c0) * (unsigned)sizeof(T);
        #pragma unroll
        for (int u = 0; u < N; ++u, e += step) {
            if (u < mine) x[u] = slab_load<T, VW>(px + e);
        }
    }
    int c[E];
    uint32_t wga[E] = {}, wbe[E] = {};   // (asked for in front of the barriers)
    #pragma unroll
    for (int i = 0; i < E; ++i) c[i] = mine ? c0 + i : 0;
    ga_param_words<E>(a.gamma, a.ptype, c, wga);
    ga_param_words<E>(a.beta, a.ptype, c, wbe);
    int lg[MULTI ? E : 1];   // the lanes' groups in the slab
    if constexpr (MULTI) {
        #pragma unroll
        for (int i = 0; i < E; ++i) lg[i] = (col * E + i) / a.cg;
    }
    double s0[MULTI ? E : 1] = {}, s1[MULTI ? E : 1] = {};
    #pragma unroll
    for (int u = 0; u < N; ++u) {
        if (u >= mine) continue;
        #pragma unroll
        for (int i = 0; i < E; ++i) {
            const double d = (double)slab_get<T>(x[u].w, i);
            s0[MULTI ? i : 0] += d; s1[MULTI ? i : 0] = fma(d, d, s1[MULTI ? i : 0]);
        }
    }
    const double cnt = (double)HW * a.cg;
    double mu[MULTI ? E : 1], r[MULTI ? E : 1];
    for (int j = 0; j < a.ng; ++j) {
        double g0 = 0.0, g1 = 0.0;
        if constexpr (MULTI) {
            #pragma unroll
            for (int i = 0; i < E; ++i) if (lg[i] == j) { g0 += s0[i]; g1 += s1[i]; }
        } else { g0 = s0[0]; g1 = s1[0]; }
        slab_sum(nt, g0, g1, sh);
        const double m = g0 / cnt;
        double var = g1 / cnt - m * m;
        var = var < 0.0 ? 0.0 : var;   // (NaN stays)
        const double rs = 1.0 / sqrt(var + a.eps);
        if (t == 0) {
            double* o = a.stats + 2 * ((size_t)(q.l * a.B + q.b) * a.G + q.sl * a.ng + j);
            o[0] = m; o[1] = rs;
        }
        if constexpr (MULTI) {
            #pragma unroll
            for (int i = 0; i < E; ++i) if (lg[i] == j) { mu[i] = m; r[i] = rs; }
        } else { mu[0] = m; r[0] = rs; }
    }
    double A[E], Bc[E];   // z = x (r gamma) + (beta - mu r gamma), one fp64 FMA
    {
        float ga[E], be[E];
        ga_param_values<E>(a.gamma, a.ptype, wga, 1.f, ga);
        ga_param_values<E>(a.beta, a.ptype, wbe, 0.f, be);
        #pragma unroll
        for (int i = 0; i < E; ++i) { A[i] = r[MULTI ? i : 0] * (double)ga[i]; Bc[i] = fma(-mu[MULTI ? i : 0], A[i], (double)be[i]); }
    }
    unsigned e = ((unsigned)row0 * a.C + c0) * (unsigned)sizeof(T);
    slab_forget(x);
    asm volatile("" : "+v"(e));   // offsets computed again: those of the loads would stay in N registers until here
    #pragma unroll
    for (int u = 0; u < N; ++u, e += step) {
        if (u >= mine) continue;
        float z[E];
        #pragma unroll
        for (int i = 0; i < E; ++i) z[i] = ga_single(fma((double)slab_get<T>(x[u].w, i), A[i], Bc[i]));
        if (a.act == kActRelu) {
            #pragma unroll
            for (int i = 0; i < E; ++i) z[i] = ga_act<kActRelu>(z[i]);
        } else if (a.act == kActSilu) {
            #pragma unroll
            for (int i = 0; i < E; ++i) z[i] = ga_act<kActSilu>(z[i]);
        }
        slab_pack<T, E>(z, x[u].w);
        slab_store<T, VW>(po + e, x[u]);
    }
}

// per-channel sums of the workgroup: every thread brings E values (channels col * E + i of its rows); in sh as [row][channel], summed eight rows at a
// time in a fixed order; the result in sh[0 .. Cs).  Barriers inside
template <int E>
__device__ __forceinline__ void slab_channels(const SlabArgs& a, int nt, int nrows, int row0, int col, const float (&v)[E], float* sh) {
    const int Cs = a.VR * E, t = threadIdx.x;
    __syncthreads();
    if (row0 < nrows) {
        #pragma unroll
        for (int i = 0; i < E; ++i) sh[row0 * Cs + col * E + i] = v[i];
    }
    __syncthreads();
    for (int n = nrows; n > 1;) {
        const int m = (n + 7) >> 3;
        for (int j = t; j < m * Cs; j += nt) {
            const int r = j / Cs, c = j - r * Cs;
            float s = sh[j];
            #pragma unroll
            for (int k = 1; k < 8; ++k) if (r + k * m < n) s += sh[(r + k * m) * Cs + c];
            sh[j] = s;   // row r < m is read by this thread only
        }
        __syncthreads();
        n = m;
    }
}

template <typename T, int VW, int NW, bool MULTI, int ACT>
__device__ __forceinline__ void slab_bwd_body(const SlabArgs& a, const SlabWhere& q, float* sh, float (*ch)[2], float (*gm)[2]) {
    constexpr int E = VW * 4 / (int)sizeof(T), N = NW / VW;
    const int HW = a.HW[q.l], t = threadIdx.x, nt = slab_threads(a, HW), nrows = HW < a.rows ? HW : a.rows, row0 = t / a.VR, col = t - row0 * a.VR;
    if (t >= nt) return;
    const int cb = q.sl * a.ng * a.cg, c0 = cb + col * E, lb = q.l * a.B + q.b;
    const char* px = reinterpret_cast<const char*>(static_cast<const T*>(a.x[q.l]) + (size_t)q.b * HW * a.C);
    const char* pd = reinterpret_cast<const char*>(static_cast<const T*>(a.dy[q.l]) + (size_t)q.b * HW * a.C);
    // atoms u <= full of all threads are rows of the slab but for the last one's tail
    const unsigned step = (unsigned)a.rows * (unsigned)a.C * (unsigned)sizeof(T);
    const int full = HW / a.rows, mine = row0 >= a.rows ? 0 : row0 < HW - full * a.rows ? full + 1 : full;
    SlabReg<VW> x[N], d[N];
    {
        unsigned e = ((unsigned)row0 * a.C + c0) * (unsigned)sizeof(T);
        #pragma unroll
        for (int u = 0; u < N; ++u, e += step) {
            if (u < mine) { x[u] = slab_load<T, VW>(px + e); d[u] = slab_load<T, VW>(pd + e); }
        }
    }
    SlabLanes<E, MULTI> k;
    const double2* st = reinterpret_cast<const double2*>(a.stats) + (size_t)lb * a.G + q.sl * a.ng;
    {
        double2 m[MULTI ? E : 1];
        int c[E];
        #pragma unroll
        for (int i = 0; i < E; ++i) {
            c[i] = mine ? c0 + i : 0;
            if constexpr (MULTI) { k.lg[i] = mine ? (col * E + i) / a.cg : 0; m[i] = st[k.lg[i]]; }
        }
        if constexpr (!MULTI) m[0] = st[0];
        uint32_t wga[E] = {}, wbe[E] = {};
        ga_param_words<E>(a.gamma, a.ptype, c, wga);
        ga_param_words<E>(a.beta, a.ptype, c, wbe);
        ga_param_values<E>(a.gamma, a.ptype, wga, 1.f, k.ga);
        ga_param_values<E>(a.beta, a.ptype, wbe, 0.f, k.be);
        #pragma unroll
        for (int i = 0; i < (MULTI ? E : 1); ++i) k.grp[i] = ga_group(m[i].x, m[i].y);
    }
    float s0[E] = {}, s1[E] = {};
    #pragma unroll
    for (int u = 0; u < N; ++u) {
        if (u >= mine) continue;
        #pragma unroll
        for (int i = 0; i < E; ++i) {
            const float xv = slab_get<T>(x[u].w, i), xh = ga_xhat(xv, k.at(i)), g = ga_grad<ACT>(slab_get<T>(d[u].w, i), xv, xh, k.at(i), k.ga[i], k.be[i]);
            s0[i] += g; s1[i] = __builtin_fmaf(g, xh, s1[i]);
            if constexpr (sizeof(T) == 4 && ACT != kActNone) d[u].w[i] = __builtin_bit_cast(uint32_t, g);
        }
    }
    const int Cs = a.VR * E;
    slab_channels<E>(a, nt, nrows, row0, col, s0, sh);
    for (int j = t; j < Cs; j += nt) ch[j][0] = sh[j];
    slab_channels<E>(a, nt, nrows, row0, col, s1, sh);
    for (int j = t; j < Cs; j += nt) {
        const float u0 = ch[j][0], u1 = sh[j];
        ch[j][1] = u1;
        if (a.csum) {
            double* o = a.csum + 2 * ((size_t)lb * a.C + cb + j);
            o[0] = (double)u0; o[1] = (double)u1;
        }
        if (a.dbeta) ga_param_store(a.dbeta, a.ptype, cb + j, u0);
        if (a.dgamma) ga_param_store(a.dgamma, a.ptype, cb + j, u1);
    }
    __syncthreads();
    const double cnt = (double)HW * a.cg;
    const int nw = nt >> 6;
    for (int j = t >> 6; j < a.ng; j += nw) {   // a wave per group
        double m1 = 0.0, m2 = 0.0;
        for (int c = t & 63; c < a.cg; c += 64) {
            const double ga = (double)ga_param(a.gamma, a.ptype, cb + j * a.cg + c, 1.f);
            m1 = fma(ga, (double)ch[j * a.cg + c][0], m1); m2 = fma(ga, (double)ch[j * a.cg + c][1], m2);
        }
        m1 = wave_sum(m1); m2 = wave_sum(m2);
        if ((t & 63) == 0) { gm[j][0] = (float)(m1 / cnt); gm[j][1] = (float)(m2 / cnt); }
    }
    if (!a.out[0]) return;
    __syncthreads();
    char* po = reinterpret_cast<char*>(static_cast<T*>(a.out[q.l]) + (size_t)q.b * HW * a.C);
    float c2[MULTI ? E : 1], c3[MULTI ? E : 1];
    #pragma unroll
    for (int i = 0; i < (MULTI ? E : 1); ++i) {
        const int j = MULTI ? k.lg[i] : 0;
        c2[i] = -k.at(i).r * gm[j][1]; c3[i] = -k.at(i).r * gm[j][0];
    }
    unsigned e = ((unsigned)row0 * a.C + c0) * (unsigned)sizeof(T);
    slab_forget(x); slab_forget(d);
    asm volatile("" : "+v"(e));   // offsets computed again: those of the loads would stay in N registers until here
    #pragma unroll
    for (int u = 0; u < N; ++u, e += step) {
        if (u >= mine) continue;
        float f[E];
        #pragma unroll
        for (int i = 0; i < E; ++i) {
            const float xv = slab_get<T>(x[u].w, i), xh = ga_xhat(xv, k.at(i));
            float g = slab_get<T>(d[u].w, i);
            if constexpr (sizeof(T) != 4) g = ga_grad<ACT>(g, xv, xh, k.at(i), k.ga[i], k.be[i]);
            f[i] = __builtin_fmaf(k.at(i).r * k.ga[i], g, __builtin_fmaf(c2[MULTI ? i : 0], xh, c3[MULTI ? i : 0]));
        }
        slab_pack<T, E>(f, x[u].w);
        slab_store<T, VW>(po + e, x[u]);
    }
}

template <typename T, int VW, int NW, bool MULTI>
__global__ __launch_bounds__(kSlabThreads) void slab_bwd_kernel(SlabArgs a) {
    constexpr int E = VW * 4 / (int)sizeof(T);
    extern __shared__ float sh[];   // rows x channels, then the channels' and the groups' pairs
    const SlabWhere q = slab_locate(a);
    if (!q.on) return;
    const int Cs = a.VR * E;
    float (*ch)[2] = reinterpret_cast<float (*)[2]>(sh + (size_t)a.rows * Cs);
    float (*gm)[2] = ch + Cs;
    if (a.act == kActNone) slab_bwd_body<T, VW, NW, MULTI, kActNone>(a, q, sh, ch, gm);
    else if (a.act == kActRelu) slab_bwd_body<T, VW, NW, MULTI, kActRelu>(a, q, sh, ch, gm);
    else slab_bwd_body<T, VW, NW, MULTI, kActSilu>(a, q, sh, ch, gm);
}

// the split of a call: dwords of an atom, registers, threads.  false: not a call for these kernels
struct SlabPlan { int VW, NT; bool large, multi; };
static bool slab_plan(SlabArgs& a, SlabPlan& p, const GaCall& c) {
    const bool shape_only = !c.x;
    const int size = c.dtype == LGD_F32 ? 4 : 2, cg = c.C / c.G;
    int most = 0;
    for (int l = 0; l < c.L; ++l) { const int n = c.hw[2 * l] * c.hw[2 * l + 1]; most = n > most ? n : most; }
    int ng = 1;
    // narrow groups side by side: rows of 16 bytes where the small kernel holds them; two at least where one group's row is no whole dword
    while (ng * cg * size % 16 && ng * cg * size < 16 && c.G % (2 * ng) == 0 && (long long)most * 2 * ng * cg * size <= 4LL * kSlabSmall * kSlabThreads) ng *= 2;
    const int row = ng * cg * size;
    if (row % 4) return false;
    p.VW = row % 16 == 0 ? 4 : row % 8 == 0 ? 2 : 1;
    if (ng > 1 && size == 2 && p.VW == 4) p.VW = 2;   // a group for each of 8 lanes does not fit the registers
    // One workgroup does all of a slab's arithmetic on one CU, the streaming kernels spread it over the chip at the price of a second read and a second
    // launch: what decides is the number of elements on the busiest CU.  Measured on 150 shapes, B 1 - 16, 33 - 1280 channels, 8^2 - 64^2 pixels (us, this
    // kernel / streaming, forward and backward):  2 K elements 4.7 / 9.8, 7.9 / 13.3;  8 K 5.3 / 9.9, 9.9 / 13.4;  18 K 8.7 / 12.7, 19.8 / 20.6;  33 K 9.9 /
    // 10.7, 19.2 / 14.9.  Rows under 16 bytes cost more of the lines' traffic (18 K at 4 bytes 17 / 11), rows of under 8 elements that only dwords divide
    // twice the accesses as well (5 fp32 channels, 20 K: 20 / 12; 11 of them, 18 K: 10.9 / 11.9), several groups their sums one by one (33 K: 11.4 / 10.1)
    long long total = 0;
    for (int l = 0; l < c.L; ++l) total += (long long)c.hw[2 * l] * c.hw[2 * l + 1] * c.B * c.C;
    const long long slab = (long long)most * ng * cg, cu = slab > total / 256 ? slab : total / 256;
    if (cu > 24576LL * (row < 16 ? row : 16) / 16 / (p.VW == 1 && row < 8 * size ? 2 : 1) / (ng > 1 ? 2 : 1)) return false;
    a = SlabArgs{};
    a.VR = row / (4 * p.VW);
    if (a.VR > kSlabThreads || ng * cg > kSlabCh || (long long)most * c.C * size >= (1LL << 32)) return false;   // (32-bit offsets in a sample)
    for (int k = 0; k < 2; ++k) {
        p.large = k == 1;
        const int N = (p.large ? kSlabLarge : kSlabSmall) / p.VW;
        const long long atoms = (long long)most * a.VR;
        if (p.large && (ng > 1 || size == 2)) return false;   // (16-bit slabs of 24576 elements fit the small one)
        // about four atoms a thread, at most N
        long long nt = (atoms + 3) / 4;
        const long long need = (atoms + N - 1) / N;
        nt = nt < need ? need : nt;
        nt = nt < a.VR ? a.VR : nt;
        nt = (nt + 63) / 64 * 64;
        if (nt > kSlabThreads) nt = kSlabThreads;
        a.rows = (int)(nt / a.VR);
        if (a.rows < 1) continue;
        while ((long long)a.rows * N < most && nt < kSlabThreads) { nt += 64; a.rows = (int)(nt / a.VR); }
        if ((long long)a.rows * N < most) continue;
        p.NT = (int)nt;
        p.multi = ng > 1;
        a.ng = ng; a.L = c.L; a.B = c.B; a.C = c.C; a.G = c.G; a.cg = cg;
        a.cnt = c.B * (c.G / ng);
        long long w = 0;
        for (int l = 0; l < LGD_MAX_LEVELS; ++l) {
            a.wg0[l] = (int)w;
            if (l >= c.L) continue;
            if (!shape_only) a.x[l] = c.x[l];
            a.dy[l] = c.dy ? c.dy[l] : nullptr; a.out[l] = c.out ? c.out[l] : nullptr;
            a.HW[l] = c.hw[2 * l] * c.hw[2 * l + 1];
            w += ((long long)a.cnt + 7) / 8 * 8;
            if (w * p.NT > 0xffffffffLL) return false;   // threads of a launch
        }
        a.wg0[LGD_MAX_LEVELS] = (int)w;
        a.act = c.act; a.ptype = c.ptype; a.eps = c.eps; a.gamma = c.gamma; a.beta = c.beta; a.stats = c.stats; a.csum = c.csum;
        return true;
    }
    return false;
}

template <typename T, int VW>
static void slab_fwd_launch(const SlabArgs& a, const SlabPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)a.wg0[LGD_MAX_LEVELS]), block((unsigned)p.NT);
    if constexpr (sizeof(T) == 4) {
        if (p.large) { LGD_LAUNCH("gn_act_slab_kernel", (slab_fwd_kernel<T, VW, kSlabLarge, false>), grid, block, 0, s, a); return; }
    }
    if constexpr (sizeof(T) == 4 || VW < 4) {
        if (p.multi) { LGD_LAUNCH("gn_act_slab_kernel", (slab_fwd_kernel<T, VW, kSlabSmall, true>), grid, block, 0, s, a); return; }
    }
    LGD_LAUNCH("gn_act_slab_kernel", (slab_fwd_kernel<T, VW, kSlabSmall, false>), grid, block, 0, s, a);
}
template <typename T, int VW>
static void slab_bwd_launch(const SlabArgs& a, const SlabPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)a.wg0[LGD_MAX_LEVELS]), block((unsigned)p.NT);
    const size_t Cs = (size_t)a.ng * a.cg, lds = (a.rows * Cs + 2 * Cs + 2 * a.ng) * sizeof(float);   // at most 32 + 8 + 8 KB
    if constexpr (sizeof(T) == 4) {
        if (p.large) { LGD_LAUNCH("gn_act_bwd_slab_kernel", (slab_bwd_kernel<T, VW, kSlabLarge, false>), grid, block, lds, s, a); return; }
    }
    if constexpr (sizeof(T) == 4 || VW < 4) {
        if (p.multi) { LGD_LAUNCH("gn_act_bwd_slab_kernel", (slab_bwd_kernel<T, VW, kSlabSmall, true>), grid, block, lds, s, a); return; }
    }
    LGD_LAUNCH("gn_act_bwd_slab_kernel", (slab_bwd_kernel<T, VW, kSlabSmall, false>), grid, block, lds, s, a);
}
template <typename T> static void slab_fwd_vw(const SlabArgs& a, const SlabPlan& p, hipStream_t s) {
    if (p.VW == 4) slab_fwd_launch<T, 4>(a, p, s); else if (p.VW == 2) slab_fwd_launch<T, 2>(a, p, s); else slab_fwd_launch<T, 1>(a, p, s);
}
template <typename T> static void slab_bwd_vw(const SlabArgs& a, const SlabPlan& p, hipStream_t s) {
    if (p.VW == 4) slab_bwd_launch<T, 4>(a, p, s); else if (p.VW == 2) slab_bwd_launch<T, 2>(a, p, s); else slab_bwd_launch<T, 1>(a, p, s);
}

bool ga_slab_takes(const int32_t* hw, int L, int B, int C, int G, int dtype) {
    SlabArgs a;
    SlabPlan p;
    GaCall c = {};
    c.hw = hw; c.L = L; c.B = B; c.C = C; c.G = G; c.dtype = dtype;
    return slab_plan(a, p, c);
}

bool ga_slab_fwd(const GaCall& c, hipStream_t s) {
    SlabArgs a;
    SlabPlan p;
    if (!slab_plan(a, p, c)) return false;
    if (c.dtype == LGD_F32) slab_fwd_vw<float>(a, p, s);
    else if (c.dtype == LGD_BF16) slab_fwd_vw<__bf16>(a, p, s);
    else slab_fwd_vw<_Float16>(a, p, s);
    return true;
}

bool ga_slab_bwd(const GaCall& c, hipStream_t s) {
    SlabArgs a;
    SlabPlan p;
    if (!slab_plan(a, p, c)) return false;
    if (c.L * c.B == 1) { a.dgamma = c.dgamma; a.dbeta = c.dbeta; }
    if (c.dtype == LGD_F32) slab_bwd_vw<float>(a, p, s);
    else if (c.dtype == LGD_BF16) slab_bwd_vw<__bf16>(a, p, s);
    else slab_bwd_vw<_Float16>(a, p, s);
    return true;
}

}  // namespace lgd
