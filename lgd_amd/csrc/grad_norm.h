// Device pieces of a norm over many tensors, shared by grad_norm.hip (any list) and optim.hip (the fused SGD step's table).
//   2: sqrt(sum g^2)   1: sum |g|   inf: max |g|
// Sums are fp64 from the first element on (cvt + FMA per element, at the rate of unpacked fp32 on gfx950): the square of any fp32 value neither
// over- nor underflows there, and 10^9 terms lose nothing that fp32 could show.  The maximum runs on the bits of |g| as fp32: unsigned order is the
// order of non-negative floats, and every NaN is above infinity, so a NaN wins.  A partial result is one 8-byte word per workgroup.
#pragma once
#include "vec16.h"

namespace lgd {

template <int NT> struct NormAcc;   // NT: LGD_NORM_*
template <int NT> struct NormAcc {
    double s = 0.0;
    __device__ __forceinline__ void add(float v) { const double d = v; if (NT == LGD_NORM_2) s = fma(d, d, s); else s += __builtin_fabs(d); }
    __device__ __forceinline__ void join(const NormAcc& o) { s += o.s; }
    __device__ __forceinline__ void wave() { s = wave_sum(s); }
    __device__ __forceinline__ double word() const { return s; }
    static __device__ __forceinline__ NormAcc from(double w) { NormAcc a; a.s = w; return a; }
    __device__ __forceinline__ float value() const { return (float)(NT == LGD_NORM_2 ? sqrt(s) : s); }
};
template <> struct NormAcc<LGD_NORM_INF> {
    uint32_t m = 0;
    __device__ __forceinline__ void add(float v) { m = max(m, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu); }
    __device__ __forceinline__ void join(const NormAcc& o) { m = max(m, o.m); }
    __device__ __forceinline__ void wave() { for (int o = 1; o < 64; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o)); }
    __device__ __forceinline__ double word() const { return __builtin_bit_cast(double, (unsigned long long)m); }
    static __device__ __forceinline__ NormAcc from(double w) { NormAcc a; a.m = (uint32_t)__builtin_bit_cast(unsigned long long, w); return a; }
    __device__ __forceinline__ float value() const { return __builtin_bit_cast(float, m); }
};

// elements in front of the first 16-byte boundary (at most count)
template <typename T> __device__ __forceinline__ int norm_head(const T* p, int count) {
    const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    return h < count ? h : count;
}

// `count` contiguous elements by 256 threads (t: 0 .. 255): 16-byte loads between an unaligned head and tail, U of them in flight
template <int NT, typename T, int U, bool STREAM>
__device__ __forceinline__ void norm_chunk(const T* __restrict__ p, int count, NormAcc<NT>& acc, int t) {
    constexpr int V = Vec16<T>::V;
    const int head = norm_head(p, count), nv = (count - head) / V, tail = head + nv * V;
    const T* q = p + head;
    for (int i0 = t; i0 < nv; i0 += 256 * U) {
        lgd_u32x4 v[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) v[u] = i0 + u * 256 < nv ? vec16_load<STREAM>(q + (size_t)(i0 + u * 256) * V) : (lgd_u32x4){0, 0, 0, 0};   // zeros add nothing to any of the norms
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
            Vec16<T>::unpack(v[u], f);
            #pragma unroll
            for (int i = 0; i < V; ++i) acc.add(f[i]);
        }
    }
    if (t < head) acc.add((float)glob_load(p + t));
    if (t < count - tail) acc.add((float)glob_load(p + tail + t));
}

// Which tensor holds block c: the last one whose first block is not behind c.  Every lane holds the first blocks of its tensors (lane, lane + 64, ...:
// ascending), a ballot counts them -- one load latency per kernel instead of a chain of dependent ones per block; lists longer than 64 K load the rest.
template <int K, typename First>
struct TensorFinder {
    First first;   // first(i): first block of tensor i
    int lo, n, b0[K];
    __device__ __forceinline__ TensorFinder(First f, int lo_, int hi) : first(f), lo(lo_), n(hi - lo_) {
        const int lane = threadIdx.x & 63;
        #pragma unroll
        for (int k = 0; k < K; ++k) b0[k] = k * 64 + lane < n ? first(lo + k * 64 + lane) : 0x7fffffff;
    }
    __device__ __forceinline__ int find(int c) const {
        int i = lo - 1;
        #pragma unroll
        for (int k = 0; k < K; ++k) i += __popcll(__ballot(b0[k] <= c));
        for (int k = K; k * 64 < n; ++k) {
            const int j = k * 64 + (int)(threadIdx.x & 63);
            i += __popcll(__ballot((j < n ? first(lo + j) : 0x7fffffff) <= c));
        }
        return __builtin_amdgcn_readfirstlane(i);
    }
};
template <int K, typename First> __device__ __forceinline__ TensorFinder<K, First> tensor_finder(First f, int lo, int hi) { return TensorFinder<K, First>(f, lo, hi); }

// the workgroup's accumulators as one, in every thread (sh: a word per wave; barriers inside)
template <int NT, int WAVES = 4>
__device__ __forceinline__ NormAcc<NT> norm_block(NormAcc<NT> acc, double* sh) {
    acc.wave();
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = acc.word();
    __syncthreads();
    acc = NormAcc<NT>::from(sh[0]);
    for (int i = 1; i < WAVES; ++i) acc.join(NormAcc<NT>::from(sh[i]));
    return acc;
}

// n partial words -> the norm, in every thread of the workgroup; the order is fixed, so every workgroup finds the same bits
template <int NT>
__device__ __forceinline__ float norm_total(const double* __restrict__ part, int n, double* sh) {
    NormAcc<NT> acc;
    for (int i = threadIdx.x; i < n; i += 256) acc.join(NormAcc<NT>::from(part[i]));
    return norm_block<NT>(acc, sh).value();
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN
__device__ __forceinline__ float norm_coef(float norm, float max_norm) {
    const double c = (double)max_norm / ((double)norm + 1e-6);
    return (float)(c >= 1.0 ? 1.0 : c);
}

}  // namespace lgd
