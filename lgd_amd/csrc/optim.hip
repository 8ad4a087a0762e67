// Gradient clipping + SGD(momentum, weight decay) of BOTH optimizers of the distillation step as ONE launch over a table of
// tensors [ref: train.py:200-204 -- stu_optimizer.step(); tea_optimizer.step() after detectron2's per-parameter gradient
// clipping (utils/build.py:514-529 maybe_add_gradient_clipping, CLIP_TYPE "value") and utils/build.py:494-512 torch.optim.SGD].
// torch's multi-tensor path runs clamp_min, clamp_max, g + wd p, mu buf, buf + g, p - lr buf as six passes per optimizer (13 tensor
// transfers per parameter element, ~40 launches) behind ~1.7 ms of Python per step (tensor grouping); at 2 images per GPU the GPU
// ran dry for 0.7 ms at the optimizer entry (tools/gap_profile.sh).  Here: one pass (read p, g, buf; write p, g, buf), one launch,
// the table is three device pointers + length + (lr, wd, mu) per tensor.
//   g   <- clamp(g, -clip, clip)            (written back: the clipped gradient is what a caller sees after the step)
//   d   <- g + wd p
//   buf <- mu buf + d                       (a zero-initialised buffer reproduces torch's first step, buf = d, exactly)
//   p   <- p - lr buf
// or, clipping by NORM (lgd_sgd_norm_step): the gradients of every optimizer are one vector, g <- c g with c = min(1, max_norm / (norm + 1e-6)) of that
// optimizer's norm; one launch more: partial sums over the same table (reads g once more), which every workgroup of the update joins for itself while its own loads
// are on their way.
#include "grad_norm.h"

#pragma clang fp contract(off)   // mu * buf + d keeps torch's two roundings (mul_ then add_); the fma calls below are explicit

namespace lgd {

constexpr int kSgdChunk = 4096;  // elements per workgroup: 256 threads x 4 float4

// 4 floats at a 4-byte-aligned address: under DistributedDataParallel(gradient_as_bucket_view=True) a gradient is a view into a flat
// bucket at the sum of the preceding parameters' sizes (train.py:279-281), i.e. dword- but not 16-byte-aligned as soon as one of them
// has a size that is not a multiple of 4 (FCOS `scales`, the centerness bias).  gfx950 runs global memory in unaligned access mode, so
// the accesses stay dwordx4 (the compiler emits them for this type).
typedef float sgd_f4u __attribute__((ext_vector_type(4), aligned(4)));

// Global accesses (the pointers come out of a table: generic to the compiler otherwise).  Loads stream past the caches; stores do (ST) where the gradients have
// just been read for their norm, and are plain in the step by value.  37 M parameters, us:
//   by norm, alone: 167; 198 - 205 with plain loads, plain stores or both
//   by value, behind a backward in training: 179; 190 with plain loads, 187 with plain loads and streaming stores, 213 with both streaming
typedef __attribute__((address_space(1))) const sgd_f4u* sgd_gptr;
typedef __attribute__((address_space(1))) sgd_f4u* sgd_gptr_rw;
typedef __attribute__((address_space(1))) const lgd_vf4* sgd_gptr4;
typedef __attribute__((address_space(1))) lgd_vf4* sgd_gptr4_rw;
__device__ __forceinline__ float4 sgd_load4(const float* p) { const lgd_vf4 v = __builtin_nontemporal_load((sgd_gptr4)p); return make_float4(v.x, v.y, v.z, v.w); }
__device__ __forceinline__ sgd_f4u sgd_loadu(const float* p) { return __builtin_nontemporal_load((sgd_gptr)p); }
template <bool ST> __device__ __forceinline__ void sgd_store4(float* p, const float4& f) {
    const lgd_vf4 v = {f.x, f.y, f.z, f.w};
    if constexpr (ST) __builtin_nontemporal_store(v, (sgd_gptr4_rw)p);
    else *(sgd_gptr4_rw)p = v;
}
template <bool ST> __device__ __forceinline__ void sgd_storeu(float* p, const sgd_f4u& v) {
    if constexpr (ST) __builtin_nontemporal_store(v, (sgd_gptr_rw)p);
    else *(sgd_gptr_rw)p = v;
}

// by value: the clamped gradient, NaN stays NaN (as torch.clamp); by norm: `clip` is the optimizer's factor
template <bool NORM> __device__ __forceinline__ float sgd_clipped(float g, float clip) {
    if (NORM) return g * clip;
    return g < -clip ? -clip : (g > clip ? clip : g);
}

// clip_of(): the clamp's bound, or (NORM) the optimizer's factor; all threads call it once, behind the vector loads
template <bool VEC, bool NORM, typename Clip>
__device__ __forceinline__ void sgd_chunk(const lgd_sgd_tensor& t, long long base, Clip clip_of) {
    float clip;
    const float lr = t.lr, wd = t.wd, mu = t.mu;
    if constexpr (VEC) {
        float4 p[4], g[4], m[4];
        bool on[4];
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long i = base + (long long)(k * 256 + threadIdx.x) * 4;
            on[k] = i + 3 < t.n;
            if (on[k]) {
                p[k] = sgd_load4(t.p + i); m[k] = sgd_load4(t.m + i);
                const sgd_f4u gv = sgd_loadu(t.g + i);
                g[k] = make_float4(gv.x, gv.y, gv.z, gv.w);
            }
        }
        clip = clip_of();
        const bool write_g = !NORM || clip != 1.f;   // a factor of 1 leaves the gradients as they are
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!on[k]) continue;
            const long long i = base + (long long)(k * 256 + threadIdx.x) * 4;
            float* pp = &p[k].x; float* gg = &g[k].x; float* mm = &m[k].x;
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float c = sgd_clipped<NORM>(gg[j], clip);
                const float d = __builtin_fmaf(wd, pp[j], c);
                const float b = mu * mm[j] + d;
                gg[j] = c; mm[j] = b; pp[j] = __builtin_fmaf(-lr, b, pp[j]);
            }
            sgd_store4<NORM>(t.p + i, p[k]);
            sgd_f4u go; go.x = g[k].x; go.y = g[k].y; go.z = g[k].z; go.w = g[k].w;
            if (write_g) sgd_storeu<NORM>(t.g + i, go);
            sgd_store4<NORM>(t.m + i, m[k]);
        }
    } else {
        clip = clip_of();
    }
    const bool write_g = !NORM || clip != 1.f;
    // scalar path: parameters / momentum buffers that are not 16-byte aligned (never torch's own allocations), and the < 4-element
    // tail of a vector chunk
    const long long end = base + kSgdChunk < t.n ? base + kSgdChunk : t.n;
    long long i0 = base;
    if constexpr (VEC) i0 = end == t.n ? (t.n & ~3LL) : end;   // only the last chunk has a tail
    for (long long i = i0 + threadIdx.x; i < end; i += 256) {
        const float c = sgd_clipped<NORM>(t.g[i], clip);
        const float d = __builtin_fmaf(wd, t.p[i], c);
        const float b = mu * t.m[i] + d;
        if (write_g) t.g[i] = c;
        t.m[i] = b; t.p[i] = __builtin_fmaf(-lr, b, t.p[i]);
    }
}

// where a kernel finds the table: in device memory, or, up to LGD_SGD_INLINE tensors (4 KB of arguments), in its own arguments: without the upload a step
// over 10 tensors takes 14 us in place of 22 (the host's time; the two kernels 8.5)
struct SgdTable {
    const lgd_sgd_tensor* e;
    const int32_t* blk;
};
struct SgdInline {
    lgd_sgd_tensor e[LGD_SGD_INLINE];
    int32_t blk[LGD_SGD_INLINE + 1];
};

// the tensor of a block: last i in [lo, hi) with blk[i] <= c (wave-uniform: scalar loads)
template <typename Table>
__device__ __forceinline__ int sgd_tensor_of(const Table& tab, int lo, int hi, int c) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.blk[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

constexpr int kSgdNormGrid = 512;   // workgroups per optimizer: one partial word each
struct SgdGroups {
    int tensor[LGD_MAX_SGD_GROUPS + 1];   // borders in the table
    int blk[LGD_MAX_SGD_GROUPS + 1];      // and in its blocks
    int n;
};

__device__ __forceinline__ bool sgd_vec(const lgd_sgd_tensor& t) {
    return ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.m)) & 15) == 0 && (reinterpret_cast<uintptr_t>(t.g) & 3) == 0;
}

__global__ __launch_bounds__(256) void sgd_clip_kernel(SgdTable tab, int nt, float clip) {
    const int lo = sgd_tensor_of(tab, 0, nt, (int)blockIdx.x);
    const lgd_sgd_tensor t = tab.e[lo];
    const long long base = (long long)((int)blockIdx.x - tab.blk[lo]) * kSgdChunk;
    if (base >= t.n) return;
    if (sgd_vec(t)) sgd_chunk<true, false>(t, base, [&] { return clip; });
    else sgd_chunk<false, false>(t, base, [&] { return clip; });
}

// the update with the gradients clipped by their optimizer's norm, of which `part` holds kSgdNormGrid partial words per group
template <int NT, typename Table>
__global__ __launch_bounds__(256) void sgd_norm_step_kernel(Table tab, SgdGroups g, const double* __restrict__ part, float max_norm,
                                                             float* __restrict__ norms) {
    __shared__ double sh[4];
    if (blockIdx.x == 0 && (int)threadIdx.x < g.n && g.blk[threadIdx.x] == g.blk[threadIdx.x + 1]) norms[threadIdx.x] = 0.f;   // groups without an element
    if ((int)blockIdx.x >= g.blk[g.n]) return;
    const int lo = sgd_tensor_of(tab, 0, g.tensor[g.n], (int)blockIdx.x);
    const lgd_sgd_tensor t = tab.e[lo];
    const long long base = (long long)((int)blockIdx.x - tab.blk[lo]) * kSgdChunk;
    const auto factor = [&] {
        const int k = t.reserved;
        const float v = norm_total<NT>(part + (size_t)k * kSgdNormGrid, kSgdNormGrid, sh);
        if ((int)blockIdx.x == g.blk[k] && threadIdx.x == 0) norms[k] = v;
        return norm_coef(v, max_norm);
    };
    if (sgd_vec(t)) sgd_chunk<true, true>(t, base, factor);
    else sgd_chunk<false, true>(t, base, factor);
}

// partial norms of the gradients of group blockIdx.y; its workgroups sweep the group's blocks side by side.  Plain loads: what fits stays in the caches
// for the update's read
template <int NT, typename Table>
__global__ __launch_bounds__(256) void sgd_norm_kernel(Table tab, SgdGroups g, double* __restrict__ part) {
    __shared__ double sh[4];
    const int k = blockIdx.y;
    NormAcc<NT> acc;
    const auto finder = tensor_finder<6>([&](int i) { return (int)tab.blk[i]; }, g.tensor[k], g.tensor[k + 1]);
    for (int c = g.blk[k] + (int)blockIdx.x; c < g.blk[k + 1]; c += kSgdNormGrid) {
        const int i = finder.find(c);
        const long long first = (long long)(c - tab.blk[i]) * kSgdChunk, left = tab.e[i].n - first;
        norm_chunk<NT, float, 4, false>(tab.e[i].g + first, (int)(left < kSgdChunk ? left : kSgdChunk), acc, threadIdx.x);
    }
    acc = norm_block<NT>(acc, sh);
    if (threadIdx.x == 0) part[k * kSgdNormGrid + blockIdx.x] = acc.word();
}

template <int NT, typename Table>
static int sgd_norm_run(const Table& tab, const SgdGroups& g, float max_norm, void* ws, float* norms, hipStream_t s) {
    double* part = static_cast<double*>(ws);
    const int n_blocks = g.blk[g.n];
    LGD_LAUNCH("sgd_norm_kernel", (sgd_norm_kernel<NT, Table>), dim3(kSgdNormGrid, (unsigned)g.n), dim3(256), 0, s, tab, g, part);
    LGD_LAUNCH("sgd_norm_step_kernel", (sgd_norm_step_kernel<NT, Table>), dim3(n_blocks < 1 ? 1u : (unsigned)n_blocks), dim3(256), 0, s, tab, g,
               (const double*)part, max_norm, norms);
    return check_launch();
}

template <typename Table>
static int sgd_norm_call(const Table& tab, int n_tensors, int n_blocks, const int32_t* group_off_host, const int32_t* group_blk_host, int n_groups,
                         int norm_type, float max_norm, void* ws, float* norms_out, hipStream_t s) {
    if (n_tensors < 1 || n_blocks < 0 || !group_off_host || !group_blk_host || n_groups < 1 || n_groups > LGD_MAX_SGD_GROUPS || !(max_norm >= 0.f) || !ws ||
        !norms_out)
        return LGD_EINVAL;
    SgdGroups g = {};
    g.n = n_groups;
    for (int k = 0; k <= n_groups; ++k) {
        g.tensor[k] = group_off_host[k]; g.blk[k] = group_blk_host[k];
        if (k > 0 && (g.tensor[k] < g.tensor[k - 1] || g.blk[k] < g.blk[k - 1] || (g.tensor[k] == g.tensor[k - 1] && g.blk[k] != g.blk[k - 1]))) return LGD_EINVAL;
    }
    if (g.tensor[0] != 0 || g.blk[0] != 0 || g.tensor[n_groups] != n_tensors || g.blk[n_groups] != n_blocks) return LGD_EINVAL;
    if (norm_type == LGD_NORM_2) return sgd_norm_run<LGD_NORM_2>(tab, g, max_norm, ws, norms_out, s);
    if (norm_type == LGD_NORM_1) return sgd_norm_run<LGD_NORM_1>(tab, g, max_norm, ws, norms_out, s);
    if (norm_type == LGD_NORM_INF) return sgd_norm_run<LGD_NORM_INF>(tab, g, max_norm, ws, norms_out, s);
    return LGD_EINVAL;
}

}  // namespace lgd

extern "C" {

int lgd_sgd_chunk_elems(void) { return lgd::kSgdChunk; }

int lgd_sgd_clip_step(const lgd_sgd_tensor* table, const int32_t* blk_off, int n_tensors, int n_blocks, float clip_value, void* stream) {
    if (!table || !blk_off || n_tensors < 1 || n_blocks < 1 || !(clip_value > 0.f)) return LGD_EINVAL;
    LGD_LAUNCH("sgd_clip_kernel", lgd::sgd_clip_kernel, dim3((unsigned)n_blocks), dim3(256), 0, (hipStream_t)stream, (lgd::SgdTable{table, blk_off}), n_tensors,
               clip_value);
    return lgd::check_launch();
}

size_t lgd_sgd_norm_ws_bytes(int n_groups) {
    return n_groups < 1 ? 0 : (size_t)n_groups * lgd::kSgdNormGrid * sizeof(double);
}

int lgd_sgd_norm_step(const lgd_sgd_tensor* table, const int32_t* blk_off, int n_tensors, int n_blocks, const int32_t* group_off_host,
                      const int32_t* group_blk_host, int n_groups, int norm_type, float max_norm, void* ws, float* norms_out, void* stream) {
    if (!table || !blk_off) return LGD_EINVAL;
    return lgd::sgd_norm_call(lgd::SgdTable{table, blk_off}, n_tensors, n_blocks, group_off_host, group_blk_host, n_groups, norm_type, max_norm, ws, norms_out,
                              (hipStream_t)stream);
}

int lgd_sgd_norm_step_host(const lgd_sgd_tensor* table_host, const int32_t* blk_off_host, int n_tensors, int n_blocks, const int32_t* group_off_host,
                           const int32_t* group_blk_host, int n_groups, int norm_type, float max_norm, void* ws, float* norms_out, void* stream) {
    if (!table_host || !blk_off_host || n_tensors < 1 || n_tensors > LGD_SGD_INLINE) return LGD_EINVAL;
    lgd::SgdInline t = {};
    for (int i = 0; i < n_tensors; ++i) t.e[i] = table_host[i];
    for (int i = 0; i <= n_tensors; ++i) t.blk[i] = blk_off_host[i];
    return lgd::sgd_norm_call(t, n_tensors, n_blocks, group_off_host, group_blk_host, n_groups, norm_type, max_norm, ws, norms_out, (hipStream_t)stream);
}

}  // extern "C"
