// Norm over every element of many tensors (fp32 / bf16 / fp16, mixed, any sizes and alignments), and clipping by it in place.
// Memory bound: the norm reads N bytes, clipping reads them twice and writes them (the factor depends on all of them).
// The tensors are cut into chunks, numbered through; workgroup w of a fixed grid takes the chunks w, w + grid, ... (all workgroups sweep the same
// region of memory at a time: 6.1 TB/s against 5.0 - 5.9 for a contiguous run each, 148 - 540 MB) and leaves one partial word, which the next
// kernel's workgroups all reduce for themselves (8 KB out of the L2): two launches, no atomics, the same bits every time.
// Clipping reads plainly the first time, so that what fits stays in the caches for the second read, which streams (non-temporal loads and stores):
// 148 MB 67 us, against 92 us all plain and 75 us all streaming.
// The list travels in the kernel arguments (no host-to-device copy: nothing to wait for, nothing a captured graph could find overwritten); beyond
// kNormInline tensors small kernels store it into the workspace first.
#include "grad_norm.h"

namespace lgd {

constexpr int kNormChunk = 32768;    // bytes.  16 - 32 KB, 1024 - 2048 workgroups, 4 - 8 accesses in flight: within 3 % of each other
constexpr int kNormGrid = 1024;      // workgroups at most: 4 per CU
constexpr int kNormUnroll = 4;       // 16-byte accesses of a thread in flight
constexpr int kNormInline = 160;     // records in the kernel arguments (24 bytes each, under 4 KB)

// Chunks of a list that one workgroup takes alone.  us, one workgroup / two launches, norm: tensors of 1000 2.5 / 4.1 at 2 chunks, 3.6 / 4.5 at 8, 4.4 / 4.4 at
// 12, 5.3 / 4.5 at 16; whole chunks of 8192 fp32 2.9 / 4.4 at 2, 4.8 / 5.0 at 8, 5.0 / 4.8 at 9, 7.7 / 4.8 at 16 (clipping the same within 0.3): the two cross
// at 8 - 12
constexpr int kNormOnce = 8;

struct NormEntry {
    void* p;
    long long n;
    int blk0;        // number of its first chunk
    int dtype;
};
struct NormTable {
    NormEntry e[kNormInline];
    const NormEntry* more;   // the whole table, when it does not fit
    int n, nblk;
};

// the chunks of workgroup `w` of `grid`: f(entry, first element, number of elements)
template <typename F>
__device__ __forceinline__ void norm_walk(const NormTable& t, int w, int grid, F f) {
    const auto finder = tensor_finder<3>([&](int i) { return t.more ? t.more[i].blk0 : t.e[i < kNormInline ? i : 0].blk0; }, 0, t.n);
    for (int c = w; c < t.nblk; c += grid) {
        const int i = finder.find(c);
        const NormEntry e = t.more ? t.more[i] : t.e[i];
        const int per = e.dtype == LGD_F32 ? kNormChunk / 4 : kNormChunk / 2;
        const long long first = (long long)(c - e.blk0) * per;
        f(e, first, (int)(e.n - first < per ? e.n - first : per));
    }
}

__global__ __launch_bounds__(256) void norm_table_kernel(NormTable t, NormEntry* dst) {
    for (int i = threadIdx.x; i < t.n; i += 256) dst[i] = t.e[i];
}

template <int NT, bool STREAM>
__device__ __forceinline__ void norm_entry(const NormEntry& e, long long first, int count, NormAcc<NT>& acc, int t) {
    if (e.dtype == LGD_F32) norm_chunk<NT, float, kNormUnroll, STREAM>(static_cast<const float*>(e.p) + first, count, acc, t);
    else if (e.dtype == LGD_BF16) norm_chunk<NT, __bf16, kNormUnroll, STREAM>(static_cast<const __bf16*>(e.p) + first, count, acc, t);
    else norm_chunk<NT, _Float16, kNormUnroll, STREAM>(static_cast<const _Float16*>(e.p) + first, count, acc, t);
}

template <int NT, bool STREAM>
__global__ __launch_bounds__(256) void norm_partial_kernel(NormTable t, double* part) {
    __shared__ double sh[4];
    NormAcc<NT> acc;
    norm_walk(t, blockIdx.x, gridDim.x, [&](const NormEntry& e, long long first, int count) { norm_entry<NT, STREAM>(e, first, count, acc, threadIdx.x); });
    acc = norm_block<NT>(acc, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = acc.word();
}

template <int NT>
__global__ __launch_bounds__(256) void norm_final_kernel(const double* part, int np, float* out) {
    __shared__ double sh[4];
    const float v = norm_total<NT>(part, np, sh);
    if (threadIdx.x == 0) *out = v;
}

template <typename T, int U>
__device__ __forceinline__ void norm_scale_chunk(T* p, int count, float c, int t) {
    constexpr int V = Vec16<T>::V;
    const int head = norm_head(p, count), nv = (count - head) / V, tail = head + nv * V;
    T* q = p + head;
    for (int i0 = t; i0 < nv; i0 += 256 * U) {
        lgd_u32x4 v[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) if (i0 + u * 256 < nv) v[u] = vec16_load<true>(q + (size_t)(i0 + u * 256) * V);
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * 256 >= nv) continue;
            float f[V];
            Vec16<T>::unpack(v[u], f);
            #pragma unroll
            for (int i = 0; i < V; ++i) f[i] *= c;
            vec16_store<true>(q + (size_t)(i0 + u * 256) * V, Vec16<T>::pack(f));
        }
    }
    if (t < head) glob_store(p + t, (T)((float)glob_load(p + t) * c));
    if (t < count - tail) glob_store(p + tail + t, (T)((float)glob_load(p + tail + t) * c));
}

__device__ __forceinline__ void scale_entry(const NormEntry& e, long long first, int count, float c, int t) {
    if (e.dtype == LGD_F32) norm_scale_chunk<float, kNormUnroll>(static_cast<float*>(e.p) + first, count, c, t);
    else if (e.dtype == LGD_BF16) norm_scale_chunk<__bf16, kNormUnroll>(static_cast<__bf16*>(e.p) + first, count, c, t);
    else norm_scale_chunk<_Float16, kNormUnroll>(static_cast<_Float16*>(e.p) + first, count, c, t);
}

template <int NT>
__global__ __launch_bounds__(256) void norm_scale_kernel(NormTable t, const double* part, int np, float max_norm, float* out) {
    __shared__ double sh[4];
    const float norm = norm_total<NT>(part, np, sh), c = norm_coef(norm, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) *out = norm;
    if (c == 1.f) return;
    norm_walk(t, blockIdx.x, gridDim.x, [&](const NormEntry& e, long long first, int count) { scale_entry(e, first, count, c, threadIdx.x); });
}

// a list of at most kNormOnce chunks: everything in one workgroup of four teams of 256, one launch
template <int NT, bool CLIP>
__global__ __launch_bounds__(1024) void norm_once_kernel(NormTable t, float max_norm, float* out) {
    __shared__ double sh[16];
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), tid = threadIdx.x & 255;
    NormAcc<NT> acc;
    norm_walk(t, team, 4, [&](const NormEntry& e, long long first, int count) { norm_entry<NT, false>(e, first, count, acc, tid); });
    const float norm = norm_block<NT, 16>(acc, sh).value();
    if (threadIdx.x == 0) *out = norm;
    if (!CLIP) return;
    const float c = norm_coef(norm, max_norm);
    if (c == 1.f) return;
    norm_walk(t, team, 4, [&](const NormEntry& e, long long first, int count) { scale_entry(e, first, count, c, tid); });
}

static size_t norm_ws_part() { return (size_t)kNormGrid * sizeof(double); }

// host list -> table (empty tensors dropped); LGD_EINVAL where a record is unusable.  *grid = workgroups
static int norm_table(NormTable& t, const lgd_grad_tensor* host, int n, void* ws, hipStream_t s, int* grid) {
    NormEntry* dev = reinterpret_cast<NormEntry*>(static_cast<char*>(ws) + norm_ws_part());
    int live = 0;
    for (int i = 0; i < n; ++i) {
        const lgd_grad_tensor& h = host[i];
        if (h.n < 0 || h.dtype < 0 || h.dtype > 2 || (h.n > 0 && (!h.p || reinterpret_cast<uintptr_t>(h.p) % (h.dtype == LGD_F32 ? 4 : 2)))) return LGD_EINVAL;
        live += h.n > 0;
    }
    t.n = 0; t.more = nullptr;
    long long blk = 0;
    int done = 0;
    for (int i = 0; i < n; ++i) {
        const lgd_grad_tensor& h = host[i];
        if (h.n == 0) continue;
        const int per = h.dtype == LGD_F32 ? kNormChunk / 4 : kNormChunk / 2;
        NormEntry& e = t.e[t.n++];
        e.p = h.p; e.n = h.n; e.blk0 = (int)blk; e.dtype = h.dtype;
        blk += (h.n + per - 1) / per;
        if (blk > 0x3fffffffLL) return LGD_EINVAL;
        if (live > kNormInline && (t.n == kNormInline || done + t.n == live)) {
            LGD_LAUNCH("grad_norm_table_kernel", norm_table_kernel, dim3(1), dim3(256), 0, s, t, dev + done);
            done += t.n; t.n = 0;
        }
    }
    if (live > kNormInline) t.more = dev;
    t.n = live; t.nblk = (int)blk;
    *grid = blk < kNormGrid ? (blk < 1 ? 1 : (int)blk) : kNormGrid;
    return LGD_OK;
}

template <int NT>
static int norm_run(const NormTable& t, int grid, bool clip, float max_norm, void* ws, float* out, hipStream_t s) {
    double* part = static_cast<double*>(ws);
    if (t.nblk <= kNormOnce && !t.more) {
        if (clip) LGD_LAUNCH("grad_clip_kernel", (norm_once_kernel<NT, true>), dim3(1), dim3(1024), 0, s, t, max_norm, out);
        else LGD_LAUNCH("grad_norm_kernel", (norm_once_kernel<NT, false>), dim3(1), dim3(1024), 0, s, t, max_norm, out);
        return check_launch();
    }
    if (clip) LGD_LAUNCH("grad_norm_kernel", (norm_partial_kernel<NT, false>), dim3((unsigned)grid), dim3(256), 0, s, t, part);
    else LGD_LAUNCH("grad_norm_kernel", (norm_partial_kernel<NT, true>), dim3((unsigned)grid), dim3(256), 0, s, t, part);
    if (clip) LGD_LAUNCH("grad_clip_kernel", norm_scale_kernel<NT>, dim3((unsigned)grid), dim3(256), 0, s, t, part, grid, max_norm, out);
    else LGD_LAUNCH("grad_norm_final_kernel", norm_final_kernel<NT>, dim3(1), dim3(256), 0, s, part, grid, out);
    return check_launch();
}

static int norm_call(const lgd_grad_tensor* host, int n, int norm_type, bool clip, float max_norm, void* ws, float* out, void* stream) {
    if (n < 0 || (n > 0 && !host) || norm_type < 0 || norm_type > 2 || !ws || !out || !(max_norm >= 0.f)) return LGD_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    NormTable t;
    int grid = 0;
    const int rc = norm_table(t, host, n, ws, s, &grid);
    if (rc != LGD_OK) return rc;
    if (norm_type == LGD_NORM_2) return norm_run<LGD_NORM_2>(t, grid, clip, max_norm, ws, out, s);
    if (norm_type == LGD_NORM_1) return norm_run<LGD_NORM_1>(t, grid, clip, max_norm, ws, out, s);
    return norm_run<LGD_NORM_INF>(t, grid, clip, max_norm, ws, out, s);
}

}  // namespace lgd

extern "C" {

size_t lgd_grad_norm_ws_bytes(int n_tensors) {
    return lgd::norm_ws_part() + (n_tensors > lgd::kNormInline ? (size_t)n_tensors * sizeof(lgd::NormEntry) : 0);
}

int lgd_grad_norm(const lgd_grad_tensor* tensors_host, int n_tensors, int norm_type, void* ws, float* norm_out, void* stream) {
    return lgd::norm_call(tensors_host, n_tensors, norm_type, false, 0.f, ws, norm_out, stream);
}

int lgd_grad_clip(const lgd_grad_tensor* tensors_host, int n_tensors, int norm_type, float max_norm, void* ws, float* norm_out, void* stream) {
    return lgd::norm_call(tensors_host, n_tensors, norm_type, true, max_norm, ws, norm_out, stream);
}

}  // extern "C"
