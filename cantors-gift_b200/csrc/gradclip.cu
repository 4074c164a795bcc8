// gradclip.cu - the global norm of a list of gradient tensors, and clipping by it.
//
// The reference has no such operator; its reductions take one tensor (src/ir/ops.cpp:417-436).
//   norm   = sqrt(sum over all tensors and elements of g^2)
//   factor = min(1, max_norm / (norm + 1e-6)),  out = g * factor
//
// HBM-bound: the list is read for the norm and again for the scaling, which cannot begin before the norm is known, and written once.
// The tensors' addresses, lengths and types travel by value in the kernel's parameters, so nothing is copied to the device first and
// nothing is kept between calls. Each tensor is cut into chunks of 16384 elements and the CTAs walk the chunks of all tensors
// gridDim.x apart; squares are added in fp32 per 16-byte packet and in fp64 beyond it, and every CTA leaves one fp64 sum in the
// workspace. The scaling kernel's CTAs each add those sums up in the same fixed order, so the norm does not depend on timing, and walk
// the chunks backwards: what the norm pass read last is still in L2.
#include <float.h>

#include "common.cuh"

namespace cgb {

constexpr int kClipTensors = 448;       // per launch: the table stays under the kernel parameter limit
constexpr int kClipChunk = 16384;
constexpr int kClipThreads = 256;

struct ClipEntry {
    const void* in;
    void* out;
    long long n;
    long long first_chunk;   // of this launch
    int32_t dtype, out_dtype;
};
struct ClipTable {
    ClipEntry e[kClipTensors];
    double* part;            // this launch's CTAs' sums
    const double* all_parts;
    float* norm;
    long long chunks;
    int count, n_parts;
    float max_norm;
};

__device__ __forceinline__ int clip_find(const ClipTable& t, long long chunk) {
    int lo = 0, hi = t.count;   // the last tensor whose first chunk is not behind `chunk`; empty tensors have no chunk of their own
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.e[mid].first_chunk <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Elements of [p, p + n) before the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int clip_head(const T* p, int n) {
    const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
    return h < n ? h : n;
}

// A packet's squares: in fp32, and again in fp64 where fp32 leaves its range (|g| above 1.8e19 or all below 1e-15).
template <typename T>
__device__ __forceinline__ double clip_squares(const Vec16<T>& v) {
    constexpr int L = Vec16<T>::N;
    float f[L], s = 0.0f;
    unpack16<T>(v, f);
#pragma unroll
    for (int l = 0; l < L; ++l) s = fmaf(f[l], f[l], s);
    if (s <= FLT_MAX && s >= 1e-30f) return (double)s;
    double d = 0.0;
#pragma unroll
    for (int l = 0; l < L; ++l) d += (double)f[l] * (double)f[l];
    return d;
}

template <typename T>
__device__ __forceinline__ double clip_chunk_squares(const T* g, int n) {
    constexpr int L = Vec16<T>::N, U = 8;
    const int head = clip_head(g, n), packets = (n - head) / L;
    double sum = 0.0;
    for (int i = threadIdx.x; i < head; i += kClipThreads) sum += (double)Elem<T>::to_f32(g[i]) * (double)Elem<T>::to_f32(g[i]);
    for (int i = head + packets * L + threadIdx.x; i < n; i += kClipThreads) sum += (double)Elem<T>::to_f32(g[i]) * (double)Elem<T>::to_f32(g[i]);
    const T* body = g + head;
    for (int k0 = threadIdx.x; k0 < packets; k0 += kClipThreads * U) {
        Vec16<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * kClipThreads < packets) v[u] = ld_keep(body + (k0 + u * kClipThreads) * L);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * kClipThreads < packets) sum += clip_squares<T>(v[u]);
    }
    return sum;
}

// Sum over the CTA, in every thread
__device__ __forceinline__ double clip_block_sum(double v, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kClipThreads / 32; ++w) s += scratch[w];
    return s;
}

__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipTable t) {
    __shared__ double scratch[kClipThreads / 32];
    double sum = 0.0;
    for (long long chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const ClipEntry& e = t.e[clip_find(t, chunk)];
        const long long at = (chunk - e.first_chunk) * kClipChunk;
        const int n = (int)(e.n - at < kClipChunk ? e.n - at : kClipChunk);
        if (e.dtype == CG_B200_F32) sum += clip_chunk_squares(static_cast<const float*>(e.in) + at, n);
        else if (e.dtype == CG_B200_BF16) sum += clip_chunk_squares(static_cast<const __nv_bfloat16*>(e.in) + at, n);
        else sum += clip_chunk_squares(static_cast<const __half*>(e.in) + at, n);
    }
    sum = clip_block_sum(sum, scratch);
    if (threadIdx.x == 0) t.part[blockIdx.x] = sum;
}

// The norm from all CTAs' sums, the same in every CTA
__device__ __forceinline__ double clip_norm(const double* parts, int n, double* scratch) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += kClipThreads) s += parts[i];
    return sqrt(clip_block_sum(s, scratch));
}

template <typename T, typename O>
__device__ __forceinline__ void clip_chunk_scale(const T* g, O* o, int n, float factor) {
    constexpr int L = Vec16<T>::N, M = Vec16<O>::N, R = L / M, U = 8;
    const int head = clip_head(g, n);
    const bool vec = ((reinterpret_cast<uintptr_t>(o + head)) & 15) == 0;   // both sides reach a boundary at the same element
    const int packets = vec ? (n - head) / L : 0, loose = vec ? head : 0;
    for (int i = threadIdx.x; i < loose; i += kClipThreads) o[i] = Elem<O>::from_f32(Elem<T>::to_f32(g[i]) * factor);
    for (int i = loose + packets * L + threadIdx.x; i < n; i += kClipThreads) o[i] = Elem<O>::from_f32(Elem<T>::to_f32(g[i]) * factor);
    const T* gb = g + head;
    O* ob = o + head;
    for (int k0 = threadIdx.x; k0 < packets; k0 += kClipThreads * U) {
        Vec16<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * kClipThreads < packets) v[u] = ld_stream(gb + (k0 + u * kClipThreads) * L);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * kClipThreads < packets) {
                float f[L];
                unpack16<T>(v[u], f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float q[M];
#pragma unroll
                    for (int i = 0; i < M; ++i) q[i] = f[r * M + i] * factor;
                    st_stream(ob + (k0 + u * kClipThreads) * L + r * M, pack16<O>(q));
                }
            }
    }
}

__global__ void __launch_bounds__(kClipThreads) clip_scale_kernel(const __grid_constant__ ClipTable t) {
    __shared__ double scratch[kClipThreads / 32];
    const double norm = clip_norm(t.all_parts, t.n_parts, scratch);
    if (t.norm && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = (float)norm;
    const double ratio = (double)t.max_norm / (norm + 1e-6);
    const float factor = ratio >= 1.0 ? 1.0f : (float)ratio;   // a norm that is not a number gives such a factor
    for (long long c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const long long chunk = t.chunks - 1 - c;
        const ClipEntry& e = t.e[clip_find(t, chunk)];
        if (e.in == e.out && factor == 1.0f) continue;   // already there
        const long long at = (chunk - e.first_chunk) * kClipChunk;
        const int n = (int)(e.n - at < kClipChunk ? e.n - at : kClipChunk);
        if (e.dtype == CG_B200_F32) {
            clip_chunk_scale(static_cast<const float*>(e.in) + at, static_cast<float*>(e.out) + at, n, factor);
        } else if (e.dtype == CG_B200_BF16) {
            const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(e.in) + at;
            if (e.out_dtype == CG_B200_F32) clip_chunk_scale(g, static_cast<float*>(e.out) + at, n, factor);
            else clip_chunk_scale(g, static_cast<__nv_bfloat16*>(e.out) + at, n, factor);
        } else {
            const __half* g = static_cast<const __half*>(e.in) + at;
            if (e.out_dtype == CG_B200_F32) clip_chunk_scale(g, static_cast<float*>(e.out) + at, n, factor);
            else clip_chunk_scale(g, static_cast<__half*>(e.out) + at, n, factor);
        }
    }
}

__global__ void __launch_bounds__(kClipThreads) clip_norm_only_kernel(const double* parts, int n, float* norm) {
    __shared__ double scratch[kClipThreads / 32];
    const double v = clip_norm(parts, n, scratch);
    if (threadIdx.x == 0) *norm = (float)v;
}

static long long clip_grid_cap() { return (long long)sm_count() * 4; }

static int clip_check(const cg_b200_grad* g, int64_t count, bool scale) {
    if (count < 0 || count > (1 << 20)) return CG_B200_ERR_INVALID_ARG;
    if (count > 0 && !g) return CG_B200_ERR_NULL_POINTER;
    for (int64_t i = 0; i < count; ++i) {
        if (g[i].n < 0 || g[i].n > (int64_t(1) << 48) || !dtype_ok(g[i].dtype)) return CG_B200_ERR_INVALID_ARG;
        if (scale && g[i].out_dtype != g[i].dtype && g[i].out_dtype != CG_B200_F32) return CG_B200_ERR_INVALID_ARG;
        if (g[i].n == 0) continue;
        if (!g[i].in || (scale && !g[i].out)) return CG_B200_ERR_NULL_POINTER;
        if (!aligned_to(g[i].in, dtype_bytes(g[i].dtype))) return CG_B200_ERR_MISALIGNED;
        if (!scale) continue;
        if (!aligned_to(g[i].out, dtype_bytes(g[i].out_dtype))) return CG_B200_ERR_MISALIGNED;
        // in place, or apart: a shifted or widened copy over its own input would read what it has overwritten
        const uintptr_t a = reinterpret_cast<uintptr_t>(g[i].in), b = reinterpret_cast<uintptr_t>(g[i].out);
        const uintptr_t ae = a + (size_t)g[i].n * dtype_bytes(g[i].dtype), be = b + (size_t)g[i].n * dtype_bytes(g[i].out_dtype);
        if (a < be && b < ae && !(a == b && g[i].dtype == g[i].out_dtype)) return CG_B200_ERR_INVALID_ARG;
    }
    return CG_B200_OK;
}

static size_t clip_workspace(int64_t count) {
    const int64_t launches = (count + kClipTensors - 1) / kClipTensors;
    return (size_t)(launches > 0 ? launches : 1) * (size_t)clip_grid_cap() * sizeof(double);
}

// The launches over the list, kClipTensors at a time: sums (scale false) or the scaled copies.
static int clip_run(const cg_b200_grad* g, int64_t count, float max_norm, float* norm, double* ws, bool scale, cudaStream_t s) {
    long long n_parts = 0;
    for (int pass = 0; pass < 2; ++pass) {
        long long at = 0;
        for (int64_t i0 = 0; i0 < count; i0 += kClipTensors) {
            ClipTable t;
            t.count = 0;
            t.chunks = 0;
            for (int64_t i = i0; i < count && i < i0 + kClipTensors; ++i) {
                if (g[i].n == 0) continue;
                ClipEntry& e = t.e[t.count++];
                e.in = g[i].in;
                e.out = g[i].out;
                e.n = g[i].n;
                e.dtype = g[i].dtype;
                e.out_dtype = g[i].out_dtype;
                e.first_chunk = t.chunks;
                t.chunks += (g[i].n + kClipChunk - 1) / kClipChunk;
            }
            if (t.count == 0) continue;
            const long long cap = clip_grid_cap();
            const unsigned grid = (unsigned)(t.chunks < cap ? t.chunks : cap);
            t.part = ws + at;
            t.all_parts = ws;
            t.n_parts = (int)n_parts;
            t.norm = at == 0 ? norm : nullptr;
            t.max_norm = max_norm;
            if (pass == 0) clip_norm_kernel<<<grid, kClipThreads, 0, s>>>(t);
            else clip_scale_kernel<<<grid, kClipThreads, 0, s>>>(t);
            CGB_CUDA(cudaGetLastError());
            at += grid;
        }
        if (pass == 0) {
            n_parts = at;
            if (!scale || n_parts == 0) {
                clip_norm_only_kernel<<<1, kClipThreads, 0, s>>>(ws, (int)n_parts, norm);
                CGB_CUDA(cudaGetLastError());
                return CG_B200_OK;
            }
        }
    }
    return CG_B200_OK;
}

static int clip_entry(const cg_b200_grad* grads, int64_t count, float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                      bool scale, void* stream) {
    int st = clip_check(grads, count, scale);
    if (st) return st;
    if (!norm) return CG_B200_ERR_NULL_POINTER;
    if (!aligned_to(norm, 4) || !aligned_to(workspace, 16)) return CG_B200_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < clip_workspace(count)) return CG_B200_ERR_WORKSPACE;
    st = require_sm100();
    if (st) return st;
    return clip_run(grads, count, max_norm, norm, static_cast<double*>(workspace), scale, (cudaStream_t)stream);
}

}  // namespace cgb

extern "C" int cg_b200_grad_norm_workspace_bytes(int64_t count, size_t* bytes) {
    if (!bytes) return CG_B200_ERR_NULL_POINTER;
    *bytes = 0;
    if (count < 0 || count > (1 << 20)) return CG_B200_ERR_INVALID_ARG;
    *bytes = cgb::clip_workspace(count);
    return CG_B200_OK;
}

extern "C" int cg_b200_grad_norm(const cg_b200_grad* host_grads, int64_t count, float* norm, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    return cgb::clip_entry(host_grads, count, 0.0f, norm, workspace, workspace_bytes, false, stream);
}

extern "C" int cg_b200_clip_grad_norm(const cg_b200_grad* host_grads, int64_t count, float max_norm, float* norm, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (!(max_norm >= 0.0f)) return CG_B200_ERR_INVALID_ARG;
    return cgb::clip_entry(host_grads, count, max_norm, norm, workspace, workspace_bytes, true, stream);
}
