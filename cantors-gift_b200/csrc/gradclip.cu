// gradclip.cu - the global norm of a list of gradient tensors, and clipping by it.
//
// The reference has no such operator; its reductions take one tensor (src/ir/ops.cpp:417-436).
//   norm   = sqrt(sum over all tensors and elements of g^2)
//   factor = min(1, max_norm / (norm + 1e-6)),  out = g * factor
//
// HBM-bound: the list is read for the norm and again for the scaling, which cannot begin before the norm is known, and written once
// (113M gradients, bf16 into fp32: 907 MB in 162 us, 85 % of the copy rate).
// The tensors' addresses, lengths and types travel by value in the kernel's parameters, so nothing is copied to the device first and
// nothing is kept between calls. The list is cut into as many equal pieces as there are CTAs; squares are added in fp32 per 16-byte packet
// and in fp64 beyond it, and every CTA leaves one fp64 sum in the workspace. The scaling kernel's CTAs each add those sums up in the same
// fixed order, so the norm does not depend on timing, and walk their pieces backwards, from what the norm pass read last: 161.3 us, forwards
// 163.4. A list of more than 448 tensors takes a launch of each pass for every 448, and every scaling launch adds up the sums of all norm
// launches: 2000 tensors of 64 elements take 0.8 ms, 20000 7.9 ms, most of it the host's table.
#include <float.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace cgb {

// The table of a launch, in the kernel's parameters: a short one for short lists (a launch costs 2.5 us with 40 tensors' worth of
// parameters and 5 us with 400), a long one of 17.9 KB for the others. (32764 bytes of parameters would hold 800; not measured.)
constexpr int kClipShort = 64, kClipLong = 448;
constexpr int kClipChunk = 2048;   // elements; what a CTA takes is a run of chunks
// Many threads with two requests each: 56 us for 34M bf16 gradients into fp32, against 57 with four requests and half the threads and 59
// with eight and three eighths.
constexpr int kClipThreads = 256, kClipCtas = 8;   // of a CTA; CTAs of an SM

struct ClipEntry {
    const void* in;
    void* out;
    long long n;
    long long first_chunk;   // of this launch
    int32_t dtype, out_dtype;
};
template <int N>
struct ClipTable {
    ClipEntry e[N];
    double* part;            // this launch's CTAs' sums
    const double* all_parts;
    float* norm;
    long long chunks;
    int count, n_parts;
    float max_norm;
};

template <int N>
__device__ __forceinline__ int clip_find(const ClipTable<N>& t, long long chunk) {
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
__device__ __forceinline__ long long clip_head(const T* p, long long n) {
    const long long h = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
    return h < n ? h : n;
}

// The chunks of this CTA: an equal share of the list, in one piece
template <int N>
__device__ __forceinline__ void clip_share(const ClipTable<N>& t, long long& from, long long& to) {
    const long long each = t.chunks / gridDim.x, more = t.chunks % gridDim.x, b = blockIdx.x;
    from = b * each + (b < more ? b : more);
    to = from + each + (b < more ? 1 : 0);
}

// A packet's squares: in fp32, and again in fp64 where fp32 leaves its range (|g| above 1.8e19 or all below 1e-15, zeros among them: the
// norm of a bf16 table of 100000 x 1024 with one row in 50 that is not zero takes 40.6 us, of a dense one 37.8; in fp32 66.5 either way).
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
__device__ __forceinline__ double clip_run_squares(const T* g, long long n) {
    constexpr int L = Vec16<T>::N, U = 2;
    const long long head = clip_head(g, n), packets = (n - head) / L;
    double sum = 0.0;
    for (long long i = threadIdx.x; i < head; i += kClipThreads) sum += (double)Elem<T>::to_f32(g[i]) * (double)Elem<T>::to_f32(g[i]);
    for (long long i = head + packets * L + threadIdx.x; i < n; i += kClipThreads) sum += (double)Elem<T>::to_f32(g[i]) * (double)Elem<T>::to_f32(g[i]);
    const T* body = g + head;
    long long k = threadIdx.x;
    for (; k + (U - 1) * kClipThreads < packets; k += kClipThreads * U) {
        Vec16<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = ld_keep(body + (k + u * kClipThreads) * L);
#pragma unroll
        for (int u = 0; u < U; ++u) sum += clip_squares<T>(v[u]);
    }
    for (; k < packets; k += kClipThreads) sum += clip_squares<T>(ld_keep(body + k * L));
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

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipCtas) clip_norm_kernel(const __grid_constant__ ClipTable<N> t) {
    __shared__ double scratch[kClipThreads / 32];
    double sum = 0.0;
    pdl_trigger();
    long long c, to;
    for (clip_share(t, c, to); c < to;) {
        const ClipEntry& e = t.e[clip_find(t, c)];
        const long long at = (c - e.first_chunk) * kClipChunk, rest = (to - c) * kClipChunk, n = e.n - at < rest ? e.n - at : rest;
        if (e.dtype == CG_B200_F32) sum += clip_run_squares(static_cast<const float*>(e.in) + at, n);
        else if (e.dtype == CG_B200_BF16) sum += clip_run_squares(static_cast<const __nv_bfloat16*>(e.in) + at, n);
        else sum += clip_run_squares(static_cast<const __half*>(e.in) + at, n);
        c += (n + kClipChunk - 1) / kClipChunk;
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

// A thread's piece is one 16-byte packet of the wider side, so that a warp's stores are contiguous: 16-bit gradients that become fp32 are
// read 8 bytes at a time.
template <typename T, typename O>
__device__ __forceinline__ void clip_run_scale(const T* g, O* o, long long n, float factor) {
    constexpr int E = Vec16<O>::N, U = 2;   // elements of a piece; sizeof(O) >= sizeof(T)
    typedef typename std::conditional<E * sizeof(T) == 16, int4, int2>::type Raw;
    const long long head = clip_head(o, n);
    const bool vec = (reinterpret_cast<uintptr_t>(g + head) & (sizeof(Raw) - 1)) == 0;   // both sides reach a boundary at the same element
    const long long pieces = vec ? (n - head) / E : 0, loose = vec ? head : 0;
    for (long long i = threadIdx.x; i < loose; i += kClipThreads) o[i] = Elem<O>::from_f32(Elem<T>::to_f32(g[i]) * factor);
    for (long long i = loose + pieces * E + threadIdx.x; i < n; i += kClipThreads) o[i] = Elem<O>::from_f32(Elem<T>::to_f32(g[i]) * factor);
    const T* gb = g + head;
    O* ob = o + head;
    auto put = [&](long long k, const Raw& raw) {
        Vec16<T> v;
        *reinterpret_cast<Raw*>(&v) = raw;
        float f[Vec16<T>::N], q[E];
        unpack16<T>(v, f);
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = f[i] * factor;
        st_stream(ob + k * E, pack16<O>(q));
    };
    long long k = pieces - 1 - threadIdx.x;
    for (; k >= (U - 1) * kClipThreads; k -= kClipThreads * U) {
        Raw raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = __ldcs(reinterpret_cast<const Raw*>(gb + (k - u * kClipThreads) * E));
#pragma unroll
        for (int u = 0; u < U; ++u) put(k - u * kClipThreads, raw[u]);
    }
    for (; k >= 0; k -= kClipThreads) put(k, __ldcs(reinterpret_cast<const Raw*>(gb + k * E)));
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipCtas) clip_scale_kernel(const __grid_constant__ ClipTable<N> t) {
    __shared__ double scratch[kClipThreads / 32];
    pdl_trigger();
    pdl_wait();
    const double norm = clip_norm(t.all_parts, t.n_parts, scratch);
    if (t.norm && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = (float)norm;
    const double ratio = (double)t.max_norm / (norm + 1e-6);
    const float factor = ratio >= 1.0 ? 1.0f : (float)ratio;   // a norm that is not a number gives such a factor
    long long from, to;
    for (clip_share(t, from, to); to > from;) {
        const ClipEntry& e = t.e[clip_find(t, to - 1)];
        const long long c = e.first_chunk > from ? e.first_chunk : from, at = (c - e.first_chunk) * kClipChunk, rest = (to - c) * kClipChunk;
        const long long n = e.n - at < rest ? e.n - at : rest;
        to = c;
        if (e.in == e.out && factor == 1.0f) continue;   // already there
        if (e.dtype == CG_B200_F32) {
            clip_run_scale(static_cast<const float*>(e.in) + at, static_cast<float*>(e.out) + at, n, factor);
        } else if (e.dtype == CG_B200_BF16) {
            const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(e.in) + at;
            if (e.out_dtype == CG_B200_F32) clip_run_scale(g, static_cast<float*>(e.out) + at, n, factor);
            else clip_run_scale(g, static_cast<__nv_bfloat16*>(e.out) + at, n, factor);
        } else {
            const __half* g = static_cast<const __half*>(e.in) + at;
            if (e.out_dtype == CG_B200_F32) clip_run_scale(g, static_cast<float*>(e.out) + at, n, factor);
            else clip_run_scale(g, static_cast<__half*>(e.out) + at, n, factor);
        }
    }
}

__global__ void __launch_bounds__(kClipThreads) clip_norm_only_kernel(const double* parts, int n, float* norm) {
    __shared__ double scratch[kClipThreads / 32];
    pdl_trigger();
    pdl_wait();
    const double v = clip_norm(parts, n, scratch);
    if (threadIdx.x == 0) *norm = (float)v;
}

static long long clip_grid_cap() { return (long long)sm_count() * kClipCtas; }

// Nothing may be written twice, and nothing written may be another's input: a tensor is scaled in place, or into memory of its own, and
// the norm, written while the list is still read, is apart from all. The address ranges are sorted and swept once.
struct ClipRange {
    uintptr_t from, to;
    bool written;
};
static int clip_check_overlap(const cg_b200_grad* g, int64_t count, const float* norm) {
    ClipRange few[2 * kClipShort + 1];
    ClipRange* r = few;
    if (count > kClipShort && !(r = static_cast<ClipRange*>(malloc(((size_t)count * 2 + 1) * sizeof(ClipRange))))) return CG_B200_ERR_NO_MEMORY;
    int64_t n = 0;
    if (norm) r[n++] = {reinterpret_cast<uintptr_t>(norm), reinterpret_cast<uintptr_t>(norm) + sizeof(float), true};
    for (int64_t i = 0; i < count; ++i) {
        if (g[i].n == 0) continue;
        const uintptr_t in = reinterpret_cast<uintptr_t>(g[i].in), out = reinterpret_cast<uintptr_t>(g[i].out);
        r[n++] = {out, out + (size_t)g[i].n * dtype_bytes(g[i].out_dtype), true};
        if (in != out || g[i].dtype != g[i].out_dtype) r[n++] = {in, in + (size_t)g[i].n * dtype_bytes(g[i].dtype), false};
    }
    std::sort(r, r + n, [](const ClipRange& a, const ClipRange& b) { return a.from < b.from; });
    uintptr_t read_to = 0, written_to = 0;
    bool bad = false;
    for (int64_t i = 0; i < n && !bad; ++i) {
        bad = r[i].from < written_to || (r[i].written && r[i].from < read_to);
        uintptr_t& to = r[i].written ? written_to : read_to;
        if (r[i].to > to) to = r[i].to;
    }
    if (r != few) free(r);
    return bad ? CG_B200_ERR_INVALID_ARG : CG_B200_OK;
}

static int clip_check(const cg_b200_grad* g, int64_t count, const float* norm, bool scale) {
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
    }
    return scale ? clip_check_overlap(g, count, norm) : CG_B200_OK;
}

static size_t clip_workspace(int64_t count) {
    const int64_t launches = (count + kClipLong - 1) / kClipLong;
    return (size_t)(launches > 0 ? launches : 1) * (size_t)clip_grid_cap() * sizeof(double);
}

// The launches over the list, N tensors at a time: sums, or the scaled copies. *parts: sums written so far, or all of them.
template <int N>
static int clip_pass(const cg_b200_grad* g, int64_t count, float max_norm, float* norm, double* ws, bool scale, int* parts, cudaStream_t s) {
    ClipTable<N> t;
    int at = 0;
    for (int64_t i0 = 0; i0 < count; i0 += N) {
        t.count = 0;
        t.chunks = 0;
        for (int64_t i = i0; i < count && i < i0 + N; ++i) {
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
        t.n_parts = *parts;
        t.norm = at == 0 ? norm : nullptr;
        t.max_norm = max_norm;
        if (!scale) {
            clip_norm_kernel<N><<<grid, kClipThreads, 0, s>>>(t);
            CGB_CUDA(cudaGetLastError());
        } else {
            CGB_CUDA(launch_pdl(clip_scale_kernel<N>, grid, kClipThreads, 0, s, t));
        }
        at += (int)grid;
    }
    if (!scale) *parts = at;
    return CG_B200_OK;
}

static int clip_run(const cg_b200_grad* g, int64_t count, float max_norm, float* norm, double* ws, bool scale, cudaStream_t s) {
    auto pass = [&](bool second, int* parts) {
        return count <= kClipShort ? clip_pass<kClipShort>(g, count, max_norm, norm, ws, second, parts, s)
                                   : clip_pass<kClipLong>(g, count, max_norm, norm, ws, second, parts, s);
    };
    int parts = 0;
    const int st = pass(false, &parts);
    if (st) return st;
    if (scale && parts > 0) return pass(true, &parts);
    CGB_CUDA(launch_pdl(clip_norm_only_kernel, 1, kClipThreads, 0, s, (const double*)ws, parts, norm));
    return CG_B200_OK;
}

static int clip_entry(const cg_b200_grad* grads, int64_t count, float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                      bool scale, void* stream) {
    int st = clip_check(grads, count, norm, scale);
    if (st) return st;
    if (!norm) return CG_B200_ERR_NULL_POINTER;
    if (!aligned_to(norm, 4) || !aligned_to(workspace, 16)) return CG_B200_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < clip_workspace(count)) return CG_B200_ERR_WORKSPACE;
    // sums are written there while the list is read, and read while it and the norm are written
    const Bytes ws(workspace, (int64_t)clip_workspace(count), 1);
    bool bad = overlap(ws, Bytes(norm, 1, sizeof(float)));
    for (int64_t i = 0; i < count; ++i)
        bad |= overlap(ws, Bytes(grads[i].in, grads[i].n, dtype_bytes(grads[i].dtype))) ||
               (scale && overlap(ws, Bytes(grads[i].out, grads[i].n, dtype_bytes(grads[i].out_dtype))));
    if (bad) return CG_B200_ERR_INVALID_ARG;
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
