// layernorm.cu - layer norm for training: a forward pass that keeps its statistics, and the backward pass.
//
// The reference names the op (mean, variance, normalise, scale + shift, src/analysis/arithmetic_intensity.cpp:138-146) and has no
// gradient for it. With R rows of C columns, h = (x - mean) * rstd and g = dy * gamma:
//   forward   y  = h * gamma + beta                                     (mean and rstd = 1 / sqrt(var + eps) kept per row, fp32)
//   backward  dx = rstd * (g - sum(g) / C - h * sum(g * h) / C)         (the two sums over the row)
//             dgamma = sum over rows of dy * h,  dbeta = sum over rows of dy
//
// HBM-bound: forward moves 2 * R * C elements, backward 3 * R * C, each once. A row is read once into registers as 16-byte packets
// (packet j of thread t is packet j * TPR + t), reduced by TPR threads - part of a warp, a warp or a whole CTA - and written; the next
// row's packets are requested before the current row's reductions, so that loads are always in flight. In the backward pass each thread
// adds its columns' share of dgamma and dbeta to fp32 registers over all rows that its CTA walks; the CTAs' sums go to the workspace and
// a second kernel adds them up in a fixed order, so the result does not depend on timing.
//
// Rows whose width no packet divides start at a different offset from a 16-byte boundary each: `off` elements. The rows of one CTA are
// gridDim.x apart, a multiple of the packet length, so they all share one offset: packets stay aligned, the first and the last of a row
// are read and written element by element (never outside the row), and gamma / beta are kept in shared memory shifted by the same
// offset. Tensors whose bases lie at different offsets, and rows too long for the registers, take the streaming kernels.
#include <math.h>

#include "common.cuh"

namespace cgb {

struct LnParams {
    const void* in;      // x
    const void* dout;    // dy (backward)
    const void* gamma;   // may be null
    const void* beta;    // may be null (forward)
    void* out;           // y (forward) or dx (backward)
    float* mean;         // written by the forward pass (may be null), read by the backward pass
    float* rstd;
    float* part;         // backward: [gridDim.x][2][cols] fp32, or null when no weight gradient is asked for
    long long rows, cols;
    int off0;            // elements from a 16-byte boundary to the first row, the same for every tensor
    float eps;
};

template <int TPR> constexpr int kLnThreads = TPR <= 32 ? 128 : TPR;   // threads of a CTA

// Sum of two values over the TPR threads that share a row; every thread gets it. Two scratch halves take turns, so one barrier per call
// is enough.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* scratch, int& phase) {
    constexpr int W = TPR < 32 ? TPR : 32;
    const unsigned mask = W == 32 ? 0xffffffffu : ((1u << W) - 1u) << (threadIdx.x & 31 & ~(W - 1));
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(mask, v.x, o);
        v.y += __shfl_xor_sync(mask, v.y, o);
    }
    if constexpr (TPR > 32) {
        constexpr int N = TPR / 32;
        float2* s = scratch + (phase & 1) * N;
        phase ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
        __syncthreads();
        v = s[threadIdx.x & (N - 1)];
#pragma unroll
        for (int o = N / 2; o > 0; o >>= 1) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
    }
    return v;
}

// Packet k of a row whose columns start `off` elements behind the packet boundary `row0`; elements outside the row read as zero.
template <typename T, bool RAGGED>
__device__ __forceinline__ Vec16<T> ln_load(const T* row0, int k, int off, int cols) {
    constexpr int L = Vec16<T>::N;
    if constexpr (!RAGGED) {
        return ld_stream(row0 + k * L);
    } else {
        const int c0 = k * L - off;
        if (c0 >= 0 && c0 + L <= cols) return ld_stream(row0 + k * L);
        Vec16<T> v;
#pragma unroll
        for (int l = 0; l < L; ++l) v.v[l] = c0 + l >= 0 && c0 + l < cols ? row0[k * L + l] : Elem<T>::from_f32(0.0f);
        return v;
    }
}

template <typename T, bool RAGGED>
__device__ __forceinline__ void ln_store(T* row0, int k, int off, int cols, const Vec16<T>& v) {
    constexpr int L = Vec16<T>::N;
    const int c0 = k * L - off;
    if (!RAGGED || (c0 >= 0 && c0 + L <= cols)) {
        st_stream(row0 + k * L, v);
    } else {
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (c0 + l >= 0 && c0 + l < cols) row0[k * L + l] = v.v[l];
    }
}

// L parameters of packet k: from global memory (L1 keeps them) where packets and columns coincide, from the shifted copy otherwise.
template <typename TP, int L, bool RAGGED>
__device__ __forceinline__ void ln_param(const TP* p, const float* shifted, int k, float (&f)[L]) {
    if constexpr (RAGGED) {
#pragma unroll
        for (int l = 0; l < L; l += 4) {
            const float4 t = *reinterpret_cast<const float4*>(shifted + k * L + l);
            f[l] = t.x; f[l + 1] = t.y; f[l + 2] = t.z; f[l + 3] = t.w;
        }
    } else {
        constexpr int M = Vec16<TP>::N;   // M <= L: the parameters have the rows' type or fp32
#pragma unroll
        for (int l = 0; l < L; l += M) {
            float t[M];
            unpack16<TP>(ld_keep(p + k * L + l), t);
#pragma unroll
            for (int i = 0; i < M; ++i) f[l + i] = t[i];
        }
    }
}

template <typename TP>
__device__ __forceinline__ void ln_stage(float* shifted, const TP* p, int off, int cols, int padded) {
    for (int i = threadIdx.x; i < padded; i += blockDim.x) {
        const int c = i - off;
        shifted[i] = c >= 0 && c < cols ? Elem<TP>::to_f32(p[c]) : 0.0f;
    }
}

template <typename T, typename TP, int TPR, int CH, bool RAGGED>
__global__ void __launch_bounds__(kLnThreads<TPR>) ln_fwd_kernel(const __grid_constant__ LnParams p) {
    constexpr int L = Vec16<T>::N, THREADS = kLnThreads<TPR>, G = THREADS / TPR;
    extern __shared__ float4 ln_smem4[];
    __shared__ float2 scratch[TPR > 32 ? TPR / 16 : 1];
    float* sg = reinterpret_cast<float*>(ln_smem4);
    int phase = 0;
    const int cols = (int)p.cols, lane = threadIdx.x % TPR;
    // all rows of this CTA share the offset of row blockIdx.x: gridDim.x is a multiple of L when rows are ragged
    const int off = RAGGED ? (int)((p.off0 + (long long)blockIdx.x * cols) % L) : 0;
    const int n_pkt = (off + cols + L - 1) / L, padded = n_pkt * L;
    float* sb = sg + padded;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    const TP* beta = static_cast<const TP*>(p.beta);
    if constexpr (RAGGED) {
        if (gamma) ln_stage(sg, gamma, off, cols, padded);
        if (beta) ln_stage(sb, beta, off, cols, padded);
        __syncthreads();
    }
    const float inv_cols = 1.0f / (float)cols;
    const long long step = (long long)gridDim.x * G;
    long long row = (long long)(threadIdx.x / TPR) * gridDim.x + blockIdx.x;
    Vec16<T> raw[CH], nxt[CH];
    auto fetch = [&](Vec16<T> (&v)[CH], long long r) {
        const T* row0 = static_cast<const T*>(p.in) + r * p.cols - off;
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j * TPR + lane < n_pkt) v[j] = ln_load<T, RAGGED>(row0, j * TPR + lane, off, cols);
    };
    if (row < p.rows) fetch(raw, row);
    for (; row < p.rows; row += step) {
        if (row + step < p.rows) fetch(nxt, row + step);
        float x[CH][L];
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j * TPR + lane < n_pkt) {
                unpack16<T>(raw[j], x[j]);
#pragma unroll
                for (int l = 0; l < L; ++l) s.x += x[j][l];
            }
        const float mean = row_sum2<TPR>(s, scratch, phase).x * inv_cols;
        s.x = 0.0f;
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j * TPR + lane < n_pkt) {
                const int c0 = (j * TPR + lane) * L - off;
#pragma unroll
                for (int l = 0; l < L; ++l) {
                    x[j][l] -= mean;
                    if (RAGGED && (c0 + l < 0 || c0 + l >= cols)) x[j][l] = 0.0f;
                    s.x = fmaf(x[j][l], x[j][l], s.x);
                }
            }
        const float rstd = 1.0f / sqrtf(row_sum2<TPR>(s, scratch, phase).x * inv_cols + p.eps);
        if (lane == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        T* out0 = static_cast<T*>(p.out) + row * p.cols - off;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int k = j * TPR + lane;
            if (k < n_pkt) {
                float f[L];
#pragma unroll
                for (int l = 0; l < L; ++l) x[j][l] *= rstd;
                if (gamma) {
                    ln_param<TP, L, RAGGED>(gamma, sg, k, f);
#pragma unroll
                    for (int l = 0; l < L; ++l) x[j][l] *= f[l];
                }
                if (beta) {
                    ln_param<TP, L, RAGGED>(beta, sb, k, f);
#pragma unroll
                    for (int l = 0; l < L; ++l) x[j][l] += f[l];
                }
                ln_store<T, RAGGED>(out0, k, off, cols, pack16<T>(x[j]));
            }
            raw[j] = nxt[j];
        }
    }
}

template <typename T, typename TP, int TPR, int CH, bool RAGGED>
__global__ void __launch_bounds__(kLnThreads<TPR>) ln_bwd_kernel(const __grid_constant__ LnParams p) {
    constexpr int L = Vec16<T>::N, THREADS = kLnThreads<TPR>, G = THREADS / TPR;
    extern __shared__ float4 ln_smem4[];
    __shared__ float2 scratch[TPR > 32 ? TPR / 16 : 1];
    float* sg = reinterpret_cast<float*>(ln_smem4);
    int phase = 0;
    const int cols = (int)p.cols, lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const int off = RAGGED ? (int)((p.off0 + (long long)blockIdx.x * cols) % L) : 0;
    const int n_pkt = (off + cols + L - 1) / L, padded = n_pkt * L;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    if constexpr (RAGGED) {
        if (gamma) ln_stage(sg, gamma, off, cols, padded);
        __syncthreads();
    }
    const float inv_cols = 1.0f / (float)cols;
    const long long step = (long long)gridDim.x * G;
    long long row = (long long)group * gridDim.x + blockIdx.x;
    float dg[CH][L], db[CH][L];
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int l = 0; l < L; ++l) dg[j][l] = db[j][l] = 0.0f;
    Vec16<T> xr[CH], yr[CH], xn[CH], yn[CH];
    float mean, rstd, mean_n = 0.0f, rstd_n = 0.0f;
    auto fetch = [&](Vec16<T> (&xv)[CH], Vec16<T> (&yv)[CH], float& m, float& r, long long at) {
        const T* x0 = static_cast<const T*>(p.in) + at * p.cols - off;
        const T* y0 = static_cast<const T*>(p.dout) + at * p.cols - off;
        m = p.mean[at];
        r = p.rstd[at];
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j * TPR + lane < n_pkt) {
                xv[j] = ln_load<T, RAGGED>(x0, j * TPR + lane, off, cols);
                yv[j] = ln_load<T, RAGGED>(y0, j * TPR + lane, off, cols);
            }
    };
    if (row < p.rows) fetch(xr, yr, mean, rstd, row);
    for (; row < p.rows; row += step) {
        if (row + step < p.rows) fetch(xn, yn, mean_n, rstd_n, row + step);
        float2 s = make_float2(0.0f, 0.0f);   // sum(g), sum(g h)
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int k = j * TPR + lane;
            if (k < n_pkt) {
                float x[L], y[L], g[L];
                unpack16<T>(xr[j], x);
                unpack16<T>(yr[j], y);
                if (gamma) ln_param<TP, L, RAGGED>(gamma, sg, k, g);
#pragma unroll
                for (int l = 0; l < L; ++l) {
                    const float h = (x[l] - mean) * rstd;
                    dg[j][l] = fmaf(y[l], h, dg[j][l]);
                    db[j][l] += y[l];
                    const float t = gamma ? y[l] * g[l] : y[l];
                    s.x += t;
                    s.y = fmaf(t, h, s.y);
                }
            }
        }
        s = row_sum2<TPR>(s, scratch, phase);
        const float a = s.x * inv_cols, b = s.y * inv_cols;
        T* out0 = static_cast<T*>(p.out) + row * p.cols - off;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int k = j * TPR + lane;
            if (k < n_pkt && p.out) {
                float x[L], y[L], g[L];
                unpack16<T>(xr[j], x);
                unpack16<T>(yr[j], y);
                if (gamma) ln_param<TP, L, RAGGED>(gamma, sg, k, g);
#pragma unroll
                for (int l = 0; l < L; ++l) {
                    const float h = (x[l] - mean) * rstd;
                    const float t = gamma ? y[l] * g[l] : y[l];
                    x[l] = rstd * (t - a - h * b);
                }
                ln_store<T, RAGGED>(out0, k, off, cols, pack16<T>(x));
            }
            xr[j] = xn[j];
            yr[j] = yn[j];
        }
        mean = mean_n;
        rstd = rstd_n;
    }
    if (!p.part) return;
    // this CTA's sums: the row groups' registers are added in the order of the groups
    float* part = p.part + (long long)blockIdx.x * 2 * p.cols;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if constexpr (G == 1) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int k = j * TPR + lane;
                if (k < n_pkt) {
#pragma unroll
                    for (int l = 0; l < L; ++l) {
                        const int c = k * L + l - off;
                        if (!RAGGED || (c >= 0 && c < cols)) part[(long long)w * cols + c] = w ? db[j][l] : dg[j][l];
                    }
                }
            }
        } else {
            constexpr int SPAN = TPR * CH * L;   // the columns a group covers
            float* sum = sg;                      // G * SPAN floats; gamma's copy is not needed any more
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int l = 0; l < L; l += 4) {
                    const float* f = w ? &db[j][l] : &dg[j][l];
                    *reinterpret_cast<float4*>(sum + group * SPAN + (j * TPR + lane) * L + l) = make_float4(f[0], f[1], f[2], f[3]);
                }
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += THREADS) {
                float t = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) t += sum[g * SPAN + c + off];
                part[(long long)w * cols + c] = t;
            }
        }
    }
}

// ---- rows of any length and alignment --------------------------------------------------------------
template <typename T, typename TP>
__global__ void __launch_bounds__(256) ln_fwd_stream_kernel(const __grid_constant__ LnParams p) {
    __shared__ float2 scratch[16];
    int phase = 0;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    const TP* beta = static_cast<const TP*>(p.beta);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* in = static_cast<const T*>(p.in) + row * p.cols;
        T* out = static_cast<T*>(p.out) + row * p.cols;
        float2 s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x; c < p.cols; c += 256) s.x += Elem<T>::to_f32(in[c]);
        const float mean = row_sum2<256>(s, scratch, phase).x / (float)p.cols;
        s.x = 0.0f;
        for (long long c = threadIdx.x; c < p.cols; c += 256) {
            const float d = Elem<T>::to_f32(in[c]) - mean;
            s.x = fmaf(d, d, s.x);
        }
        const float rstd = 1.0f / sqrtf(row_sum2<256>(s, scratch, phase).x / (float)p.cols + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        // in == out is allowed: an element is read and written by the same thread
        for (long long c = threadIdx.x; c < p.cols; c += 256) {
            float v = (Elem<T>::to_f32(in[c]) - mean) * rstd;
            if (gamma) v *= Elem<TP>::to_f32(gamma[c]);
            if (beta) v += Elem<TP>::to_f32(beta[c]);
            out[c] = Elem<T>::from_f32(v);
        }
    }
}

template <typename T, typename TP>
__global__ void __launch_bounds__(256) ln_bwd_stream_kernel(const __grid_constant__ LnParams p) {
    __shared__ float2 scratch[16];
    int phase = 0;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.in) + row * p.cols;
        const T* y = static_cast<const T*>(p.dout) + row * p.cols;
        T* out = static_cast<T*>(p.out) + row * p.cols;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float2 s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x; c < p.cols; c += 256) {
            const float h = (Elem<T>::to_f32(x[c]) - mean) * rstd;
            const float t = Elem<T>::to_f32(y[c]) * (gamma ? Elem<TP>::to_f32(gamma[c]) : 1.0f);
            s.x += t;
            s.y = fmaf(t, h, s.y);
        }
        s = row_sum2<256>(s, scratch, phase);
        const float a = s.x / (float)p.cols, b = s.y / (float)p.cols;
        for (long long c = threadIdx.x; c < p.cols; c += 256) {
            const float h = (Elem<T>::to_f32(x[c]) - mean) * rstd;
            const float t = Elem<T>::to_f32(y[c]) * (gamma ? Elem<TP>::to_f32(gamma[c]) : 1.0f);
            out[c] = Elem<T>::from_f32(rstd * (t - a - h * b));
        }
    }
}

// The weight gradients' share of a slice of rows (blockIdx.y of gridDim.y) for 32 columns.
template <typename T>
__global__ void __launch_bounds__(256) ln_bwd_columns_kernel(const __grid_constant__ LnParams p) {
    __shared__ float2 sum[8][32];
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < p.cols)
        for (long long r = (long long)blockIdx.y * 8 + threadIdx.y; r < p.rows; r += (long long)gridDim.y * 8) {
            const float y = Elem<T>::to_f32(static_cast<const T*>(p.dout)[r * p.cols + c]);
            const float h = (Elem<T>::to_f32(static_cast<const T*>(p.in)[r * p.cols + c]) - p.mean[r]) * p.rstd[r];
            s.x = fmaf(y, h, s.x);
            s.y += y;
        }
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < p.cols) {
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            s.x += sum[i][threadIdx.x].x;
            s.y += sum[i][threadIdx.x].y;
        }
        float* part = p.part + (long long)blockIdx.y * 2 * p.cols;
        part[c] = s.x;
        part[p.cols + c] = s.y;
    }
}

// dgamma (blockIdx.y == 0) and dbeta (1): the sums of `parts` rows of the workspace, in a fixed order
template <typename TP>
__global__ void __launch_bounds__(256) ln_weight_grad_kernel(const float* part, long long parts, long long cols, TP* dgamma, TP* dbeta) {
    __shared__ float sum[8][32];
    TP* out = blockIdx.y ? dbeta : dgamma;
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (out && c < cols) {
        const float* q = part + blockIdx.y * cols + c;
#pragma unroll 4
        for (long long i = threadIdx.y; i < parts; i += 8) s += q[i * 2 * cols];
    }
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && out && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += sum[i][threadIdx.x];
        out[c] = Elem<TP>::from_f32(s);
    }
}

// CTAs that the backward pass starts at most: their sums are the workspace
static long long ln_max_parts(long long rows) {
    const long long cap = (long long)sm_count() * 3;
    return ((rows < cap ? rows : cap) + 7) / 8 * 8;
}

template <typename T, typename TP, int TPR, int CH, bool BWD>
static int ln_launch(const LnParams& p, bool ragged, int* parts, cudaStream_t s) {
    constexpr int L = Vec16<T>::N, THREADS = kLnThreads<TPR>, G = THREADS / TPR;
    // Backward CTAs are resident all at once (three of 128 threads per SM, or 384 threads' worth); the forward pass keeps more in flight.
    const long long cap = BWD ? (long long)sm_count() * (THREADS >= 512 ? 1 : THREADS == 256 ? 2 : 3) : (long long)sm_count() * (2048 / THREADS);
    long long grid = (p.rows + G - 1) / G;
    if (grid > cap) grid = cap;
    if (ragged) grid = (grid + L - 1) / L * L;
    const int padded = (int)((p.cols + 2 * L - 2) / L) * L;   // of the largest offset
    size_t smem = ragged ? (size_t)padded * 4 * (BWD ? 1 : 2) : 0;
    if (BWD && G > 1 && smem < (size_t)G * TPR * CH * L * 4) smem = (size_t)G * TPR * CH * L * 4;
    if (parts) *parts = (int)grid;
#define CGB_LN_GO(R)                                                                                                        \
    {                                                                                                                       \
        auto k = BWD ? ln_bwd_kernel<T, TP, TPR, CH, R> : ln_fwd_kernel<T, TP, TPR, CH, R>;                                 \
        if (smem > 48 * 1024) CGB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));    \
        k<<<(unsigned)grid, THREADS, smem, s>>>(p);                                                                         \
    }
    if (ragged) CGB_LN_GO(true) else CGB_LN_GO(false)
#undef CGB_LN_GO
    CGB_CUDA(cudaGetLastError());
    return CG_B200_OK;
}

// Whether all tensors start the same number of elements behind a 16-byte boundary
static bool ln_congruent(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0; }

// The register kernels' variants: threads per row and packets per thread by the packets of a row. -1: none, the streaming kernels take it.
template <typename T, typename TP, bool BWD>
static int ln_registers(LnParams p, bool params_aligned, int* parts, cudaStream_t s) {
    constexpr int L = Vec16<T>::N;
    if (!ln_congruent(p.in, p.out ? p.out : p.in) || (BWD && !ln_congruent(p.in, p.dout))) return -1;
    p.off0 = (int)((reinterpret_cast<uintptr_t>(p.in) & 15) / sizeof(T));
    const bool ragged = p.off0 != 0 || p.cols % L != 0 || !params_aligned;
    const long long n = ragged ? (p.cols + 2 * L - 2) / L : p.cols / L;
    if (n <= 8) return ln_launch<T, TP, 8, 1, BWD>(p, ragged, parts, s);
    if (n <= 32) return ln_launch<T, TP, 32, 1, BWD>(p, ragged, parts, s);
    if (n <= 64) return ln_launch<T, TP, 32, 2, BWD>(p, ragged, parts, s);
    if (n <= 128) return ln_launch<T, TP, 32, 4, BWD>(p, ragged, parts, s);
    if (n <= 256) return ln_launch<T, TP, 128, 2, BWD>(p, ragged, parts, s);
    if (n <= 512) return ln_launch<T, TP, 128, 4, BWD>(p, ragged, parts, s);
    if (n <= 1024) return ln_launch<T, TP, 256, 4, BWD>(p, ragged, parts, s);
    if (n <= 2048) return ln_launch<T, TP, 512, 4, BWD>(p, ragged, parts, s);
    return -1;
}

template <typename T, typename TP>
static int ln_forward(const LnParams& p, cudaStream_t s) {
    const bool aligned = aligned_to(p.gamma, 16) && aligned_to(p.beta, 16);
    const int st = ln_registers<T, TP, false>(p, aligned, nullptr, s);
    if (st >= 0) return st;
    const long long cap = (long long)sm_count() * 8;
    ln_fwd_stream_kernel<T, TP><<<(unsigned)(p.rows < cap ? p.rows : cap), 256, 0, s>>>(p);
    CGB_CUDA(cudaGetLastError());
    return CG_B200_OK;
}

template <typename T, typename TP>
static int ln_backward(const LnParams& p, void* dgamma, void* dbeta, cudaStream_t s) {
    int parts = 0;
    if (p.rows > 0 && (p.out || p.part)) {
        const int st = ln_registers<T, TP, true>(p, aligned_to(p.gamma, 16), &parts, s);
        if (st > 0) return st;
        if (st < 0) {
            const long long cap = (long long)sm_count() * 8;
            if (p.part) {   // before dx, which may lie where dy does
                const long long tiles = (p.cols + 31) / 32;
                long long slices = cap / tiles;
                const long long most = ln_max_parts(p.rows) < (p.rows + 7) / 8 ? ln_max_parts(p.rows) : (p.rows + 7) / 8;
                slices = slices < 1 ? 1 : slices > most ? most : slices;
                parts = (int)slices;
                ln_bwd_columns_kernel<T><<<dim3((unsigned)tiles, (unsigned)slices), dim3(32, 8), 0, s>>>(p);
                CGB_CUDA(cudaGetLastError());
            }
            if (p.out) {
                ln_bwd_stream_kernel<T, TP><<<(unsigned)(p.rows < cap ? p.rows : cap), 256, 0, s>>>(p);
                CGB_CUDA(cudaGetLastError());
            }
        }
    }
    if (dgamma || dbeta) {
        ln_weight_grad_kernel<TP><<<dim3((unsigned)((p.cols + 31) / 32), 2), dim3(32, 8), 0, s>>>(p.part, parts, p.cols, static_cast<TP*>(dgamma),
                                                                                                  static_cast<TP*>(dbeta));
        CGB_CUDA(cudaGetLastError());
    }
    return CG_B200_OK;
}

#define CGB_LN_DISPATCH(FN, ...)                                                                                            \
    switch (dtype) {                                                                                                        \
        case CG_B200_F32: return FN<float, float>(__VA_ARGS__);                                                             \
        case CG_B200_BF16: return param_dtype == CG_B200_F32 ? FN<__nv_bfloat16, float>(__VA_ARGS__)                        \
                                                             : FN<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__);               \
        default: return param_dtype == CG_B200_F32 ? FN<__half, float>(__VA_ARGS__) : FN<__half, __half>(__VA_ARGS__);      \
    }

static int ln_dispatch_forward(int dtype, int param_dtype, const LnParams& p, cudaStream_t s) { CGB_LN_DISPATCH(ln_forward, p, s) }
static int ln_dispatch_backward(int dtype, int param_dtype, const LnParams& p, void* dgamma, void* dbeta, cudaStream_t s) {
    CGB_LN_DISPATCH(ln_backward, p, dgamma, dbeta, s)
}
#undef CGB_LN_DISPATCH

// The largest row count / width whose element offsets and grids stay inside the types used here
static bool ln_sizes_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && cols >= 0 && (cols == 0 || rows <= (int64_t(1) << 62) / cols) && cols <= (int64_t(1) << 36);
}

}  // namespace cgb

extern "C" int cg_b200_layernorm_forward(int dtype, int param_dtype, const void* in, const void* gamma, const void* beta, float eps,
                                         void* out, float* mean, float* rstd, int64_t rows, int64_t cols, void* stream) {
    using namespace cgb;
    if (!dtype_ok(dtype) || (param_dtype != dtype && param_dtype != CG_B200_F32) || !ln_sizes_ok(rows, cols)) return CG_B200_ERR_INVALID_ARG;
    if (!(eps >= 0.0f)) return CG_B200_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return CG_B200_OK;
    if (!in || !out) return CG_B200_ERR_NULL_POINTER;
    const size_t esz = dtype_bytes(dtype), psz = dtype_bytes(param_dtype);
    if (!aligned_to(in, esz) || !aligned_to(out, esz) || !aligned_to(gamma, psz) || !aligned_to(beta, psz) || !aligned_to(mean, 4) ||
        !aligned_to(rstd, 4))
        return CG_B200_ERR_MISALIGNED;
    int st = require_sm100();
    if (st) return st;
    LnParams p{};
    p.in = in;
    p.gamma = gamma;
    p.beta = beta;
    p.out = out;
    p.mean = mean;
    p.rstd = rstd;
    p.rows = rows;
    p.cols = cols;
    p.eps = eps;
    return ln_dispatch_forward(dtype, param_dtype, p, (cudaStream_t)stream);
}

extern "C" int cg_b200_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols, size_t* bytes) {
    using namespace cgb;
    if (!bytes) return CG_B200_ERR_NULL_POINTER;
    *bytes = 0;
    if (!ln_sizes_ok(rows, cols)) return CG_B200_ERR_INVALID_ARG;
    *bytes = (size_t)ln_max_parts(rows) * 2 * (size_t)cols * sizeof(float);
    return CG_B200_OK;
}

extern "C" int cg_b200_layernorm_backward(int dtype, int param_dtype, const void* dout, const void* in, const void* gamma, const float* mean,
                                          const float* rstd, void* din, void* dgamma, void* dbeta, int64_t rows, int64_t cols,
                                          void* workspace, size_t workspace_bytes, void* stream) {
    using namespace cgb;
    if (!dtype_ok(dtype) || (param_dtype != dtype && param_dtype != CG_B200_F32) || !ln_sizes_ok(rows, cols)) return CG_B200_ERR_INVALID_ARG;
    if (cols == 0 || (rows == 0 && !dgamma && !dbeta)) return CG_B200_OK;
    if (rows > 0 && (!dout || !in || !mean || !rstd)) return CG_B200_ERR_NULL_POINTER;
    if (!din && !dgamma && !dbeta) return CG_B200_ERR_NULL_POINTER;
    const size_t esz = dtype_bytes(dtype), psz = dtype_bytes(param_dtype);
    if (!aligned_to(dout, esz) || !aligned_to(in, esz) || !aligned_to(din, esz) || !aligned_to(gamma, psz) || !aligned_to(dgamma, psz) ||
        !aligned_to(dbeta, psz) || !aligned_to(mean, 4) || !aligned_to(rstd, 4) || !aligned_to(workspace, 16))
        return CG_B200_ERR_MISALIGNED;
    size_t need = 0;
    cg_b200_layernorm_backward_workspace_bytes(rows, cols, &need);
    if ((dgamma || dbeta) && need > 0 && (!workspace || workspace_bytes < need)) return CG_B200_ERR_WORKSPACE;
    int st = require_sm100();
    if (st) return st;
    LnParams p{};
    p.in = in;
    p.dout = dout;
    p.gamma = gamma;
    p.out = din;
    p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd);
    p.part = dgamma || dbeta ? static_cast<float*>(workspace) : nullptr;
    p.rows = rows;
    p.cols = cols;
    return ln_dispatch_backward(dtype, param_dtype, p, dgamma, dbeta, (cudaStream_t)stream);
}
