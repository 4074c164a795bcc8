// layernorm.cu - layer norm for training: a forward pass that keeps its statistics, and the backward pass.
//
// The reference names the op (mean, variance, normalise, scale + shift, src/analysis/arithmetic_intensity.cpp:138-146) and has no
// gradient for it. With R rows of C columns, h = (x - mean) * rstd and g = dy * gamma:
//   forward   y  = h * gamma + beta                                     (mean and rstd = 1 / sqrt(var + eps) kept per row, fp32)
//   backward  dx = rstd * (g - sum(g) / C - h * sum(g * h) / C)         (the two sums over the row)
//             dgamma = sum over rows of dy * h,  dbeta = sum over rows of dy
//
// HBM-bound: forward moves 2 * R * C elements, backward 3 * R * C, each once (measured: 65536 x 1024 bf16 forward 48 us, 85 % of the copy
// rate; 32768 x 4096 bf16 backward 135 us, 91 %; 14000 x 8000 fp32 147 and 215 us, 93 and 95 %). One CTA per SM
// walks the rows; its threads form groups, a row (forward: two rows at once) to a group: eight threads, a warp, or up to 16 warps with a
// barrier of their own. A row is 16-byte packets, packet j * TPR + t for thread t, copied asynchronously into shared memory ahead of
// its use: a thread copies and reads its own packets only, so nothing but its own copies has to be waited for, and loads stay in flight
// while rows are reduced without costing registers (loads into registers, with a row's lookahead: 59 and 229 us). In the backward pass
// each thread adds its columns' share of dgamma and dbeta to fp32 registers over all rows of its group; the groups' sums are joined in
// shared memory, the CTAs' sums go to the workspace and a second kernel adds them up, all in a fixed order, so the result does not
// depend on timing. (A group's running sum takes rows / (148 * groups) terms, 110 for 32768 x 4096 bf16; the register kernels' error in
// dgamma and dbeta grows with that, the streaming kernels' does not.) Arithmetic is on fp32 pairs: with single instructions the backward
// pass is bound by issue before it is bound by HBM.
//
// Rows whose width no packet divides start at a different offset from a 16-byte boundary each. The rows of one CTA are gridDim.x apart, a
// multiple of the packet length, so they all share one offset and a column stays with its thread. The columns before a row's first
// boundary and behind its last one, fewer than a packet each, are single columns of the group's first threads, which read them one
// iteration ahead; everything between is packets as elsewhere. (Ends inside packets, masked, made two threads slower than the group
// that waits for them: 65 us instead of 38 for 8192 rows of 4097 bf16, forward.) Tensors whose bases lie at different offsets, and
// rows too long for the registers, take the streaming kernels.
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

constexpr int kLnThreads = 512;   // of a CTA at most: 128 registers each
constexpr int kLnWarps = kLnThreads / 32;
// Dynamic shared memory of a CTA at most: of 227 KB, with the static scratch and what the system keeps per CTA
constexpr int kLnSmem = 208 * 1024;

// Sums of N values over the threads that share a row (8 lanes of a warp when SUB, else `warps` warps); every thread gets them. The warps
// of a group meet at barrier `bar`; two scratch halves take turns, so one barrier per call is enough.
template <int N> struct alignas(N % 2 == 0 ? 8 : 4) LnSums {
    float v[N];
};
template <int N>
__device__ __forceinline__ void ln_add_across(LnSums<N>& s, unsigned mask, int o) {
    LnSums<N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = __shfl_xor_sync(mask, s.v[i], o);
#pragma unroll
    for (int i = 0; i < N; ++i) s.v[i] += t.v[i];
}
template <bool SUB, int N>
__device__ __forceinline__ void row_sum(LnSums<N>& s, LnSums<N>* scratch, int& phase, int bar, int warps) {
    const unsigned mask = SUB ? 0xffu << (threadIdx.x & 24) : 0xffffffffu;
#pragma unroll
    for (int o = SUB ? 4 : 16; o > 0; o >>= 1) ln_add_across(s, mask, o);
    if (!SUB && warps > 1) {
        const int lane = threadIdx.x & 31;
        LnSums<N>* at = scratch + phase;
        phase ^= 16;
        if (lane == 0) at[(threadIdx.x >> 5) % warps] = s;
        asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
        if (warps <= 4) {
            s = at[0];
            for (int w = 1; w < warps; ++w)
#pragma unroll
                for (int i = 0; i < N; ++i) s.v[i] += at[w].v[i];
            return;
        }
        s = at[lane < warps ? lane : 0];
#pragma unroll
        for (int i = 0; i < N; ++i) s.v[i] = lane < warps ? s.v[i] : 0.0f;
        if (warps > 8) ln_add_across(s, 0xffffffffu, 8);
        ln_add_across(s, 0xffffffffu, 4);
        ln_add_across(s, 0xffffffffu, 2);
        ln_add_across(s, 0xffffffffu, 1);
        // lanes 0 .. 7 (0 .. 15) hold the sums, the others added zeros
#pragma unroll
        for (int i = 0; i < N; ++i) s.v[i] = __shfl_sync(0xffffffffu, s.v[i], 0);
    }
}

// The same for two values, which is what the kernels below reduce, with half the shuffles: from the first exchange on, one half of the lanes
// adds up the first value and the other half the second. Behind the barrier every thread reads all warps' sums, two to a 16-byte read;
// entries from `warps` on are zero (row_sum2_prepare). warp: the thread's in its group.
template <bool SUB>
__device__ __forceinline__ void row_sum2(LnSums<2>& s, LnSums<2>* scratch, int& phase, int bar, int warps, int warp) {
    constexpr int HALF = SUB ? 4 : 16;
    const int lane = threadIdx.x & 31;
    const unsigned mask = SUB ? 0xffu << (lane & 24) : 0xffffffffu;
    const bool second = lane & HALF;
    float v = second ? s.v[1] : s.v[0];
    v += __shfl_xor_sync(mask, second ? s.v[0] : s.v[1], HALF);
#pragma unroll
    for (int o = HALF / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    if (SUB || warps == 1) {
        s.v[0] = __shfl_sync(mask, v, SUB ? lane & 24 : 0);
        s.v[1] = __shfl_sync(mask, v, (SUB ? lane & 24 : 0) + HALF);
        return;
    }
    LnSums<2>* at = scratch + phase;
    phase ^= 16;
    if ((lane & 15) == 0) at[warp].v[lane >> 4] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
    const float4* q = reinterpret_cast<const float4*>(at);
    auto two = [&](int i) {
        const float4 t = q[i];
        return __fadd2_rn(make_float2(t.x, t.y), make_float2(t.z, t.w));
    };
    float2 t = __fadd2_rn(two(0), two(1));
    if (warps > 4) t = __fadd2_rn(t, __fadd2_rn(two(2), two(3)));
    if (warps > 8) t = __fadd2_rn(t, __fadd2_rn(__fadd2_rn(two(4), two(5)), __fadd2_rn(two(6), two(7))));
    s.v[0] = t.x;
    s.v[1] = t.y;
}
// By all threads of a group, lane their number in it, before its first row_sum2
__device__ __forceinline__ void row_sum2_prepare(LnSums<2>* scratch, int lane, int warps) {
    if (lane < 32 && (lane & 15) >= warps) scratch[lane] = LnSums<2>{};
}

// until at most `stages` - 1 of this thread's groups are under way
__device__ __forceinline__ void ln_wait(int stages) {
    if (stages >= 3) copy_wait<2>();
    else if (stages == 2) copy_wait<1>();
    else copy_wait<0>();
}

// Where the packets of a ragged row lie: `head` columns, `packets` packets, `tail` columns from `tail0` on.
struct LnSpan {
    int head, packets, tail0, tail;
};
template <int L, bool RAGGED>
__device__ __forceinline__ LnSpan ln_span(const LnParams& p) {
    // all rows of this CTA share the offset of row blockIdx.x: gridDim.x is a multiple of L when rows are ragged
    const int cols = (int)p.cols, off = RAGGED ? (int)((p.off0 + (long long)blockIdx.x * cols) % L) : 0;
    LnSpan s;
    s.head = off == 0 ? 0 : L - off < cols ? L - off : cols;
    s.packets = (cols - s.head) / L;
    s.tail0 = s.head + s.packets * L;
    s.tail = cols - s.tail0;
    return s;
}

// L values as fp32 pairs
template <typename T>
__device__ __forceinline__ void ln_pairs(const Vec16<T>& v, float2* f) {
    float t[Vec16<T>::N];
    unpack16<T>(v, t);
#pragma unroll
    for (int i = 0; i < Vec16<T>::N / 2; ++i) f[i] = make_float2(t[2 * i], t[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ Vec16<T> ln_packet(const float2* f) {
    float t[Vec16<T>::N];
#pragma unroll
    for (int i = 0; i < Vec16<T>::N / 2; ++i) {
        t[2 * i] = f[i].x;
        t[2 * i + 1] = f[i].y;
    }
    return pack16<T>(t);
}

// The L parameters of the packet with the columns c0 ..; `none` without parameters.
template <typename TP, int L, bool RAGGED>
__device__ __forceinline__ void ln_param(const TP* p, int c0, float none, float2 (&f)[L / 2]) {
    if (!p) {
#pragma unroll
        for (int l = 0; l < L / 2; ++l) f[l] = make_float2(none, none);
    } else if constexpr (RAGGED) {
#pragma unroll
        for (int l = 0; l < L / 2; ++l) f[l] = make_float2(Elem<TP>::to_f32(p[c0 + 2 * l]), Elem<TP>::to_f32(p[c0 + 2 * l + 1]));
    } else {
        constexpr int M = Vec16<TP>::N;   // M <= L: the parameters have the rows' type or fp32
#pragma unroll
        for (int l = 0; l < L; l += M) ln_pairs<TP>(ld_keep(p + c0 + l), f + l / 2);
    }
}

// The single columns of a thread: number `lane` of the head and of the tail, where there are so many.
struct LnSingles {
    bool have[2];
    int col[2];
};
__device__ __forceinline__ LnSingles ln_singles(const LnSpan& s, int lane) {
    return LnSingles{{lane < s.head, lane < s.tail}, {lane, s.tail0 + lane}};
}

// How a CTA's threads share its rows (the launch's choice, see ln_launch)
struct LnShape {
    int tpr;        // threads per row: 8 when SUB, else a multiple of 32
    int groups;     // rows at a time
    int stages;     // steps of a group in shared memory: the one in work and the next ones
};

// CH packets per thread; the parameters stay in registers. A group takes R rows at a time: the dependent reductions of a row are latency,
// which the rows share.
template <typename T, typename TP, int CH, int R, bool SUB, bool RAGGED>
__global__ void __launch_bounds__(kLnThreads, 1) ln_fwd_kernel(const __grid_constant__ LnParams p, const LnShape sh) {
    constexpr int L = Vec16<T>::N;
    extern __shared__ float4 ln_smem4[];
    __shared__ alignas(16) LnSums<R> scratch_all[SUB ? 1 : kLnWarps * 32];
    const int tpr = SUB ? 8 : sh.tpr, group = threadIdx.x / tpr, lane = threadIdx.x - group * tpr, warps = tpr >> 5;
    LnSums<R>* scratch = scratch_all + (SUB ? 0 : group * 32);
    int phase = 0;
    if constexpr (R == 2 && !SUB) row_sum2_prepare(scratch, lane, warps);
    const int cols = (int)p.cols;
    const LnSpan span = ln_span<L, RAGGED>(p);
    Vec16<T>* ring = reinterpret_cast<Vec16<T>*>(ln_smem4) + threadIdx.x;   // this thread's slots: [stages][R][CH], kLnThreads apart
    const long long step = (long long)gridDim.x * sh.groups, first = (long long)group * gridDim.x + blockIdx.x;
    const int left = first < p.rows ? (int)((p.rows - 1 - first) / step) + 1 : 0;   // rows of this group
    const int c_lane = span.head + lane * L, c_step = tpr * L;
    auto live = [&](int j) { return j * tpr + lane < span.packets; };
    const T* src = static_cast<const T*>(p.in) + first * p.cols + c_lane;   // of the next row to fetch
    int to_fetch = left;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    // Rows read first make room in L2 for rows being written: 131072 x 512 bf16 51.3 -> 49.4 us, 24576 x 4096 fp32 145 -> 139 us (bf16 of
    // that shape 66 -> 69 us). Not of ragged rows, whose ends share sectors with their neighbours: 32700 x 1027 fp32 51.1 -> 53.6 us.
    const uint64_t once = leaves_l2_first();
    auto fetch = [&](Vec16<T>* slot) {
        const uint32_t to = ring_at + (uint32_t)(slot - ring) * 16;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to_fetch-- > 0) {
#pragma unroll
                for (int j = 0; j < CH; ++j)
                    if (live(j)) {
                        if constexpr (RAGGED) copy16_async(to + (r * CH + j) * (kLnThreads * 16), src + j * c_step);
                        else copy16_async(to + (r * CH + j) * (kLnThreads * 16), src + j * c_step, once);
                    }
                src += step * p.cols;
            } else if (r > 0) {
#pragma unroll
                for (int j = 0; j < CH; ++j) slot[(r * CH + j) * kLnThreads] = Vec16<T>{};
            }
        copy_commit();
    };
    // what a thread does not fetch it reads as zero: the arithmetic below asks nothing about packets and rows that are not there
    for (int i = 0; i < sh.stages * R; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (!live(j)) ring[(i * CH + j) * kLnThreads] = Vec16<T>{};
    for (int i = 0; i < sh.stages; ++i) fetch(ring + i * R * CH * kLnThreads);
    // single columns of the next rows, zero where there are none
    const LnSingles one = ln_singles(span, lane);
    T next[R][2];
    auto singles = [&](int i) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                next[r][k] = Elem<T>::from_f32(0.0f);
                if (one.have[k] && i + r < left) next[r][k] = static_cast<const T*>(p.in)[(first + (i + r) * step) * p.cols + one.col[k]];
            }
    };
    float g1[2] = {1.0f, 1.0f}, b1[2] = {0.0f, 0.0f};
    if constexpr (RAGGED) {
        singles(0);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (one.have[k]) {
                if (p.gamma) g1[k] = Elem<TP>::to_f32(static_cast<const TP*>(p.gamma)[one.col[k]]);
                if (p.beta) b1[k] = Elem<TP>::to_f32(static_cast<const TP*>(p.beta)[one.col[k]]);
            }
    }
    float2 g[CH][L / 2], b[CH][L / 2];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        ln_param<TP, L, RAGGED>(live(j) ? static_cast<const TP*>(p.gamma) : nullptr, c_lane + j * c_step, 1.0f, g[j]);
        ln_param<TP, L, RAGGED>(live(j) ? static_cast<const TP*>(p.beta) : nullptr, c_lane + j * c_step, 0.0f, b[j]);
    }
    const float inv_cols = 1.0f / (float)cols;
    T* dst = static_cast<T*>(p.out) + first * p.cols + c_lane;
    long long row = first;
    int stage = 0;
    for (int i = 0; i < left; i += R) {
        Vec16<T>* slot = ring + stage * R * CH * kLnThreads;
        stage = stage + 1 == sh.stages ? 0 : stage + 1;
        ln_wait(sh.stages);
        float2 x[R][CH][L / 2];
        LnSums<R> s;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < CH; ++j) ln_pairs<T>(slot[(r * CH + j) * kLnThreads], x[r][j]);
        fetch(slot);
        float e[R][2];
        if constexpr (RAGGED) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) e[r][k] = Elem<T>::to_f32(next[r][k]);
            singles(i + R);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int l = 0; l < L / 2; ++l) t = __fadd2_rn(t, x[r][j][l]);
            if constexpr (RAGGED) t = __fadd2_rn(t, make_float2(e[r][0], e[r][1]));
            s.v[r] = t.x + t.y;
        }
        if constexpr (R == 2) row_sum2<SUB>(s, scratch, phase, group + 1, warps, lane >> 5);
        else row_sum<SUB>(s, scratch, phase, group + 1, warps);
        float mean[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = s.v[r] * inv_cols;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const float neg = live(j) ? -mean[r] : 0.0f;   // what is not there stays zero
#pragma unroll
                for (int l = 0; l < L / 2; ++l) x[r][j][l] = __fadd2_rn(x[r][j][l], make_float2(neg, neg));
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int l = 0; l < L / 2; ++l) t = __ffma2_rn(x[r][j][l], x[r][j][l], t);
            if constexpr (RAGGED) {
#pragma unroll
                for (int k = 0; k < 2; ++k) e[r][k] = one.have[k] ? e[r][k] - mean[r] : 0.0f;
                const float2 d = make_float2(e[r][0], e[r][1]);
                t = __ffma2_rn(d, d, t);
            }
            s.v[r] = t.x + t.y;
        }
        if constexpr (R == 2) row_sum2<SUB>(s, scratch, phase, group + 1, warps, lane >> 5);
        else row_sum<SUB>(s, scratch, phase, group + 1, warps);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r == 0 || i + r < left) {
                const float rstd = rsqrtf(s.v[r] * inv_cols + p.eps);
                if (lane == 0) {
                    if (p.mean) p.mean[row] = mean[r];
                    if (p.rstd) p.rstd[row] = rstd;
                }
                const float2 rstd2 = make_float2(rstd, rstd);
#pragma unroll
                for (int j = 0; j < CH; ++j) {
#pragma unroll
                    for (int l = 0; l < L / 2; ++l) x[r][j][l] = __ffma2_rn(__fmul2_rn(x[r][j][l], rstd2), g[j][l], b[j][l]);
                    if (live(j)) st_stream(dst + j * c_step, ln_packet<T>(x[r][j]));
                }
                if constexpr (RAGGED) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (one.have[k])
                            static_cast<T*>(p.out)[row * p.cols + one.col[k]] = Elem<T>::from_f32(fmaf(e[r][k] * rstd, g1[k], b1[k]));
                }
                row += step;
                dst += step * p.cols;
            }
    }
}

// KEEP: the parameters and, from the first to the second pass over a row, its g and h stay in registers (up to 16 columns per thread);
// otherwise both passes read the row from shared memory and the parameters anew (32 columns, one row at a time).
template <typename T, typename TP, int CH, int R, bool SUB, bool RAGGED>
__global__ void __launch_bounds__(kLnThreads, 1) ln_bwd_kernel(const __grid_constant__ LnParams p, const LnShape sh) {
    constexpr int L = Vec16<T>::N;
    constexpr bool KEEP = CH * L <= 16;
    static_assert(KEEP || R == 1, "rows at a time are kept in registers");
    extern __shared__ float4 ln_smem4[];
    __shared__ alignas(16) LnSums<2 * R> scratch_all[SUB ? 1 : kLnWarps * 32];
    const int tpr = SUB ? 8 : sh.tpr, group = threadIdx.x / tpr, lane = threadIdx.x - group * tpr, warps = tpr >> 5;
    LnSums<2 * R>* scratch = scratch_all + (SUB ? 0 : group * 32);
    int phase = 0;
    pdl_trigger();
    if constexpr (R == 1 && !SUB) row_sum2_prepare(scratch, lane, warps);
    const int cols = (int)p.cols;
    const LnSpan span = ln_span<L, RAGGED>(p);
    Vec16<T>* ring = reinterpret_cast<Vec16<T>*>(ln_smem4) + threadIdx.x;   // this thread's slots: [stages][R][x, dy][CH], kLnThreads apart
    const TP* gamma = static_cast<const TP*>(p.gamma);
    const long long step = (long long)gridDim.x * sh.groups, first = (long long)group * gridDim.x + blockIdx.x;
    const int left = first < p.rows ? (int)((p.rows - 1 - first) / step) + 1 : 0;
    const int c_lane = span.head + lane * L, c_step = tpr * L;
    auto live = [&](int j) { return j * tpr + lane < span.packets; };
    const T* x_src = static_cast<const T*>(p.in) + first * p.cols + c_lane;
    const T* y_src = static_cast<const T*>(p.dout) + first * p.cols + c_lane;
    int to_fetch = left;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    auto fetch = [&](Vec16<T>* slot) {
        const uint32_t to = ring_at + (uint32_t)(slot - ring) * 16;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to_fetch-- > 0) {
#pragma unroll
                for (int j = 0; j < CH; ++j)
                    if (live(j)) {
                        copy16_async(to + (r * 2 * CH + j) * (kLnThreads * 16), x_src + j * c_step);
                        copy16_async(to + (r * 2 * CH + CH + j) * (kLnThreads * 16), y_src + j * c_step);
                    }
                x_src += step * p.cols;
                y_src += step * p.cols;
            } else if (r > 0) {
#pragma unroll
                for (int j = 0; j < 2 * CH; ++j) slot[(r * 2 * CH + j) * kLnThreads] = Vec16<T>{};
            }
        copy_commit();
    };
    for (int i = 0; i < sh.stages * R * 2; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (!live(j)) ring[(i * CH + j) * kLnThreads] = Vec16<T>{};
    for (int i = 0; i < sh.stages; ++i) fetch(ring + i * R * 2 * CH * kLnThreads);
    float mean_n[R], rstd_n[R];   // of the next rows, read in time; zero for rows that are not there
    const float *mean_at = p.mean + first, *rstd_at = p.rstd + first;
    auto statistics = [&](int i) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean_n[r] = rstd_n[r] = 0.0f;
            if (i + r < left) {
                mean_n[r] = *mean_at;
                rstd_n[r] = *rstd_at;
            }
            mean_at += step;
            rstd_at += step;
        }
    };
    statistics(0);
    // single columns of the next rows, zero where there are none
    const LnSingles one = ln_singles(span, lane);
    T next_x[R][2], next_y[R][2];
    auto singles = [&](int i) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                next_x[r][k] = next_y[r][k] = Elem<T>::from_f32(0.0f);
                if (one.have[k] && i + r < left) {
                    const long long at = (first + (i + r) * step) * p.cols + one.col[k];
                    next_x[r][k] = static_cast<const T*>(p.in)[at];
                    next_y[r][k] = static_cast<const T*>(p.dout)[at];
                }
            }
    };
    float g1[2] = {1.0f, 1.0f}, dg1[2] = {0.0f, 0.0f}, db1[2] = {0.0f, 0.0f};
    if constexpr (RAGGED) {
        singles(0);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (one.have[k] && gamma) g1[k] = Elem<TP>::to_f32(gamma[one.col[k]]);
    }
    const float inv_cols = 1.0f / (float)cols;
    float2 dg[CH][L / 2], db[CH][L / 2], g[KEEP ? CH : 1][L / 2];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
#pragma unroll
        for (int l = 0; l < L / 2; ++l) dg[j][l] = db[j][l] = make_float2(0.0f, 0.0f);
        if (KEEP) ln_param<TP, L, RAGGED>(live(j) ? gamma : nullptr, c_lane + j * c_step, 1.0f, g[KEEP ? j : 0]);
    }
    T* dst = static_cast<T*>(p.out) + first * p.cols + c_lane;
    int stage = 0;
    for (int i = 0; i < left; i += R) {
        Vec16<T>* slot = ring + stage * R * 2 * CH * kLnThreads;
        stage = stage + 1 == sh.stages ? 0 : stage + 1;
        float mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = mean_n[r];
            rstd[r] = rstd_n[r];
        }
        statistics(i + R);
        ln_wait(sh.stages);
        constexpr int K = KEEP ? CH : 1;   // packets held at a time
        float2 h[R][K][L / 2], t[R][K][L / 2];
        // x and dy of packets j0 .. j0 + K - 1 of row r, into h and t
        auto read = [&](int r, int j0) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                ln_pairs<T>(slot[(r * 2 * CH + j0 + j) * kLnThreads], h[r][j]);
                ln_pairs<T>(slot[(r * 2 * CH + CH + j0 + j) * kLnThreads], t[r][j]);
            }
        };
        // What is not there has x = dy = 0 and so adds nothing: to the sums over rows as dy, to the sums over columns as g.
        LnSums<2 * R> s;   // sum(g), sum(g h) of each row
        if (KEEP) {
#pragma unroll
            for (int r = 0; r < R; ++r) read(r, 0);
            fetch(slot);
        }
        float e_h[R][2], e_t[R][2];
        if constexpr (RAGGED) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    e_h[r][k] = Elem<T>::to_f32(next_x[r][k]);
                    e_t[r][k] = Elem<T>::to_f32(next_y[r][k]);
                }
            singles(i + R);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float2 neg_mean = make_float2(-mean[r], -mean[r]), rstd2 = make_float2(rstd[r], rstd[r]);
            float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                constexpr int Z = KEEP ? 1 : 0;
                if (!KEEP) {
                    read(r, j);
                    ln_param<TP, L, RAGGED>(live(j) ? gamma : nullptr, c_lane + j * c_step, 1.0f, g[0]);
                }
#pragma unroll
                for (int l = 0; l < L / 2; ++l) {
                    float2 &hl = h[r][j * Z][l], &tl = t[r][j * Z][l];
                    hl = __fmul2_rn(__fadd2_rn(hl, neg_mean), rstd2);
                    dg[j][l] = __ffma2_rn(tl, hl, dg[j][l]);
                    db[j][l] = __fadd2_rn(db[j][l], tl);
                    tl = __fmul2_rn(tl, g[j * Z][l]);
                    s1 = __fadd2_rn(s1, tl);
                    s2 = __ffma2_rn(tl, hl, s2);
                }
            }
            if constexpr (RAGGED) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    e_h[r][k] = (e_h[r][k] - mean[r]) * rstd[r];
                    dg1[k] = fmaf(e_t[r][k], e_h[r][k], dg1[k]);
                    db1[k] += e_t[r][k];
                    e_t[r][k] *= g1[k];
                }
                s1 = __fadd2_rn(s1, make_float2(e_t[r][0], e_t[r][1]));
                s2 = __ffma2_rn(make_float2(e_t[r][0], e_t[r][1]), make_float2(e_h[r][0], e_h[r][1]), s2);
            }
            s.v[2 * r] = s1.x + s1.y;
            s.v[2 * r + 1] = s2.x + s2.y;
        }
        if constexpr (R == 1) row_sum2<SUB>(s, scratch, phase, group + 1, warps, lane >> 5);
        else row_sum<SUB>(s, scratch, phase, group + 1, warps);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r == 0 || i + r < left) {
                const float a = -rstd[r] * (s.v[2 * r] * inv_cols), b = -rstd[r] * (s.v[2 * r + 1] * inv_cols);
                const float2 a2 = make_float2(a, a), b2 = make_float2(b, b), neg_mean = make_float2(-mean[r], -mean[r]),
                             rstd2 = make_float2(rstd[r], rstd[r]);
                if (p.out) {
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        constexpr int Z = KEEP ? 1 : 0;
                        if constexpr (!KEEP) {
                            read(r, j);
                            ln_param<TP, L, RAGGED>(live(j) ? gamma : nullptr, c_lane + j * c_step, 1.0f, g[0]);
#pragma unroll
                            for (int l = 0; l < L / 2; ++l) {
                                h[0][0][l] = __fmul2_rn(__fadd2_rn(h[0][0][l], neg_mean), rstd2);
                                t[0][0][l] = __fmul2_rn(t[0][0][l], g[0][l]);
                            }
                        }
                        float2 f[L / 2];
#pragma unroll
                        for (int l = 0; l < L / 2; ++l) f[l] = __ffma2_rn(t[r][j * Z][l], rstd2, __ffma2_rn(h[r][j * Z][l], b2, a2));
                        if (live(j)) st_stream(dst + j * c_step, ln_packet<T>(f));
                    }
                    if constexpr (RAGGED) {
                        T* row0 = static_cast<T*>(p.out) + (first + (i + r) * step) * p.cols;
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (one.have[k]) row0[one.col[k]] = Elem<T>::from_f32(fmaf(e_t[r][k], rstd[r], fmaf(e_h[r][k], b, a)));
                    }
                }
                dst += step * p.cols;
            }
        if (!KEEP) fetch(slot);
    }
    if (!p.part) return;
    // this CTA's sums: the groups' registers are added in the order of the groups
    copy_wait<0>();
    float* sum = reinterpret_cast<float*>(ln_smem4);
    float* part = p.part + (long long)blockIdx.x * 2 * p.cols;
    const int width = tpr * CH * L, stride = width + 16;   // a group's columns in packets, and with its single ones
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int l = 0; l < L / 2; l += 2) {
                const float2 u = w ? db[j][l] : dg[j][l], v = w ? db[j][l + 1] : dg[j][l + 1];
                *reinterpret_cast<float4*>(sum + group * stride + (j * tpr + lane) * L + 2 * l) = make_float4(u.x, u.y, v.x, v.y);
            }
        if (RAGGED && lane < 8) {
            sum[group * stride + width + lane] = w ? db1[0] : dg1[0];
            sum[group * stride + width + 8 + lane] = w ? db1[1] : dg1[1];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += blockDim.x) {
            const int at = c < span.head ? width + c : c < span.tail0 ? c - span.head : width + 8 + c - span.tail0;
            float t = 0.0f;
            for (int q = 0; q < sh.groups; ++q) t += sum[q * stride + at];
            part[(long long)w * cols + c] = t;
        }
    }
}

// ---- rows of any length and alignment --------------------------------------------------------------
// Sums of the streaming kernels are runs of 64 terms in fp32 and the runs' sums in fp64, so that the error does not grow with the length.
// (In one fp32 chain, where equal terms round the same way every time, y of 2^20 columns was off by 4.7e-5 at |y| = 1, and dgamma of
// 60000 rows of 40000 columns by 1.0e-4 of itself.) Here a thread's N sums over its columns of a row, every 256th; add(c, s) adds
// column c's terms.
template <int N, typename F>
__device__ __forceinline__ LnSums<N> ln_long_sums(long long cols, const F& add) {
    double total[N] = {};
    long long c = threadIdx.x;
    for (; c + 63 * 256 < cols; c += 64 * 256) {
        LnSums<N> s{};
#pragma unroll 8
        for (int k = 0; k < 64; ++k) add(c + k * 256, s.v);
#pragma unroll
        for (int n = 0; n < N; ++n) total[n] += (double)s.v[n];
    }
    LnSums<N> s{};
#pragma unroll 4
    for (; c < cols; c += 256) add(c, s.v);
#pragma unroll
    for (int n = 0; n < N; ++n) s.v[n] = (float)(total[n] + (double)s.v[n]);
    return s;
}

template <typename T, typename TP>
__global__ void __launch_bounds__(256, 8) ln_fwd_stream_kernel(const __grid_constant__ LnParams p) {
    __shared__ LnSums<1> scratch[32];
    int phase = 0;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    const TP* beta = static_cast<const TP*>(p.beta);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* in = static_cast<const T*>(p.in) + row * p.cols;
        T* out = static_cast<T*>(p.out) + row * p.cols;
        LnSums<1> s = ln_long_sums<1>(p.cols, [&](long long c, float* v) { v[0] += Elem<T>::to_f32(in[c]); });
        row_sum<false>(s, scratch, phase, 1, 8);
        const float mean = s.v[0] / (float)p.cols;
        s = ln_long_sums<1>(p.cols, [&](long long c, float* v) {
            const float d = Elem<T>::to_f32(in[c]) - mean;
            v[0] = fmaf(d, d, v[0]);
        });
        row_sum<false>(s, scratch, phase, 1, 8);
        const float rstd = rsqrtf(s.v[0] / (float)p.cols + p.eps);
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
__global__ void __launch_bounds__(256, 8) ln_bwd_stream_kernel(const __grid_constant__ LnParams p) {
    __shared__ LnSums<2> scratch[32];
    int phase = 0;
    const TP* gamma = static_cast<const TP*>(p.gamma);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.in) + row * p.cols;
        const T* y = static_cast<const T*>(p.dout) + row * p.cols;
        T* out = static_cast<T*>(p.out) + row * p.cols;
        const float mean = p.mean[row], rstd = p.rstd[row];
        LnSums<2> s = ln_long_sums<2>(p.cols, [&](long long c, float* v) {
            const float h = (Elem<T>::to_f32(x[c]) - mean) * rstd;
            const float t = Elem<T>::to_f32(y[c]) * (gamma ? Elem<TP>::to_f32(gamma[c]) : 1.0f);
            v[0] += t;
            v[1] = fmaf(t, h, v[1]);
        });
        row_sum<false>(s, scratch, phase, 1, 8);
        const float a = s.v[0] / (float)p.cols, b = s.v[1] / (float)p.cols;
        for (long long c = threadIdx.x; c < p.cols; c += 256) {
            const float h = (Elem<T>::to_f32(x[c]) - mean) * rstd;
            const float t = Elem<T>::to_f32(y[c]) * (gamma ? Elem<TP>::to_f32(gamma[c]) : 1.0f);
            out[c] = Elem<T>::from_f32(rstd * (t - a - h * b));
        }
    }
}

// The weight gradients' share of a slice of rows (blockIdx.y of gridDim.y) for 32 columns. Rows requested at once and CTAs of an SM, the
// whole backward pass: 8 and 5 300 us for 65536 x 1024 bf16 and 389 for 4096 x 20000, 8 and 6 317 and 449, 8 and 4 305 and 458, 6 and 6 303
// and 416, 4 and 6 353 and 484.
constexpr int kLnColumnsRows = 8, kLnColumnsCtas = 5;
template <typename T>
__global__ void __launch_bounds__(256, kLnColumnsCtas) ln_bwd_columns_kernel(const __grid_constant__ LnParams p) {
    __shared__ float2 sum[8][32];
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
    // runs of 64 rows in fp32 and the runs' sums in fp64, as in ln_long_sums
    const T *x = static_cast<const T*>(p.in), *dy = static_cast<const T*>(p.dout);
    const long long step = (long long)gridDim.y * 8, stride = step * p.cols;
    long long r = (long long)blockIdx.y * 8 + threadIdx.y, at = r * p.cols + c;
    long long left = c < p.cols && r < p.rows ? (p.rows - 1 - r) / step + 1 : 0;
    double total[2] = {};
    while (left > 0) {
        int run = left < 64 ? (int)left : 64;
        left -= run;
        float2 t = make_float2(0.0f, 0.0f);
        auto add = [&](float y, float v, float mean, float rstd) {
            t.x = fmaf(y, (v - mean) * rstd, t.x);
            t.y += y;
        };
        for (; run >= kLnColumnsRows; run -= kLnColumnsRows) {   // so many rows requested at once
            T xs[kLnColumnsRows], ys[kLnColumnsRows];
            float mean[kLnColumnsRows], rstd[kLnColumnsRows];
#pragma unroll
            for (int u = 0; u < kLnColumnsRows; ++u) {
                xs[u] = x[at];
                ys[u] = dy[at];
                mean[u] = p.mean[r];
                rstd[u] = p.rstd[r];
                at += stride;
                r += step;
            }
#pragma unroll
            for (int u = 0; u < kLnColumnsRows; ++u) add(Elem<T>::to_f32(ys[u]), Elem<T>::to_f32(xs[u]), mean[u], rstd[u]);
        }
#pragma unroll 1
        for (; run > 0; --run, at += stride, r += step) add(Elem<T>::to_f32(dy[at]), Elem<T>::to_f32(x[at]), p.mean[r], p.rstd[r]);
        total[0] += (double)t.x;
        total[1] += (double)t.y;
    }
    float2 s = make_float2((float)total[0], (float)total[1]);
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
__global__ void __launch_bounds__(512) ln_weight_grad_kernel(const float* part, long long parts, long long cols, TP* dgamma, TP* dbeta) {
    __shared__ float sum[16][32];
    pdl_trigger();
    pdl_wait();
    TP* out = blockIdx.y ? dbeta : dgamma;
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (out && c < cols) {
        const float* q = part + blockIdx.y * cols + c;
#pragma unroll 8
        for (long long i = threadIdx.y; i < parts; i += 16) s += q[i * 2 * cols];
    }
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && out && c < cols) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += sum[i][threadIdx.x];
        out[c] = Elem<TP>::from_f32(s);
    }
}

// CTAs that the backward pass starts at most: their sums are the workspace
static long long ln_max_parts(long long rows) {
    const long long cap = sm_count();
    return ((rows < cap ? rows : cap) + 7) / 8 * 8;
}

template <typename T, typename TP, int CH, int R, bool SUB, bool BWD>
static int ln_launch(const LnParams& p, bool ragged, int* parts, cudaStream_t s) {
    constexpr int L = Vec16<T>::N;
    const int packets = (int)(p.cols / L);   // of a row at most
    LnShape sh;
    sh.tpr = SUB ? 8 : packets == 0 ? 32 : ((packets + CH - 1) / CH + 31) / 32 * 32;
    // few rows: fewer groups per CTA, so that every SM has some
    const long long sms = sm_count(), want = (p.rows + sms - 1) / sms;
    const int most = kLnThreads / sh.tpr;
    sh.groups = (int)(want < most ? want : most);
    if (SUB) sh.groups = (sh.groups + 3) / 4 * 4;   // whole warps
    const int threads = sh.groups * sh.tpr;
    const size_t row = (size_t)R * CH * kLnThreads * 16 * (BWD ? 2 : 1);
    // Steps in shared memory, the one in work included. More rows at once upset the memory's order of service, fewer leave it idle while
    // rows are reduced. The short rows of SUB take three (524288 x 64 bf16 forward 27.4 us, with two 30.6). 16-bit rows, which compute twice
    // as much per byte, take two (65536 x 1024 bf16 forward 49.5 us, with three 51.7; 24576 x 4096 69 us, with one 74). fp32 rows take
    // one where enough threads have rows (24576 x 4096 forward 133 us and backward 192, with two 137 and 203; 16000 x 2500 backward 82 and 93),
    // two where one group leaves many threads out (6000 x 5000, 320 threads: forward 43 us and backward 63, with one 48 and 72). The borders
    // at 352 and 448 threads lie between the shapes named here; nothing nearer to them was measured.
    const bool one = sizeof(T) == 4 && (sh.groups > 1 || threads >= (BWD ? 448 : 352));
    sh.stages = SUB ? 3 : one ? 1 : 2;
    while (row * sh.stages > kLnSmem) --sh.stages;
    size_t smem = row * sh.stages;
    const size_t join = (size_t)(threads * CH * L + sh.groups * 16) * 4;
    static_assert((kLnThreads * CH * L + kLnThreads / 8 * 16) * 4 <= kLnSmem, "the join fits for every shape");
    if (BWD && smem < join) smem = join;
    long long grid = (p.rows + sh.groups - 1) / sh.groups;
    if (grid > sms) grid = sms;
    if (ragged) grid = grid >= L ? grid / L * L : L;   // down: a CTA more than fits would be a wave of its own
    if (parts) *parts = (int)grid;
    // The limit is the kernel's, not the launch's, and other host threads launch the same kernel with other shapes: every call sets the same
    // one. (Set to each call's own size, it was lowered between another thread's setting and its launch, which was then refused.)
#define CGB_LN_GO(M)                                                                                                        \
    {                                                                                                                       \
        void (*k)(const LnParams, const LnShape);                                                                           \
        if constexpr (BWD) k = ln_bwd_kernel<T, TP, CH, R, SUB, M>;                                                         \
        else k = ln_fwd_kernel<T, TP, CH, R, SUB, M>;                                                                       \
        if (smem > 32 * 1024) CGB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kLnSmem));      \
        k<<<(unsigned)grid, threads, smem, s>>>(p, sh);                                                                     \
    }
    if (ragged) CGB_LN_GO(true) else CGB_LN_GO(false)
#undef CGB_LN_GO
    CGB_CUDA(cudaGetLastError());
    return CG_B200_OK;
}

// Whether all tensors start the same number of elements behind a 16-byte boundary
static bool ln_congruent(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0; }

// The register kernels' variants: packets per thread by the length of a row. -1: none, the streaming kernels take it.
template <typename T, typename TP, bool BWD>
static int ln_registers(LnParams p, bool params_aligned, int* parts, cudaStream_t s) {
    constexpr int L = Vec16<T>::N;
    if (!ln_congruent(p.in, p.out ? p.out : p.in) || (BWD && !ln_congruent(p.in, p.dout))) return -1;
    p.off0 = (int)((reinterpret_cast<uintptr_t>(p.in) & 15) / sizeof(T));
    const bool ragged = p.off0 != 0 || p.cols % L != 0 || !params_aligned;
    const long long n = p.cols;
    // rows at a time (see the kernels): one in the backward pass, whose registers are its sums over rows, but two of up to 256 columns
    // (131072 x 256 bf16: 41 us instead of 48)
    if (n <= 64) return ln_launch<T, TP, 8 / L, BWD ? 1 : 2, true, BWD>(p, ragged, parts, s);
    if (n <= 256) return ln_launch<T, TP, 8 / L, 2, false, BWD>(p, ragged, parts, s);
    if (n <= 16 * kLnThreads) return ln_launch<T, TP, 16 / L, BWD ? 1 : 2, false, BWD>(p, ragged, parts, s);
    if (n <= 32 * kLnThreads) return ln_launch<T, TP, 32 / L, 1, false, BWD>(p, ragged, parts, s);
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
                long long slices = (long long)sm_count() * kLnColumnsCtas / tiles;
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
        CGB_CUDA(launch_pdl(ln_weight_grad_kernel<TP>, dim3((unsigned)((p.cols + 31) / 32), 2), dim3(32, 16), 0, s, (const float*)p.part,
                            (long long)parts, p.cols, static_cast<TP*>(dgamma), static_cast<TP*>(dbeta)));
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
    // what one CTA writes, another may still have to read
    const Bytes x(in, rows * cols, esz), y(out, rows * cols, esz), g(gamma, cols, psz), b(beta, cols, psz), m(mean, rows, 4), r(rstd, rows, 4);
    if ((in != out && overlap(y, x)) || overlaps_any(y, g, b, m, r) || overlaps_any(m, x, g, b, r) || overlaps_any(r, x, g, b))
        return CG_B200_ERR_INVALID_ARG;
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
    // what one CTA writes, another may still have to read. (The weight gradients are written when all inputs have been read.)
    const Bytes x(in, rows * cols, esz), dy(dout, rows * cols, esz), dx(din, rows * cols, esz), g(gamma, cols, psz), m(mean, rows, 4),
        r(rstd, rows, 4), dg(dgamma, cols, psz), db(dbeta, cols, psz), ws(dgamma || dbeta ? workspace : nullptr, (int64_t)need, 1);
    if ((din != in && overlap(dx, x)) || (din != dout && overlap(dx, dy)) || overlaps_any(dx, g, m, r, dg, db) || overlap(dg, db) ||
        overlaps_any(ws, x, dy, dx, g, m, r, dg, db))
        return CG_B200_ERR_INVALID_ARG;
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
