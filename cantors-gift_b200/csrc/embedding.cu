// embedding.cu - rows of a table by token id, scaled, and the table's gradient.
//
// The reference has no such operator on its executed path; the encoder block here takes activations, and this is what makes them.
//   forward   out[n] = scale * table[id[n]]
//   backward  dtable[v] = scale * (sum of dout[n] over the n with id[n] == v, in the order of n)
// An id outside [0, vocab) selects nothing: its output row is zero and its gradient is dropped, as is the padding id's gradient.
//
// Both are HBM-bound. Forward moves the rows that occur (L2 serves repeats) and the output. Backward reads dout once and writes the table
// once. It sorts the (id, n) pairs by id - a stable radix sort, so equal ids stay in the order of n and the sums do not depend on
// timing - and walks the sorted list in chunks of 32 pairs: a warp adds the rows of its chunk for 512 bytes of columns in fp32
// registers and writes each table row that lies wholly inside the chunk. Sums of ids that reach over a chunk's edge go to the workspace
// and a second kernel joins them in order; the table rows that no id names are zeroed beside the sums.
#include <math.h>

#include "common.cuh"

namespace cgb {

// ---- forward ------------------------------------------------------------------------------------------
struct EmbParams {
    const void* table;
    const void* ids;
    void* out;
    long long n, vocab, cols;
    float scale;
};

template <typename I>
__device__ __forceinline__ bool emb_id(const void* ids, long long n, long long vocab, long long& id) {
    id = (long long)__ldg(static_cast<const I*>(ids) + n);
    return id >= 0 && id < vocab;
}

// A warp takes one token and up to 128 packets (four per lane, all requested before the first is used).
template <typename T, typename TT, typename I>
__global__ void __launch_bounds__(256) emb_fwd_vec_kernel(const __grid_constant__ EmbParams p, int segments) {
    constexpr int L = Vec16<T>::N, M = Vec16<TT>::N, R = L / M, U = 4;   // R table packets make one output packet
    const int lane = threadIdx.x & 31;
    const int packets = (int)(p.cols / L);
    const long long units = p.n * segments, step = (long long)gridDim.x * 8;
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
        const long long n = u / segments;
        const int k0 = (int)(u - n * segments) * (32 * U) + lane;
        long long id;
        const bool ok = emb_id<I>(p.ids, n, p.vocab, id);
        const TT* src = static_cast<const TT*>(p.table) + (ok ? id : 0) * p.cols;
        T* dst = static_cast<T*>(p.out) + n * p.cols;
        Vec16<TT> v[U][R];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (ok && k0 + j * 32 < packets) {
#pragma unroll
                for (int r = 0; r < R; ++r) v[j][r] = ld_keep(src + (long long)(k0 + j * 32) * L + r * M);
            }
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (k0 + j * 32 < packets) {
                float f[L];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float t[M];
                    unpack16<TT>(v[j][r], t);
#pragma unroll
                    for (int i = 0; i < M; ++i) f[r * M + i] = ok ? t[i] * p.scale : 0.0f;
                }
                st_stream(dst + (long long)(k0 + j * 32) * L, pack16<T>(f));
            }
    }
}

// Any width and alignment: a warp takes one token and up to 256 elements.
template <typename T, typename TT, typename I>
__global__ void __launch_bounds__(256) emb_fwd_scalar_kernel(const __grid_constant__ EmbParams p, long long segments) {
    constexpr int U = 8;
    const int lane = threadIdx.x & 31;
    const long long units = p.n * segments, step = (long long)gridDim.x * 8;
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
        const long long n = u / segments, c0 = (u - n * segments) * (32 * U) + lane;
        long long id;
        const bool ok = emb_id<I>(p.ids, n, p.vocab, id);
        const TT* src = static_cast<const TT*>(p.table) + (ok ? id : 0) * p.cols;
        T* dst = static_cast<T*>(p.out) + n * p.cols;
        float f[U];
#pragma unroll
        for (int j = 0; j < U; ++j) f[j] = ok && c0 + j * 32 < p.cols ? Elem<TT>::to_f32(src[c0 + j * 32]) * p.scale : 0.0f;
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (c0 + j * 32 < p.cols) dst[c0 + j * 32] = Elem<T>::from_f32(f[j]);
    }
}

template <typename T, typename TT, typename I>
static int emb_forward(const EmbParams& p, cudaStream_t s) {
    const bool vec = p.cols % Vec16<T>::N == 0 && p.cols < (1ll << 30) && aligned_to(p.table, 16) && aligned_to(p.out, 16);
    const long long per = vec ? 128 * Vec16<T>::N : 256, segments = (p.cols + per - 1) / per;
    const long long blocks = (p.n * segments + 7) / 8, cap = 1ll << 30;
    const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
    if (vec) emb_fwd_vec_kernel<T, TT, I><<<grid, 256, 0, s>>>(p, (int)segments);
    else emb_fwd_scalar_kernel<T, TT, I><<<grid, 256, 0, s>>>(p, segments);
    CGB_CUDA(cudaGetLastError());
    return CG_B200_OK;
}

// ---- sorting the ids ------------------------------------------------------------------------------------
// Stable least-significant-digit radix sort of 32-bit keys with their positions. Dropped ids get the key `vocab` and end up last.
// A tile is 2048 pairs; a warp owns 128 consecutive ones and takes them 32 at a time, in order, so a pair's rank within the tile is
// (equal digits in earlier warps) + (earlier rounds of this warp) + (lower lanes of this round).
constexpr int kSortTile = 2048, kSortWarps = 16, kSortRounds = kSortTile / (32 * kSortWarps), kSortBins = 512;

struct SortParams {
    const void* ids;
    const uint32_t* key_in;
    const uint32_t* pos_in;
    uint32_t* key_out;
    uint32_t* pos_out;
    uint32_t* count;        // [tiles][bins] of this pass
    uint32_t* count_next;   // of the next pass, or null
    long long n, vocab, padding;
    int tiles, bins, shift, shift_next;
};

template <typename I>
__device__ __forceinline__ uint32_t sort_key(const SortParams& p, long long i) {
    const long long id = (long long)__ldg(static_cast<const I*>(p.ids) + i);
    return id < 0 || id >= p.vocab || id == p.padding ? (uint32_t)p.vocab : (uint32_t)id;
}

// First pass only: the tile's digit counts, and a cleared table for the next pass.
template <typename I>
__global__ void __launch_bounds__(kSortWarps * 32) sort_count_kernel(const __grid_constant__ SortParams p) {
    __shared__ uint32_t hist[kSortBins];
    for (int b = threadIdx.x; b < p.bins; b += blockDim.x) hist[b] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * kSortTile;
    for (int i = threadIdx.x; i < kSortTile; i += blockDim.x)
        if (base + i < p.n) atomicAdd(&hist[(sort_key<I>(p, base + i) >> p.shift) & (p.bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += blockDim.x) {
        p.count[(long long)blockIdx.x * p.bins + b] = hist[b];
        if (p.count_next) p.count_next[(long long)blockIdx.x * p.bins + b] = 0;
    }
}

// One pass: ranks within the tile, the tile's place in every bin from the counts of all tiles, the scatter, and the next pass's counts.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortWarps * 32) sort_scatter_kernel(const __grid_constant__ SortParams p) {
    __shared__ uint32_t cnt[kSortWarps][kSortBins];
    __shared__ uint32_t base[kSortBins];
    __shared__ uint32_t warp_total[kSortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < p.bins * kSortWarps; b += blockDim.x) cnt[b / p.bins][b % p.bins] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * kSortTile + warp * (32 * kSortRounds);
    uint32_t key[kSortRounds], pos[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const long long i = first + r * 32 + lane;
        key[r] = 0xffffffffu;
        pos[r] = 0;
        if (i < p.n) {
            key[r] = FIRST ? sort_key<I>(p, i) : p.key_in[i];
            pos[r] = FIRST ? (uint32_t)i : p.pos_in[i];
        }
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const bool live = first + r * 32 + lane < p.n;
        const uint32_t digit = live ? (key[r] >> p.shift) & (p.bins - 1) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        const int below = __popc(peers & ((1u << lane) - 1u));
        uint32_t before = 0;
        if (live) before = cnt[warp][digit];
        __syncwarp();
        if (live && below == 0) cnt[warp][digit] = before + __popc(peers);
        __syncwarp();
        rank[r] = before + below;
    }
    __syncthreads();
    // thread b: bin b. Where the tile's pairs of this bin start: all pairs of lower bins, then this bin's pairs of earlier tiles.
    uint32_t total = 0, earlier = 0;
    if (threadIdx.x < p.bins) {
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = cnt[w][threadIdx.x];
            cnt[w][threadIdx.x] = run;
            run += c;
        }
#pragma unroll 8
        for (int t = 0; t < p.tiles; ++t) {
            const uint32_t c = p.count[(long long)t * p.bins + threadIdx.x];
            total += c;
            if (t < blockIdx.x) earlier += c;
        }
    }
    uint32_t scan = total;   // inclusive over the bins
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += t;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    uint32_t lower = 0;
    for (int w = 0; w < warp; ++w) lower += warp_total[w];
    if (threadIdx.x < p.bins) base[threadIdx.x] = lower + scan - total + earlier;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        if (first + r * 32 + lane < p.n) {
            const uint32_t digit = (key[r] >> p.shift) & (p.bins - 1);
            const uint32_t to = base[digit] + cnt[warp][digit] + rank[r];
            p.key_out[to] = key[r];
            p.pos_out[to] = pos[r];
            if (p.count_next) atomicAdd(&p.count_next[(long long)(to / kSortTile) * p.bins + ((key[r] >> p.shift_next) & (p.bins - 1))], 1u);
        }
    }
}

// ---- sums over the sorted list ---------------------------------------------------------------------------
constexpr int kChunk = 32;

struct EmbGradParams {
    const void* dout;
    const uint32_t* key;   // sorted
    const uint32_t* pos;
    void* dtable;
    float* part;           // [chunks][2][cols]: a chunk's sum of the id that reaches in from before it, of the id that reaches out behind it
    long long n, vocab, cols, chunks;
    long long sum_blocks;  // blocks that add; the others zero
    float scale;
    int accumulate;
    int tiles;             // column tiles of a row
};

// W columns from c0 on of table row `row` (fewer at the row's end)
template <typename G, int W, bool VEC>
__device__ __forceinline__ void emb_write(const EmbGradParams& p, long long row, long long c0, const float (&acc)[W]) {
    G* dst = static_cast<G*>(p.dtable) + row * p.cols + c0;
    if constexpr (VEC) {
        constexpr int M = Vec16<G>::N;   // M <= W: the table's gradient has the rows' type or fp32
#pragma unroll
        for (int l = 0; l < W; l += M) {
            float f[M];
#pragma unroll
            for (int i = 0; i < M; ++i) f[i] = acc[l + i] * p.scale;
            if (p.accumulate) {
                float old[M];
                unpack16<G>(*reinterpret_cast<const Vec16<G>*>(dst + l), old);
#pragma unroll
                for (int i = 0; i < M; ++i) f[i] += old[i];
            }
            st_stream(dst + l, pack16<G>(f));
        }
    } else {
#pragma unroll
        for (int l = 0; l < W; ++l) {
            const long long c = c0 + l * 32;
            if (c < p.cols) {
                float f = acc[l] * p.scale;
                if (p.accumulate) f += Elem<G>::to_f32(dst[l * 32]);
                dst[l * 32] = Elem<G>::from_f32(f);
            }
        }
    }
}

template <int W, bool VEC>
__device__ __forceinline__ void emb_write_part(const EmbGradParams& p, long long chunk, int slot, long long c0, const float (&acc)[W]) {
    float* dst = p.part + (chunk * 2 + slot) * p.cols + c0;
#pragma unroll
    for (int l = 0; l < W; ++l) {
        if constexpr (VEC) {
            if (l % 4 == 0) *reinterpret_cast<float4*>(dst + l) = make_float4(acc[l], acc[l + 1], acc[l + 2], acc[l + 3]);
        } else if (c0 + l * 32 < p.cols) {
            dst[l * 32] = acc[l];
        }
    }
}

// VEC: lane t owns the L columns of packet t of the tile; otherwise columns t, t + 32, ... (8 of them), read one by one.
template <typename T, typename G, bool VEC>
__global__ void __launch_bounds__(256) emb_grad_kernel(const __grid_constant__ EmbGradParams p) {
    constexpr int W = VEC ? Vec16<T>::N : 8, U = 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= p.sum_blocks) {
        // table rows that no id names: a lane looks one row up in the sorted list, the warp zeroes those that are missing
        const long long step = ((long long)gridDim.x - p.sum_blocks) * 8;
        for (long long r0 = (((long long)blockIdx.x - p.sum_blocks) * 8 + warp) * 32; r0 < p.vocab; r0 += step * 32) {
            bool missing = false;
            if (r0 + lane < p.vocab) {
                const uint32_t v = (uint32_t)(r0 + lane);
                long long lo = 0, hi = p.n;
                while (lo < hi) {
                    const long long mid = (lo + hi) >> 1;
                    if (__ldg(p.key + mid) < v) lo = mid + 1;
                    else hi = mid;
                }
                missing = lo == p.n || __ldg(p.key + lo) != v;
            }
            unsigned todo = __ballot_sync(0xffffffffu, missing);
            while (todo) {
                const long long row = r0 + __ffs(todo) - 1;
                todo &= todo - 1;
                G* dst = static_cast<G*>(p.dtable) + row * p.cols;
                if (VEC && p.cols % Vec16<G>::N == 0) {
                    for (long long k = lane; k < p.cols / Vec16<G>::N; k += 32) __stcs(reinterpret_cast<int4*>(dst) + k, make_int4(0, 0, 0, 0));
                } else {
                    for (long long c = lane; c < p.cols; c += 32) dst[c] = Elem<G>::from_f32(0.0f);
                }
            }
        }
        return;
    }
    const long long unit = (long long)blockIdx.x * 8 + warp;
    const long long chunk = unit / p.tiles;
    if (chunk >= p.chunks) return;
    const long long c0 = (unit - chunk * p.tiles) * (32 * W) + (VEC ? lane * W : lane);
    const bool in = c0 < p.cols;
    const long long first = chunk * kChunk;
    const int count = (int)(p.n - first < kChunk ? p.n - first : kChunk);
    const uint32_t none = (uint32_t)p.vocab;
    const uint32_t key = lane < count ? p.key[first + lane] : none;
    const uint32_t pos = lane < count ? p.pos[first + lane] : 0;
    const uint32_t before = first > 0 ? p.key[first - 1] : none;
    const uint32_t behind = first + count < p.n ? p.key[first + count] : none;
    const T* dout = static_cast<const T*>(p.dout);
    float acc[W];
#pragma unroll
    for (int l = 0; l < W; ++l) acc[l] = 0.0f;
    uint32_t cur = __shfl_sync(0xffffffffu, key, 0);
    bool head = cur == before;   // the current id began in an earlier chunk
    if (cur == none) return;     // dropped ids are last: nothing here
    for (int i0 = 0; i0 < count; i0 += U) {
        Vec16<T> raw[U];
        float one[VEC ? 1 : U][VEC ? 1 : W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = __shfl_sync(0xffffffffu, key, i0 + u);
            const T* src = dout + (long long)__shfl_sync(0xffffffffu, pos, i0 + u) * p.cols + c0;
            if (k != none && in) {
                if constexpr (VEC) {
                    raw[u] = ld_stream(src);
                } else {
#pragma unroll
                    for (int l = 0; l < W; ++l) one[u][l] = c0 + l * 32 < p.cols ? Elem<T>::to_f32(src[l * 32]) : 0.0f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = __shfl_sync(0xffffffffu, key, i0 + u);
            if (k != cur && cur != none) {
                if (in) {
                    if (head) emb_write_part<W, VEC>(p, chunk, 0, c0, acc);
                    else emb_write<G, W, VEC>(p, cur, c0, acc);
                }
                head = false;
                cur = k;
#pragma unroll
                for (int l = 0; l < W; ++l) acc[l] = 0.0f;
            }
            if (k != none && in) {
                float f[W];
                if constexpr (VEC) {
                    unpack16<T>(raw[u], f);
                } else {
#pragma unroll
                    for (int l = 0; l < W; ++l) f[l] = one[u][l];
                }
#pragma unroll
                for (int l = 0; l < W; ++l) acc[l] += f[l];
            }
        }
    }
    if (cur != none && in) {
        if (head) emb_write_part<W, VEC>(p, chunk, 0, c0, acc);
        else if (cur == behind) emb_write_part<W, VEC>(p, chunk, 1, c0, acc);
        else emb_write<G, W, VEC>(p, cur, c0, acc);
    }
}

// Joins an id's sums over the chunks it reaches across. A CTA per chunk and share of the columns; only the chunk where an id begins that
// reaches beyond it has work. A few sums are added by the warp that owns the columns, many by all eight warps of the CTA, each every
// eighth sum: the split depends on the number of sums alone.
template <typename G>
__global__ void __launch_bounds__(256) emb_join_kernel(const __grid_constant__ EmbGradParams p) {
    __shared__ float sum[8][32];
    const long long chunk = blockIdx.x, first = chunk * kChunk, end = first + kChunk;
    if (end >= p.n) return;
    const uint32_t none = (uint32_t)p.vocab, id = p.key[end - 1];
    if (id == none || p.key[end] != id) return;                             // nothing reaches out of this chunk
    if (p.key[first] == id && first > 0 && p.key[first - 1] == id) return;    // it began earlier
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the chunk with the id's last pair: chunk `last` begins with a pair of the id, chunk `hi` does not; 32 probes per step
    long long last = chunk + 1, hi = p.chunks;
    while (hi - last > 1) {
        const long long span = (hi - last + 31) / 32, at = last + span * (lane + 1);
        const int passed = __popc(__ballot_sync(0xffffffffu, at < hi && p.key[at * kChunk] == id));
        const long long beyond = last + span * (passed + 1);
        last += span * passed;
        if (beyond < hi) hi = beyond;
    }
    const bool together = last - chunk > 16;
    const int from = together ? warp : 0, step = together ? 8 : 1;
    const long long tiles = (p.cols + 31) / 32;
    for (long long t = together ? blockIdx.y : (long long)blockIdx.y * 8 + warp; t < tiles; t += (long long)gridDim.y * (together ? 1 : 8)) {
        const long long c = t * 32 + lane;
        float s = 0.0f;
        if (c < p.cols) {
            if (from == 0) s = p.part[(chunk * 2 + 1) * p.cols + c];
#pragma unroll 8
            for (long long k = chunk + 1 + from; k <= last; k += step) s += p.part[k * 2 * p.cols + c];
        }
        if (together) {
            __syncthreads();
            sum[warp][lane] = s;
            __syncthreads();
            if (warp != 0) continue;
#pragma unroll
            for (int w = 1; w < 8; ++w) s += sum[w][lane];
        }
        if (c < p.cols) {
            G* dst = static_cast<G*>(p.dtable) + (long long)id * p.cols + c;
            float f = s * p.scale;
            if (p.accumulate) f += Elem<G>::to_f32(*dst);
            *dst = Elem<G>::from_f32(f);
        }
    }
}

// Parts of the workspace, each 256-byte aligned
struct EmbWorkspace {
    size_t key[2], pos[2], count[2], part, bytes;
    long long chunks;
    int tiles, passes, digit_bits;
};

static EmbWorkspace emb_workspace(long long n, long long vocab, long long cols) {
    EmbWorkspace w{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;   // keys 0 .. vocab
    w.passes = (bits + 8) / 9;
    w.digit_bits = (bits + w.passes - 1) / w.passes;
    w.tiles = (int)((n + kSortTile - 1) / kSortTile);
    w.chunks = (n + kChunk - 1) / kChunk;
    for (int i = 0; i < 2; ++i) {
        w.key[i] = take((size_t)n * 4);
        w.pos[i] = take((size_t)n * 4);
        w.count[i] = take(((size_t)w.tiles << w.digit_bits) * 4);
    }
    w.part = take((size_t)w.chunks * 2 * (size_t)cols * 4);
    w.bytes = at;
    return w;
}

template <typename I>
static int emb_sort(const EmbWorkspace& w, char* ws, const void* ids, long long n, long long vocab, long long padding, int* result, cudaStream_t s) {
    SortParams p{};
    p.ids = ids;
    p.n = n;
    p.vocab = vocab;
    p.padding = padding;
    p.tiles = w.tiles;
    p.bins = 1 << w.digit_bits;
    int cur = 0;
    for (int pass = 0; pass < w.passes; ++pass) {
        p.shift = pass * w.digit_bits;
        p.shift_next = p.shift + w.digit_bits;
        p.count = reinterpret_cast<uint32_t*>(ws + w.count[pass & 1]);
        p.count_next = pass + 1 < w.passes ? reinterpret_cast<uint32_t*>(ws + w.count[(pass + 1) & 1]) : nullptr;
        p.key_in = reinterpret_cast<const uint32_t*>(ws + w.key[cur]);
        p.pos_in = reinterpret_cast<const uint32_t*>(ws + w.pos[cur]);
        p.key_out = reinterpret_cast<uint32_t*>(ws + w.key[cur ^ 1]);
        p.pos_out = reinterpret_cast<uint32_t*>(ws + w.pos[cur ^ 1]);
        if (pass == 0) {
            sort_count_kernel<I><<<w.tiles, kSortWarps * 32, 0, s>>>(p);
            sort_scatter_kernel<I, true><<<w.tiles, kSortWarps * 32, 0, s>>>(p);
        } else {
            if (p.count_next) CGB_CUDA(cudaMemsetAsync(p.count_next, 0, ((size_t)w.tiles << w.digit_bits) * 4, s));
            sort_scatter_kernel<I, false><<<w.tiles, kSortWarps * 32, 0, s>>>(p);
        }
        CGB_CUDA(cudaGetLastError());
        cur ^= 1;
    }
    *result = cur;
    return CG_B200_OK;
}

template <typename T, typename G>
static int emb_backward(EmbGradParams p, cudaStream_t s) {
    const bool vec = p.cols % Vec16<T>::N == 0 && p.cols % Vec16<G>::N == 0 && aligned_to(p.dout, 16) && aligned_to(p.dtable, 16);
    const long long per = vec ? 32 * Vec16<T>::N : 256;
    p.tiles = (int)((p.cols + per - 1) / per);
    p.sum_blocks = (p.chunks * p.tiles + 7) / 8;
    const long long zero_cap = (long long)sm_count() * 8, want = (p.vocab + 255) / 256;
    const long long blocks = p.sum_blocks + (p.accumulate ? 0 : want < zero_cap ? want : zero_cap);
    if (blocks > 0x7fffffffll) return CG_B200_ERR_UNSUPPORTED;
    if (blocks > 0) {
        if (vec) emb_grad_kernel<T, G, true><<<(unsigned)blocks, 256, 0, s>>>(p);
        else emb_grad_kernel<T, G, false><<<(unsigned)blocks, 256, 0, s>>>(p);
        CGB_CUDA(cudaGetLastError());
    }
    if (p.chunks > 1) {
        emb_join_kernel<G><<<dim3((unsigned)p.chunks, p.cols > 256 ? 4 : 1), 256, 0, s>>>(p);
        CGB_CUDA(cudaGetLastError());
    }
    return CG_B200_OK;
}

static bool emb_sizes_ok(int64_t n, int64_t vocab, int64_t cols) {
    return n >= 0 && vocab >= 0 && cols >= 0 && n <= 0x7fffffff && vocab < 0x7fffffff && cols <= 0x7fffffff;
}

}  // namespace cgb

extern "C" int cg_b200_embedding(int dtype, int table_dtype, const void* table, int64_t vocab, int64_t cols, const void* ids, int id_bytes,
                                 int64_t n, float scale, void* out, void* stream) {
    using namespace cgb;
    if (!dtype_ok(dtype) || (table_dtype != dtype && table_dtype != CG_B200_F32) || (id_bytes != 4 && id_bytes != 8) ||
        !emb_sizes_ok(n, vocab, cols))
        return CG_B200_ERR_INVALID_ARG;
    if (n == 0 || cols == 0) return CG_B200_OK;
    if ((!table && vocab > 0) || !ids || !out) return CG_B200_ERR_NULL_POINTER;
    if (!aligned_to(table, dtype_bytes(table_dtype)) || !aligned_to(ids, id_bytes) || !aligned_to(out, dtype_bytes(dtype)))
        return CG_B200_ERR_MISALIGNED;
    int st = require_sm100();
    if (st) return st;
    const EmbParams p{table, ids, out, n, vocab, cols, scale};
    cudaStream_t s = (cudaStream_t)stream;
#define CGB_EMB_IDS(T, TT) return id_bytes == 4 ? emb_forward<T, TT, int32_t>(p, s) : emb_forward<T, TT, int64_t>(p, s)
    switch (dtype) {
        case CG_B200_F32: CGB_EMB_IDS(float, float);
        case CG_B200_BF16:
            if (table_dtype == CG_B200_F32) CGB_EMB_IDS(__nv_bfloat16, float);
            CGB_EMB_IDS(__nv_bfloat16, __nv_bfloat16);
        default:
            if (table_dtype == CG_B200_F32) CGB_EMB_IDS(__half, float);
            CGB_EMB_IDS(__half, __half);
    }
#undef CGB_EMB_IDS
}

extern "C" int cg_b200_embedding_backward_workspace_bytes(int64_t n, int64_t vocab, int64_t cols, size_t* bytes) {
    using namespace cgb;
    if (!bytes) return CG_B200_ERR_NULL_POINTER;
    *bytes = 0;
    if (!emb_sizes_ok(n, vocab, cols)) return CG_B200_ERR_INVALID_ARG;
    *bytes = emb_workspace(n, vocab, cols).bytes;
    return CG_B200_OK;
}

extern "C" int cg_b200_embedding_backward(int dtype, int grad_dtype, const void* dout, const void* ids, int id_bytes, int64_t n, float scale,
                                          int64_t padding_id, int accumulate, void* dtable, int64_t vocab, int64_t cols, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    using namespace cgb;
    if (!dtype_ok(dtype) || (grad_dtype != dtype && grad_dtype != CG_B200_F32) || (id_bytes != 4 && id_bytes != 8) ||
        !emb_sizes_ok(n, vocab, cols))
        return CG_B200_ERR_INVALID_ARG;
    if (vocab == 0 || cols == 0 || (n == 0 && accumulate)) return CG_B200_OK;
    if (!dtable || (n > 0 && (!dout || !ids))) return CG_B200_ERR_NULL_POINTER;
    if (!aligned_to(dout, dtype_bytes(dtype)) || !aligned_to(dtable, dtype_bytes(grad_dtype)) || !aligned_to(ids, id_bytes) ||
        !aligned_to(workspace, 256))
        return CG_B200_ERR_MISALIGNED;
    const EmbWorkspace w = emb_workspace(n, vocab, cols);
    if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes)) return CG_B200_ERR_WORKSPACE;
    int st = require_sm100();
    if (st) return st;
    cudaStream_t s = (cudaStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    int sorted = 0;
    if (n > 0) {
        st = id_bytes == 4 ? emb_sort<int32_t>(w, ws, ids, n, vocab, padding_id, &sorted, s)
                           : emb_sort<int64_t>(w, ws, ids, n, vocab, padding_id, &sorted, s);
        if (st) return st;
    }
    EmbGradParams p{};
    p.dout = dout;
    p.key = reinterpret_cast<const uint32_t*>(ws + w.key[sorted]);
    p.pos = reinterpret_cast<const uint32_t*>(ws + w.pos[sorted]);
    p.dtable = dtable;
    p.part = reinterpret_cast<float*>(ws + w.part);
    p.n = n;
    p.vocab = vocab;
    p.cols = cols;
    p.chunks = w.chunks;
    p.scale = scale;
    p.accumulate = accumulate;
    switch (dtype) {
        case CG_B200_F32: return emb_backward<float, float>(p, s);
        case CG_B200_BF16: return grad_dtype == CG_B200_F32 ? emb_backward<__nv_bfloat16, float>(p, s) : emb_backward<__nv_bfloat16, __nv_bfloat16>(p, s);
        default: return grad_dtype == CG_B200_F32 ? emb_backward<__half, float>(p, s) : emb_backward<__half, __half>(p, s);
    }
}
