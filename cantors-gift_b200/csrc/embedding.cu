// embedding.cu - rows of a table by token id, scaled, and the table's gradient.
//
// The reference has no such operator on its executed path; the encoder block here takes activations, and this is what makes them.
//   forward   out[n] = scale * table[id[n]]
//   backward  dtable[v] = scale * (sum of dout[n] over the n with id[n] == v)
// An id outside [0, vocab) selects nothing: its output row is zero and its gradient is dropped, as is the padding id's gradient.
//
// Both are HBM-bound. Forward moves the rows that occur (L2 serves repeats) and the output. Backward reads dout once and writes the table
// once. It sorts the (id, n) pairs by id - a stable radix sort, so equal ids stay in the order of n, and the ids alone decide in what
// order rows are added, never the timing - and walks the sorted list in chunks of 32 pairs. A warp takes a chunk for 512 bytes of columns: it adds the rows of every id
// that begins in the chunk, in fp32 registers, following the last one into the next chunk, and writes the id's table row. Only an id
// whose pairs cover a whole chunk and reach beyond it is added by several warps: their sums go to the workspace and a last kernel joins
// them, in eight strands of every eighth chunk. The table rows that no id names are cleared beside the sort, as far as that takes no longer than the sort, and beside
// the sums.
#include <cooperative_groups.h>

#include <type_traits>

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

// Words `by` .. `by` + OUT - 1 of w, by < 4 (zero where w has no more)
template <int OUT, int IN>
__device__ __forceinline__ void shift_words(uint32_t (&w)[IN], int by) {
#pragma unroll
    for (int i = 0; i < OUT + 1 && i < IN; ++i) w[i] = by & 2 ? (i + 2 < IN ? w[i + 2 < IN ? i + 2 : 0] : 0u) : w[i];
#pragma unroll
    for (int i = 0; i < OUT && i < IN; ++i) w[i] = by & 1 ? (i + 1 < IN ? w[i + 1 < IN ? i + 1 : 0] : 0u) : w[i];
}

// A warp takes TOK tokens and STEPS * 32 packets of their rows and requests all of them before it uses the first. (A flat walk over the
// output's packets, with a division per packet, took 37 us instead of 28 for 65536 rows of 1024 bf16.)
// RAGGED: the packets are the output's, whose rows start anywhere between 16-byte boundaries; a packet's columns lie in the table between
// two other boundaries, `shift` elements on, the same for all packets of a row. So one aligned table packet more is read (L1 has it: it
// is the next lane's) and the columns are shifted out of the words. Element loads and stores took 31 us for 30000 rows of 777 bf16.
template <typename T, typename TT, typename I, bool RAGGED, int TOK, int STEPS>
__global__ void __launch_bounds__(256) emb_fwd_kernel(const __grid_constant__ EmbParams p, int segments) {
    constexpr int L = Vec16<T>::N, M = Vec16<TT>::N, R = L / M, MORE = RAGGED ? 1 : 0;   // R table packets make one output packet
    const int lane = threadIdx.x & 31, cols = (int)p.cols;
    const long long units = (p.n + TOK - 1) / TOK * segments, step = (long long)gridDim.x * 8;
    const TT* const table = static_cast<const TT*>(p.table);
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
        const long long n0 = segments == 1 ? u : u / segments;
        const int k0 = (int)(u - n0 * segments) * (32 * STEPS) + lane;
        Vec16<TT> v[TOK][STEPS][R + MORE];
        bool ok[TOK];
        int off[TOK], shift[TOK];
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            long long id = 0;
            ok[t] = n0 * TOK + t < p.n && emb_id<I>(p.ids, n0 * TOK + t, p.vocab, id);
            off[t] = shift[t] = 0;
            const TT* row = table + id * p.cols;
            if (RAGGED) {
                off[t] = (int)((reinterpret_cast<uintptr_t>(static_cast<T*>(p.out) + (n0 * TOK + t) * p.cols) & 15) / sizeof(T));
                shift[t] = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(TT) - off[t]) & (M - 1));
            }
            const int lead = off[t] + shift[t];   // packet k begins `lead` columns before column k * L of the row
            const TT* src = row + (k0 * L - lead);
            // a row far enough from the table's ends is read in whole packets, with what lies beside it
            if (!RAGGED || (id * p.cols >= L + M && (p.vocab - id) * p.cols >= p.cols + 2 * L + M)) {
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
                    if (ok[t] && (k0 + j * 32) * L < off[t] + cols) {
#pragma unroll
                        for (int r = 0; r < R + MORE; ++r) v[t][j][r] = ld_keep(src + j * 32 * L + r * M);
                    }
            } else {   // (id 0 is often the most frequent one: its first packet only is read by elements)
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
#pragma unroll
                    for (int r = 0; r < R + MORE; ++r) {
                        const int c0 = (k0 + j * 32) * L - lead + r * M;
                        const long long at = id * p.cols + c0;
                        if (ok[t] && c0 < cols && at >= 0 && at + M <= p.vocab * p.cols) {
                            v[t][j][r] = ld_keep(row + c0);
                        } else {
#pragma unroll
                            for (int l = 0; l < M; ++l)
                                v[t][j][r].v[l] = ok[t] && c0 + l >= 0 && c0 + l < cols ? row[c0 + l] : Elem<TT>::from_f32(0.0f);
                        }
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            if (n0 * TOK + t >= p.n) break;
            T* dst = static_cast<T*>(p.out) + (n0 * TOK + t) * p.cols + (k0 * L - off[t]);
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int c0 = (k0 + j * 32) * L - off[t];
                if (c0 < cols) {
                    Vec16<TT> in[R];
                    if constexpr (RAGGED) {
                        uint32_t w[(R + 1) * 4];
#pragma unroll
                        for (int i = 0; i < (R + 1) * 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(&v[t][j][i / 4])[i % 4];
                        if constexpr (sizeof(TT) == 4) {
                            shift_words<R * 4>(w, shift[t]);
                        } else {   // two elements to a word: words first, then half a word
                            shift_words<5>(w, shift[t] >> 1);
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16 * (shift[t] & 1));
                        }
#pragma unroll
                        for (int i = 0; i < R * 4; ++i) reinterpret_cast<uint32_t*>(&in[i / 4])[i % 4] = w[i];
                    } else {
#pragma unroll
                        for (int r = 0; r < R; ++r) in[r] = v[t][j][r];
                    }
                    Vec16<T> o{};
                    if (ok[t]) {   // the whole warp's token is, or is not
                        float f[L];
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            float q[M];
                            unpack16<TT>(in[r], q);
#pragma unroll
                            for (int i = 0; i < M; i += 2) {
                                const float2 v2 = __fmul2_rn(make_float2(q[i], q[i + 1]), make_float2(p.scale, p.scale));
                                f[r * M + i] = v2.x;
                                f[r * M + i + 1] = v2.y;
                            }
                        }
                        o = pack16<T>(f);
                    }
                    if (!RAGGED || (c0 >= 0 && c0 + L <= cols)) {
                        st_stream(dst + j * 32 * L, o);
                    } else {
#pragma unroll
                        for (int l = 0; l < L; ++l)
                            if (c0 + l >= 0 && c0 + l < cols) dst[j * 32 * L + l] = o.v[l];
                    }
                }
            }
        }
    }
}

template <typename T, typename TT, typename I, bool RAGGED, int TOK, int STEPS>
static void emb_forward_go(const EmbParams& p, long long per_row, cudaStream_t s) {
    const long long segments = (per_row + 32 * STEPS - 1) / (32 * STEPS);
    const long long blocks = ((p.n + TOK - 1) / TOK * segments + 7) / 8, cap = 1ll << 30;
    emb_fwd_kernel<T, TT, I, RAGGED, TOK, STEPS><<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, s>>>(p, (int)segments);
}

template <typename T, typename TT, typename I>
static int emb_forward(const EmbParams& p, cudaStream_t s) {
    constexpr int L = Vec16<T>::N;
    const bool ragged = p.cols % L != 0 || !aligned_to(p.table, 16) || !aligned_to(p.out, 16);
    const long long per_row = ragged ? (p.cols + 2 * L - 2) / L : p.cols / L;   // packets of a row at most
    // little work: less of it per warp, so that every SM has some
    const bool few = p.n * ((per_row + 31) / 32) < (long long)sm_count() * 64;
    if (ragged && few) emb_forward_go<T, TT, I, true, 1, 1>(p, per_row, s);
    else if (ragged) emb_forward_go<T, TT, I, true, 1, 4>(p, per_row, s);
    else if (few) emb_forward_go<T, TT, I, false, 1, 1>(p, per_row, s);
    else if (per_row <= 32) emb_forward_go<T, TT, I, false, 4, 1>(p, per_row, s);
    else if (per_row <= 64) emb_forward_go<T, TT, I, false, 2, 2>(p, per_row, s);
    else emb_forward_go<T, TT, I, false, 1, 4>(p, per_row, s);
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
    const uint2* in;        // pairs: key, position
    uint2* out;
    uint32_t* count;        // [tiles + 1][bins] of this pass
    uint32_t* joins;        // length of the list of joins, cleared
    long long n, vocab, padding;
    int tiles, bins, shift;
    char* zero_from;        // what the CTAs that do not sort clear meanwhile
    long long zero_bytes;
};

// Clears [from, from + bytes): thread `at` of `of`.
__device__ __forceinline__ void zero_range(char* from, long long bytes, long long at, long long of) {
    const long long to_edge = (16 - (reinterpret_cast<uintptr_t>(from) & 15)) & 15, head = to_edge < bytes ? to_edge : bytes;
    const long long packets = (bytes - head) / 16;
    for (long long i = at; i < head; i += of) from[i] = 0;
    for (long long i = head + packets * 16 + at; i < bytes; i += of) from[i] = 0;
    int4* body = reinterpret_cast<int4*>(from + head);
    for (long long i = at; i < packets; i += of) __stcs(body + i, make_int4(0, 0, 0, 0));
}

template <typename I>
__device__ __forceinline__ uint32_t sort_key(const SortParams& p, long long i) {
    const long long id = (long long)__ldg(static_cast<const I*>(p.ids) + i);
    return id < 0 || id >= p.vocab || id == p.padding ? (uint32_t)p.vocab : (uint32_t)id;
}

// The tile's digit counts; in the first pass the list of joins is cleared too. (Counting the next pass's digits in the scatter instead, by
// additions in global memory, is no faster: 262144 ids 90.7 and 92.0 us, 1M 233 and 229, 4M 835 and 824.)
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortWarps * 32) sort_count_kernel(const __grid_constant__ SortParams p) {
    __shared__ uint32_t hist[kSortBins];
    pdl_trigger();
    for (int b = threadIdx.x; b < p.bins; b += blockDim.x) hist[b] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * kSortTile;
    pdl_wait();
    for (int i = threadIdx.x; i < kSortTile; i += blockDim.x)
        if (base + i < p.n) atomicAdd(&hist[((FIRST ? sort_key<I>(p, base + i) : p.in[base + i].x) >> p.shift) & (p.bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += blockDim.x) p.count[(long long)blockIdx.x * p.bins + b] = hist[b];
    if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) *p.joins = 0;
}

// Inclusive scan over a warp
__device__ __forceinline__ uint32_t warp_scan(uint32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// Turns a pass's counts of every tile into those of the earlier tiles, in place, and leaves the bins' totals in the row behind the last
// tile. 32 bins to a CTA, the tiles in 32 runs. (Every CTA of the scatter adding up all tiles' counts itself is quadratic in their number:
// with it 4M rows of 256 bf16 took 2339 us, 1M 393, 262144 106.)
__global__ void __launch_bounds__(1024) sort_offsets_kernel(uint32_t* count, int tiles, int bins) {
    __shared__ uint32_t sum[32][33];
    pdl_trigger();
    const int bin = blockIdx.x * 32 + threadIdx.x, run = (tiles + 31) / 32;
    const int from = threadIdx.y * run, to = from + run < tiles ? from + run : tiles;
    uint32_t* const at = count + bin;
    pdl_wait();
    uint32_t s = 0;
    if (bin < bins)
#pragma unroll 8
        for (int t = from; t < to; ++t) s += at[(long long)t * bins];
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (bin >= bins) return;
    uint32_t before = 0;
    for (int y = 0; y < threadIdx.y; ++y) before += sum[y][threadIdx.x];
    if (threadIdx.y == 31) at[(long long)tiles * bins] = before + s;
    for (int t0 = from; t0 < to; t0 += 8) {   // eight reads before the first write
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = t0 + i < to ? at[(long long)(t0 + i) * bins] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (t0 + i < to) {
                at[(long long)(t0 + i) * bins] = before;
                before += c[i];
            }
    }
}

// Ranks of a warp's pairs, ROUNDS times 32 in order, among the equal digits of this warp, counted in `cnt` (one counter per bin).
// Rounds that are not there (live false in every lane) count nothing.
template <int ROUNDS, typename C>
__device__ __forceinline__ void sort_rank(C* cnt, const uint32_t (&key)[ROUNDS], const bool (&live)[ROUNDS], int shift, int bins, int lane,
                                          uint32_t (&rank)[ROUNDS]) {
    // lanes with the same digit, by a ballot for each of its bits: __match_any_sync takes a step for each different digit of the warp,
    // 1900 cycles for a round of 32 warps where the ids are well mixed
    unsigned peers[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        peers[r] = __ballot_sync(0xffffffffu, live[r]);
#pragma unroll
        for (int b = 0; b < 9; ++b)
            if ((1 << b) < bins) {
                const bool one = (key[r] >> (shift + b)) & 1;
                const unsigned with = __ballot_sync(0xffffffffu, one);
                peers[r] &= one ? with : ~with;
            }
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t digit = (key[r] >> shift) & (bins - 1);
        const int below = __popc(peers[r] & ((1u << lane) - 1u));
        uint32_t before = 0;
        if (live[r]) before = cnt[digit];
        __syncwarp();
        if (live[r] && below == 0) cnt[digit] = (C)(before + __popc(peers[r]));
        __syncwarp();
        rank[r] = before + below;
    }
}

// One pass: ranks within the tile, the tile's place in every bin from the counts of the earlier tiles, and the scatter.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortWarps * 32) sort_scatter_kernel(const __grid_constant__ SortParams p) {
    __shared__ uint32_t cnt[kSortWarps][kSortBins];
    __shared__ uint32_t base[kSortBins];
    __shared__ uint32_t warp_total[kSortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    for (int b = threadIdx.x; b < p.bins * kSortWarps; b += blockDim.x) cnt[b / p.bins][b % p.bins] = 0;
    __syncthreads();
    pdl_wait();
    const long long first = (long long)blockIdx.x * kSortTile + warp * (32 * kSortRounds);
    uint32_t key[kSortRounds], pos[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const long long i = first + r * 32 + lane;
        key[r] = 0xffffffffu;
        pos[r] = 0;
        if (i < p.n) {
            const uint2 v = FIRST ? make_uint2(sort_key<I>(p, i), (uint32_t)i) : p.in[i];
            key[r] = v.x;
            pos[r] = v.y;
        }
    }
    // thread b: bin b's pairs in all tiles and in earlier ones, as sort_offsets_kernel left them
    uint32_t total = 0, earlier = 0;
    if (threadIdx.x < p.bins) {
        total = p.count[(long long)p.tiles * p.bins + threadIdx.x];
        earlier = p.count[(long long)blockIdx.x * p.bins + threadIdx.x];
    }
    bool live[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) live[r] = first + r * 32 + lane < p.n;
    sort_rank<kSortRounds>(cnt[warp], key, live, p.shift, p.bins, lane, rank);
    const uint32_t scan = warp_scan(total, lane);
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    // where the tile's pairs of this bin start: all pairs of lower bins, then this bin's pairs of earlier tiles
    if (threadIdx.x < p.bins) {
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = cnt[w][threadIdx.x];
            cnt[w][threadIdx.x] = run;
            run += c;
        }
        uint32_t lower = 0;
        for (int w = 0; w < warp; ++w) lower += warp_total[w];
        base[threadIdx.x] = lower + scan - total + earlier;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        if (!live[r]) continue;
        const uint32_t digit = (key[r] >> p.shift) & (p.bins - 1);
        p.out[base[digit] + cnt[warp][digit] + rank[r]] = make_uint2(key[r], pos[r]);
    }
}

// Up to 16 * 8192 pairs by one cluster of CTAs, in one launch: a pass's pairs go from registers through the shared memory of the CTA
// that owns their place, and the counts of all CTAs are read there too, so nothing but the ids and the result is in global memory.
// CTA c owns the places c * span .. (c + 1) * span - 1, span = 1024 * ROUNDS; a thread holds ROUNDS pairs.
// The sort keeps sixteen SMs busy and memory idle, so the other clusters of the launch clear the end of the table's gradient meanwhile.
constexpr int kClusterWarps = 32, kClusterThreads = kClusterWarps * 32;
template <int ROUNDS> struct SortShared {
    uint2 pair[ROUNDS * kClusterThreads];     // the pairs whose places this CTA owns
    uint2 local[ROUNDS * kClusterThreads];    // its own pairs in the order of their digits: what leaves for one bin leaves in runs
    uint16_t cnt[kClusterWarps][kSortBins];
    uint32_t hist[kSortBins], start[kSortBins], warp_total[kClusterWarps];
};
// Exclusive scan over the bins: thread b's value, 0 from the threads behind the last bin.
__device__ __forceinline__ uint32_t bins_before(uint32_t v, uint32_t* warp_total, int lane, int warp) {
    const uint32_t scan = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    const uint32_t below = warp_scan(lane < kSortBins / 32 ? warp_total[lane] : 0, lane);
    return scan - v + (warp > 0 ? __shfl_sync(0xffffffffu, below, (warp - 1) & 31) : 0u);
}
template <typename I, int ROUNDS>
__global__ void __launch_bounds__(kClusterThreads) sort_cluster_kernel(const __grid_constant__ SortParams p, int passes, int digit_bits) {
    extern __shared__ float4 sort_smem4[];
    typedef SortShared<ROUNDS> Shared;
    Shared& sm = *reinterpret_cast<Shared*>(sort_smem4);
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, me = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), n = (int)p.n;
    constexpr int span = ROUNDS * kClusterThreads;
    const int place = warp * (32 * ROUNDS) + lane, first = me * span + place, mine = n - me * span < span ? n - me * span : span;
    const uint32_t low = p.bins - 1;
    const bool bin = threadIdx.x < p.bins;
    uint32_t key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
    bool live[ROUNDS];
    pdl_trigger();
    if (blockIdx.x >= ctas)
        return zero_range(p.zero_from, p.zero_bytes, (long long)(blockIdx.x - ctas) * kClusterThreads + threadIdx.x,
                          (long long)(gridDim.x - ctas) * kClusterThreads);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        live[r] = first + r * 32 < n;
        pos[r] = (uint32_t)(first + r * 32);
        key[r] = live[r] ? sort_key<I>(p, first + r * 32) : 0u;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        for (int b = threadIdx.x; b < kSortBins * kClusterWarps / 8; b += kClusterThreads) reinterpret_cast<uint4*>(sm.cnt)[b] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        sort_rank<ROUNDS>(sm.cnt[warp], key, live, shift, p.bins, lane, rank);
        __syncthreads();
        uint32_t here = 0;   // thread b: bin b's pairs of this CTA
        if (bin) {
#pragma unroll
            for (int w = 0; w < kClusterWarps; ++w) {
                const uint32_t c = sm.cnt[w][threadIdx.x];
                sm.cnt[w][threadIdx.x] = (uint16_t)here;
                here += c;
            }
            sm.hist[threadIdx.x] = here;
        }
        const uint32_t start = bins_before(here, sm.warp_total, lane, warp);
        if (bin) sm.start[threadIdx.x] = start;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (live[r]) {
                const uint32_t digit = (key[r] >> shift) & low;
                sm.local[sm.start[digit] + sm.cnt[warp][digit] + rank[r]] = make_uint2(key[r], pos[r]);
            }
        const bool last = pass + 1 == passes;
        if (ctas == 1) {   // `local` is the order of all
            __syncthreads();
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (live[r]) {
                    const uint2 v = sm.local[place + r * 32];
                    key[r] = v.x;
                    pos[r] = v.y;
                    if (last) p.out[place + r * 32] = v;
                }
            continue;
        }
        cluster.sync();   // every CTA's counts are there, and its pairs of the last pass have been taken out
        uint32_t total = 0, earlier = 0;
        if (bin)
#pragma unroll 16
            for (int c = 0; c < ctas; ++c) {
                const uint32_t v = *cluster.map_shared_rank(&sm.hist[threadIdx.x], c);
                total += v;
                if (c < me) earlier += v;
            }
        const uint32_t before = bins_before(total, sm.warp_total, lane, warp);
        if (bin) sm.start[threadIdx.x] = before + earlier - start;   // from a pair's place in `local` to its place among all
        __syncthreads();
        for (int i = threadIdx.x; i < mine; i += kClusterThreads) {
            const uint2 v = sm.local[i];
            const uint32_t to = sm.start[(v.x >> shift) & low] + i;
            if (last) p.out[to] = v;
            else *cluster.map_shared_rank(&sm.pair[to % span], to / span) = v;
        }
        cluster.sync();   // the pairs have arrived, and nobody reads this CTA's counts any more
        if (!last) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (live[r]) {
                    const uint2 v = sm.pair[place + r * 32];
                    key[r] = v.x;
                    pos[r] = v.y;
                }
        }
    }
    if (me == 0 && threadIdx.x == 0) *p.joins = 0;
}

// MB cleared beside a sort of so many rounds: what the six or so other clusters that find room write in its time (a sort of four rounds with
// 120 MB beside it took 37 us, with 78 MB 21, with none 21). Four rounds are the one point measured; the line through it for one, two and
// eight rounds is an estimate.
constexpr long long kZeroBase = 30, kZeroPerRound = 12;

// *placed: whether it was launched. Where no cluster of so many CTAs finds room at all (a partition of a GPU with few SMs to a GPC), it is not,
// and the launches over all ids sort them.
template <typename I, int ROUNDS>
static cudaError_t sort_cluster(const SortParams& p, int passes, int digit_bits, int ctas, bool* placed, cudaStream_t s) {
    auto k = sort_cluster_kernel<I, ROUNDS>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared<ROUNDS>));
    if (e == cudaSuccess && ctas > 8) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    // clusters that clear, each CTA at least 64 KB: no more than find room beside the sort, a cluster to a GPC where it has sixteen CTAs
    const long long want = p.zero_bytes / (65536ll * ctas) + (p.zero_bytes > 0), most = 96 / ctas;
    cfg.gridDim = dim3(ctas * (unsigned)(1 + (want < most ? want : most)));
    cfg.blockDim = dim3(kClusterThreads);
    cfg.dynamicSmemBytes = sizeof(SortShared<ROUNDS>);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    *placed = ctas == 1 || (cudaOccupancyMaxActiveClusters(&clusters, k, &cfg) == cudaSuccess && clusters > 0);
    if (!*placed) {
        cudaGetLastError();   // the answer may be an error; it is nobody else's
        return cudaSuccess;
    }
    return cudaLaunchKernelEx(&cfg, k, p, passes, digit_bits);
}

// ---- sums over the sorted list ---------------------------------------------------------------------------
constexpr int kChunk = 32;

struct EmbGradParams {
    const void* dout;
    const uint2* pair;     // sorted: key, position
    void* dtable;
    float* part;           // [chunks][2][cols]: a chunk's sum of an id that began before it, and of one that begins in it and is joined
    uint32_t* joins;       // how many ids are joined, and the chunks where they begin
    long long n, vocab, cols, chunks;
    long long zero_rows;   // of these rows those that no id names are still to be cleared, the rest is
    int zero_blocks;       // the first blocks clear, the others add
    float scale;
    int accumulate;
    int tiles;             // column tiles of a row
};

// The columns of a lane: NP pieces of E columns, 32 * E apart; E columns are one store of the table's type. Without vectors E is 1.
template <typename G, int E, int NP>
struct EmbLane {
    float v[NP][E];
    __device__ void clear() {
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int l = 0; l < E; ++l) v[q][l] = 0.0f;
    }
    // into row `row` of the table's gradient
    __device__ void write(const EmbGradParams& p, long long row, long long c0) const {
        G* dst = static_cast<G*>(p.dtable) + row * p.cols + c0;
#pragma unroll
        for (int q = 0; q < NP; ++q)
            if (c0 + q * 32 * E < p.cols) {
                float f[E];
#pragma unroll
                for (int l = 0; l < E; ++l) f[l] = v[q][l] * p.scale;
                if constexpr (E == 1) {
                    if (p.accumulate) f[0] += Elem<G>::to_f32(dst[q * 32]);
                    dst[q * 32] = Elem<G>::from_f32(f[0]);
                } else {
                    if (p.accumulate) {
                        float old[E];
                        unpack16<G>(*reinterpret_cast<const Vec16<G>*>(dst + q * 32 * E), old);
#pragma unroll
                        for (int l = 0; l < E; ++l) f[l] += old[l];
                    }
                    st_stream(dst + q * 32 * E, pack16<G>(f));
                }
            }
    }
    // into the workspace
    __device__ void write_part(const EmbGradParams& p, long long chunk, int slot, long long c0) const {
        float* dst = p.part + (chunk * 2 + slot) * p.cols + c0;
#pragma unroll
        for (int q = 0; q < NP; ++q)
            if (c0 + q * 32 * E < p.cols) {
                if constexpr (E == 1) {
                    dst[q * 32] = v[q][0];
                } else {
#pragma unroll
                    for (int l = 0; l < E; l += 4)
                        *reinterpret_cast<float4*>(dst + q * 32 * E + l) = make_float4(v[q][l], v[q][l + 1], v[q][l + 2], v[q][l + 3]);
                }
            }
    }
};

// Warps of a CTA of emb_grad_kernel. They share nothing, and a CTA ends with its longest: with eight of them 57344 rows of 1024 bf16 took 68 us
// in all, with four 67, alone 65 (wide rows the other way: 16384 of 4096, 127, 127 and 131).
constexpr int kEmbWarps = 1;
constexpr int kZeroRows = 8;   // of a warp at a time
// Table rows that no id names: a lane looks one row up in the sorted list, the warp zeroes those that are missing.
template <typename G>
__device__ __forceinline__ void emb_zero(const EmbGradParams& p, int lane, int warp) {
    const long long step = (long long)p.zero_blocks * kEmbWarps * kZeroRows;
    for (long long r0 = ((long long)blockIdx.x * kEmbWarps + warp) * kZeroRows; r0 < p.zero_rows; r0 += step) {
        bool missing = false;
        if (lane < kZeroRows && r0 + lane < p.zero_rows) {
            const uint32_t v = (uint32_t)(r0 + lane);
            long long lo = 0, hi = p.n;
            while (lo < hi) {
                const long long mid = (lo + hi) >> 1;
                if (p.pair[mid].x < v) lo = mid + 1;
                else hi = mid;
            }
            missing = lo == p.n || p.pair[lo].x != v;
        }
        unsigned todo = __ballot_sync(0xffffffffu, missing);
        while (todo) {
            const long long row = r0 + __ffs(todo) - 1;
            todo &= todo - 1;
            zero_range(reinterpret_cast<char*>(static_cast<G*>(p.dtable) + row * p.cols), p.cols * (long long)sizeof(G), lane, 32);
        }
    }
}

// What a warp does with its chunk: the pairs begin .. end - 1 of this chunk and the next one's are its own.
struct EmbSpan {
    uint32_t key, pos, key2, pos2;   // lane l's pair of this chunk and of the next
    unsigned long long change;       // bit i: pair i has another id than pair i - 1
    int begin, end;
    int slot;        // where the sum of the last id goes: -1 the table, 0 / 1 the workspace
    bool head_part;  // the first id's sum goes to the workspace (and it is not the last id)
    __device__ uint32_t id(int i) const { return __shfl_sync(0xffffffffu, i < kChunk ? key : key2, i & 31); }
    __device__ uint32_t at(int i) const { return __shfl_sync(0xffffffffu, i < kChunk ? pos : pos2, i & 31); }
};
__device__ __forceinline__ EmbSpan emb_span(const EmbGradParams& p, long long chunk, int lane) {
    const long long first = chunk * kChunk;
    const uint32_t none = (uint32_t)p.vocab;
    const bool here = first + lane < p.n, there = first + kChunk + lane < p.n;
    EmbSpan s;
    const uint2 v = here ? p.pair[first + lane] : make_uint2(none, 0), v2 = there ? p.pair[first + kChunk + lane] : make_uint2(none, 0);
    s.key = v.x;
    s.pos = v.y;
    s.key2 = v2.x;
    s.pos2 = v2.y;
    const uint32_t before = first > 0 ? p.pair[first - 1].x : none, before32 = first > 0 ? p.pair[first - kChunk].x : none;
    const uint32_t id0 = __shfl_sync(0xffffffffu, s.key, 0), id31 = __shfl_sync(0xffffffffu, s.key, 31);
    const uint32_t id32 = __shfl_sync(0xffffffffu, s.key2, 0), id63 = __shfl_sync(0xffffffffu, s.key2, 31);
    const uint32_t left = __shfl_up_sync(0xffffffffu, s.key, 1), left2 = __shfl_up_sync(0xffffffffu, s.key2, 1);
    s.change = __ballot_sync(0xffffffffu, lane > 0 && s.key != left) |
               (unsigned long long)__ballot_sync(0xffffffffu, s.key2 != (lane > 0 ? left2 : id31)) << 32;
    s.begin = 0;
    s.end = __popc(__ballot_sync(0xffffffffu, s.key != none));   // dropped ids are last
    s.slot = -1;
    s.head_part = false;
    const bool full = id0 == id31 && id0 != none, head = id0 == before && id0 != none;
    if (head && !full) {
        const int same = __popc(__ballot_sync(0xffffffffu, s.key == id0));
        if (before32 == id0) s.head_part = true;   // joined
        else s.begin = same;                        // the warp of the chunk before adds it
    }
    if (full && head) {
        s.slot = 0;
    } else if (id31 != none && id32 == id31) {      // the last id goes on
        const int more = __popc(__ballot_sync(0xffffffffu, s.key2 == id31));
        if (full || id63 == id31) s.slot = 1;
        else s.end += more;                         // into the next chunk, to its end
    }
    return s;
}

// The rows come through shared memory, sixteen of a warp's 512-byte pieces under way at a time: requested as register loads they would
// either cost the registers of as many packets or be waited for one by one (86 us instead of 45 for 57344 rows of 1024 bf16).
// VEC: a lane owns the columns of one store of the table's type (or two). Otherwise, for widths that no packet divides, a row's piece is
// copied as the packets that cover it, one more than it fills, and a lane owns every 32nd column and finds it behind the row's own offset.
constexpr int kEmbRows = 4, kEmbGroups = 4;   // rows of a copy group, groups in flight
template <typename T, typename G, bool VEC>
__global__ void __launch_bounds__(kEmbWarps * 32, 24 / kEmbWarps) emb_grad_kernel(const __grid_constant__ EmbGradParams p) {
    constexpr int L = Vec16<T>::N, E = !VEC ? 1 : Vec16<G>::N < L ? Vec16<G>::N : L, NP = L / E, SLOT = VEC ? 32 : 33;
    extern __shared__ float4 emb_smem4[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x < p.zero_blocks) return emb_zero<G>(p, lane, warp);
    const long long unit = (long long)(blockIdx.x - p.zero_blocks) * kEmbWarps + warp;
    const long long chunk = unit / p.tiles;
    if (chunk >= p.chunks) return;
    const long long tile0 = (unit - chunk * p.tiles) * (32 * L), c0 = tile0 + lane * E;
    const EmbSpan span = emb_span(p, chunk, lane);
    if (span.begin >= span.end) return;
    if (span.slot == 1 && tile0 == 0 && lane == 0) p.joins[1 + atomicAdd(p.joins, 1u)] = (uint32_t)chunk;   // in any order: each is joined by itself
    // a warp's ring: [groups][rows][SLOT packets]
    Vec16<T>* ring = reinterpret_cast<Vec16<T>*>(emb_smem4) + warp * (kEmbGroups * kEmbRows * SLOT);
    const T* const dout = static_cast<const T*>(p.dout);
    const int width = (int)(p.cols - tile0 < 32 * L ? p.cols - tile0 : 32 * L);
    auto offset = [&](long long pos) { return VEC ? 0 : (int)((reinterpret_cast<uintptr_t>(dout + pos * p.cols + tile0) & 15) / sizeof(T)); };
    const T* const mine = dout + tile0 + lane * L;   // of row 0
    const bool in = lane * L < width;
    auto fetch = [&](int group, int i) {   // rows i .. of the span into group `group`
#pragma unroll
        for (int r = 0; r < kEmbRows; ++r)
            if (i + r < span.end) {
                const uint32_t pos = span.at(i + r);
                Vec16<T>* to = ring + (group * kEmbRows + r) * SLOT;
                if constexpr (VEC) {
                    if (in) copy16_async(to + lane, mine + (long long)pos * p.cols);
                } else {
                    const int off = offset(pos);
                    const T* from = dout + pos * p.cols + tile0 - off;
                    for (int k = lane; k * L < off + width; k += 32) {
                        const T* src = from + k * L;
                        if (src >= dout && src + L <= dout + p.n * p.cols) {
                            copy16_async(to + k, src);
                        } else {   // the packets at the tensor's ends: only what is inside
                            Vec16<T> v;
#pragma unroll
                            for (int l = 0; l < L; ++l) v.v[l] = src + l >= dout && src + l < dout + p.n * p.cols ? src[l] : Elem<T>::from_f32(0.0f);
                            to[k] = v;
                        }
                    }
                }
            }
        copy_commit();
    };
#pragma unroll
    for (int g = 0; g < kEmbGroups; ++g) fetch(g, span.begin + g * kEmbRows);
    EmbLane<G, E, NP> acc;
    acc.clear();
    uint32_t cur = span.id(span.begin);
    bool head_part = span.head_part;
    const unsigned long long change = span.change & ~(1ull << span.begin);   // the first pair of all begins nothing new
    auto add = [&](int i, const Vec16<T>* slot) {   // pair i, whose piece is in `slot`
        if (change >> i & 1) {
            if (head_part) acc.write_part(p, chunk, 0, c0);
            else acc.write(p, cur, c0);
            head_part = false;
            cur = span.id(i);
            acc.clear();
        }
        const T* row = reinterpret_cast<const T*>(slot) + (VEC ? 0 : offset(span.at(i))) + lane * E;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if constexpr (E == 1) {
                acc.v[q][0] += Elem<T>::to_f32(row[q * 32]);   // (behind the row's end: what is there, added to a column that is not written)
            } else {
                Vec16<T> v;
                if constexpr (NP == 1) v = *reinterpret_cast<const Vec16<T>*>(row);
                else *reinterpret_cast<int2*>(&v) = *reinterpret_cast<const int2*>(row + q * 32 * E);   // half a packet
                float t[L];
                unpack16<T>(v, t);
#pragma unroll
                for (int l = 0; l < E; l += 2) {
                    const float2 a = __fadd2_rn(make_float2(acc.v[q][l], acc.v[q][l + 1]), make_float2(t[l], t[l + 1]));
                    acc.v[q][l] = a.x;
                    acc.v[q][l + 1] = a.y;
                }
            }
        }
    };
    int group = 0;
    for (int i0 = span.begin; i0 < span.end; i0 += kEmbRows) {
        copy_wait<kEmbGroups - 1>();
        __syncwarp();
        const Vec16<T>* slot = ring + group * (kEmbRows * SLOT);
        if (i0 + kEmbRows <= span.end) {
#pragma unroll
            for (int r = 0; r < kEmbRows; ++r) add(i0 + r, slot + r * SLOT);
        } else {
            for (int r = 0; i0 + r < span.end; ++r) add(i0 + r, slot + r * SLOT);
        }
        __syncwarp();
        fetch(group, i0 + kEmbGroups * kEmbRows);
        group = group + 1 == kEmbGroups ? 0 : group + 1;
    }
    if (head_part) acc.write_part(p, chunk, 0, c0);
    else if (span.slot >= 0) acc.write_part(p, chunk, span.slot, c0);
    else acc.write(p, cur, c0);
}

// Joins the sums of an id over the chunks that it covers: a CTA per id and 32 * E columns, eight strands of sums, each in order.
template <typename G, int E>
__global__ void __launch_bounds__(256) emb_join_kernel(const __grid_constant__ EmbGradParams p) {
    __shared__ float sum[8][32 * E + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    const long long tiles = (p.cols + 32 * E - 1) / (32 * E), units = (long long)p.joins[0] * tiles;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const long long chunk = p.joins[1 + u / tiles], c = u % tiles * (32 * E) + lane * E;
        const uint32_t id = p.pair[chunk * kChunk + kChunk - 1].x;
        // the chunk with the id's last pair: chunk `last` begins with a pair of the id, chunk `hi` does not; 32 probes per step
        long long last = chunk + 1, hi = p.chunks;
        for (long long span = 1; hi - last > 1; span = (hi - last + 31) / 32) {   // the next 32 chunks first, where most ids end
            const long long at = last + span * (lane + 1);
            const int passed = __popc(__ballot_sync(0xffffffffu, at < hi && p.pair[at * kChunk].x == id));
            const long long beyond = last + span * (passed + 1);
            last += span * passed;
            if (passed < 32 && beyond < hi) hi = beyond;
        }
        float s[E];
#pragma unroll
        for (int l = 0; l < E; ++l) s[l] = 0.0f;
        auto add = [&](const float* from) {
            if constexpr (E == 4) {
                const float4 t = *reinterpret_cast<const float4*>(from);
                s[0] += t.x; s[1] += t.y; s[2] += t.z; s[3] += t.w;
            } else {
                s[0] += *from;
            }
        };
        if (c < p.cols) {
            if (warp == 0) add(p.part + (chunk * 2 + 1) * p.cols + c);
#pragma unroll 8
            for (long long k = chunk + 1 + warp; k <= last; k += 8) add(p.part + k * 2 * p.cols + c);
        }
        __syncthreads();
#pragma unroll
        for (int l = 0; l < E; ++l) sum[warp][lane * E + l] = s[l];
        __syncthreads();
        const long long cc = u % tiles * (32 * E) + threadIdx.x;
        if (threadIdx.x < 32 * E && cc < p.cols) {
            float f = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) f += sum[w][threadIdx.x];
            G* dst = static_cast<G*>(p.dtable) + (long long)id * p.cols + cc;
            f *= p.scale;
            if (p.accumulate) f += Elem<G>::to_f32(*dst);
            *dst = Elem<G>::from_f32(f);
        }
    }
}

// Parts of the workspace, each 256-byte aligned
struct EmbWorkspace {
    size_t pair[2], count, joins, part, bytes;
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
    for (int i = 0; i < 2; ++i) w.pair[i] = take((size_t)n * 8);
    w.count = take((((size_t)w.tiles + 1) << w.digit_bits) * 4);
    w.joins = take((size_t)(w.chunks + 1) * 4);
    w.part = take((size_t)w.chunks * 2 * (size_t)cols * 4);
    w.bytes = at;
    return w;
}

template <typename I>
static int emb_sort(const EmbWorkspace& w, char* ws, const void* ids, long long n, long long vocab, long long padding, void* dtable,
                    long long row_bytes, long long* zero_rows, int* result, cudaStream_t s) {
    SortParams p{};
    p.ids = ids;
    p.n = n;
    p.vocab = vocab;
    p.padding = padding;
    p.tiles = w.tiles;
    p.bins = 1 << w.digit_bits;
    p.joins = reinterpret_cast<uint32_t*>(ws + w.joins);
    constexpr int kRound = kClusterThreads;   // pairs of a round of one CTA
    if (n <= 16 * 8 * kRound) {
        // as many CTAs as have a round to do, then as few rounds as sixteen CTAs leave
        p.out = reinterpret_cast<uint2*>(ws + w.pair[0]);
        int ctas = 1, rounds = 1;
        while (ctas < 16 && ctas * kRound < n) ctas *= 2;
        while (rounds * ctas * kRound < n) rounds *= 2;
        // rows to clear meanwhile: what memory takes in the time of the sort
        const long long fit = ((kZeroBase + kZeroPerRound * rounds) << 20) / row_bytes, rows = fit < *zero_rows ? fit : *zero_rows;
        p.zero_from = static_cast<char*>(dtable) + (*zero_rows - rows) * row_bytes;
        p.zero_bytes = rows * row_bytes;
        bool placed = false;
        switch (rounds) {
            case 1: CGB_CUDA((sort_cluster<I, 1>(p, w.passes, w.digit_bits, ctas, &placed, s))); break;
            case 2: CGB_CUDA((sort_cluster<I, 2>(p, w.passes, w.digit_bits, ctas, &placed, s))); break;
            case 4: CGB_CUDA((sort_cluster<I, 4>(p, w.passes, w.digit_bits, ctas, &placed, s))); break;
            default: CGB_CUDA((sort_cluster<I, 8>(p, w.passes, w.digit_bits, ctas, &placed, s)));
        }
        if (placed) {
            *zero_rows -= rows;
            *result = 0;
            return CG_B200_OK;
        }
    }
    p.count = reinterpret_cast<uint32_t*>(ws + w.count);
    int cur = 0;
    for (int pass = 0; pass < w.passes; ++pass) {
        p.shift = pass * w.digit_bits;
        p.in = reinterpret_cast<const uint2*>(ws + w.pair[cur]);
        p.out = reinterpret_cast<uint2*>(ws + w.pair[cur ^ 1]);
        if (pass == 0) sort_count_kernel<I, true><<<w.tiles, kSortWarps * 32, 0, s>>>(p);
        else CGB_CUDA(launch_pdl(sort_count_kernel<I, false>, w.tiles, kSortWarps * 32, 0, s, p));
        CGB_CUDA(launch_pdl(sort_offsets_kernel, (p.bins + 31) / 32, dim3(32, 32), 0, s, p.count, p.tiles, p.bins));
        CGB_CUDA(launch_pdl(pass == 0 ? sort_scatter_kernel<I, true> : sort_scatter_kernel<I, false>, w.tiles, kSortWarps * 32, 0, s, p));
        CGB_CUDA(cudaGetLastError());
        cur ^= 1;
    }
    *result = cur;
    return CG_B200_OK;
}

// Column tiles of a row of packets of `packet` elements, and whether a grid holds all chunks' tiles and the blocks that clear
constexpr long long kZeroBlocks = 1 << 20;   // of those at most
static long long emb_tiles(long long cols, int packet) { return (cols + 32 * packet - 1) / (32 * packet); }
static bool emb_grid_ok(long long chunks, long long cols, int dtype) {
    return chunks * emb_tiles(cols, 16 / (int)dtype_bytes(dtype)) <= 0x7fffffffll - kZeroBlocks;
}

template <typename T, typename G>
static int emb_backward(EmbGradParams p, cudaStream_t s) {
    constexpr int L = Vec16<T>::N;
    const bool vec = p.cols % L == 0 && aligned_to(p.dout, 16) && aligned_to(p.dtable, 16);
    p.tiles = (int)emb_tiles(p.cols, L);
    const long long most = (long long)sm_count() * 256 / kEmbWarps, zero_cap = most < kZeroBlocks ? most : kZeroBlocks, want = (p.zero_rows + kEmbWarps * kZeroRows - 1) / (kEmbWarps * kZeroRows);
    p.zero_blocks = (int)(want < zero_cap ? want : zero_cap);
    const long long blocks = (p.chunks * p.tiles + kEmbWarps - 1) / kEmbWarps + p.zero_blocks;   // fit a grid, see emb_grid_ok
    auto k = vec ? emb_grad_kernel<T, G, true> : emb_grad_kernel<T, G, false>;
    const int smem = kEmbWarps * kEmbGroups * kEmbRows * (vec ? 32 : 33) * 16;
    if (blocks > 0) {
        CGB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        CGB_CUDA(launch_pdl(k, (unsigned)blocks, kEmbWarps * 32, smem, s, p));
    }
    if (p.n > kChunk) {   // fewer cannot cover a chunk and reach beyond it
        const int e = p.cols % 4 == 0 ? 4 : 1;
        const long long units = p.chunks * ((p.cols + 32 * e - 1) / (32 * e)), cap = (long long)sm_count() * 8;
        CGB_CUDA(launch_pdl(e == 4 ? emb_join_kernel<G, 4> : emb_join_kernel<G, 1>, (unsigned)(units < cap ? units : cap), 256, 0, s, p));
    }
    return CG_B200_OK;
}

static bool emb_sizes_ok(int64_t n, int64_t vocab, int64_t cols) {
    return n >= 0 && vocab >= 0 && cols >= 0 && n <= 0x7fffffff && vocab < 0x7fffffff && cols <= (1 << 30);
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
    if (overlaps_any(Bytes(out, n * cols, dtype_bytes(dtype)), Bytes(table, vocab * cols, dtype_bytes(table_dtype)), Bytes(ids, n, id_bytes)))
        return CG_B200_ERR_INVALID_ARG;
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
    if (!emb_grid_ok(w.chunks, cols, dtype)) return CG_B200_ERR_UNSUPPORTED;
    if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes)) return CG_B200_ERR_WORKSPACE;
    // rows of the table are cleared beside the sort, before dout is read
    const Bytes dy(dout, n * cols, dtype_bytes(dtype)), dt(dtable, vocab * cols, dtype_bytes(grad_dtype)), id(ids, n, id_bytes),
        scratch(workspace, (int64_t)w.bytes, 1);
    if (overlaps_any(dt, dy, id) || overlaps_any(scratch, dy, dt, id)) return CG_B200_ERR_INVALID_ARG;
    int st = require_sm100();
    if (st) return st;
    cudaStream_t s = (cudaStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    int sorted = 0;
    long long zero_rows = accumulate ? 0 : vocab;
    if (n > 0) {
        const long long row_bytes = cols * (long long)dtype_bytes(grad_dtype);
        st = id_bytes == 4 ? emb_sort<int32_t>(w, ws, ids, n, vocab, padding_id, dtable, row_bytes, &zero_rows, &sorted, s)
                           : emb_sort<int64_t>(w, ws, ids, n, vocab, padding_id, dtable, row_bytes, &zero_rows, &sorted, s);
        if (st) return st;
    }
    EmbGradParams p{};
    p.dout = dout;
    p.pair = reinterpret_cast<const uint2*>(ws + w.pair[sorted]);
    p.dtable = dtable;
    p.part = reinterpret_cast<float*>(ws + w.part);
    p.joins = reinterpret_cast<uint32_t*>(ws + w.joins);
    p.n = n;
    p.vocab = vocab;
    p.cols = cols;
    p.chunks = w.chunks;
    p.scale = scale;
    p.accumulate = accumulate;
    p.zero_rows = zero_rows;
    switch (dtype) {
        case CG_B200_F32: return emb_backward<float, float>(p, s);
        case CG_B200_BF16: return grad_dtype == CG_B200_F32 ? emb_backward<__nv_bfloat16, float>(p, s) : emb_backward<__nv_bfloat16, __nv_bfloat16>(p, s);
        default: return grad_dtype == CG_B200_F32 ? emb_backward<__half, float>(p, s) : emb_backward<__half, __half>(p, s);
    }
}
