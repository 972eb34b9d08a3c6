// Operators on the rows of a table: rows looked up by ids and the gradient of the table, rows sorted by the
// partitions (experts) they chose, brought back with weights, and the gradients of that. They follow a search (ids to
// rows) or an assignment (partitions to rows) and precede an index (the table it is built over); the reference has
// no counterpart. All calls enqueue on the caller's stream and return; scratch is the caller's.
//
// Everything here is bound by bytes. Rows are read and written in the widest words their addresses allow (16 bytes where
// base, stride and length are multiples of it), sums are fp32 in an order that the arguments alone determine, and each
// value is rounded once, when it is stored.
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/glide_b200.h"
#include "ctx.h"

namespace glide {
namespace {

constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kMaxPartitions = 4096;   // of dispatch_rows: a counter for each and warp in shared memory
constexpr uint32_t kMaxChoices = 128;       // as many as glide_bruteforce_knn returns neighbours
constexpr uint32_t kMaxDim = 1u << 20;
constexpr uint32_t kTile = 2048;            // items of a CTA in the counting sort
constexpr uint32_t kSortThreads = 256, kSortWarps = kSortThreads / 32, kWarpItems = kTile / kSortWarps;
constexpr uint32_t kChunk = 32;             // sorted items that one group of lanes joins in the gradient

// ---- rows as words ----------------------------------------------------------------------------------------
template<int B> struct Word;
template<> struct Word<16> { using type = uint4; };
template<> struct Word<8> { using type = uint2; };
template<> struct Word<4> { using type = uint32_t; };
template<> struct Word<2> { using type = uint16_t; };
template<> struct Word<1> { using type = uint8_t; };
template<typename T, int V> using WordOf = typename Word<(int) sizeof(T) * V>::type;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(uint8_t x) { return (float) x; }
template<typename T> __device__ __forceinline__ T from_float(float x);
template<> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template<> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template<typename T, int V>
__device__ __forceinline__ void unpack(const WordOf<T, V> &w, float (&f)[V]) {
    T t[V];
    memcpy(t, &w, sizeof w);
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = to_float(t[i]);
}

// V values stored as T; fp32 values of wider groups go out in words of 16 bytes
template<typename T, int V>
__device__ __forceinline__ void store(T *p, const float (&f)[V]) {
    if constexpr (sizeof(T) * V <= 16) {
        T t[V];
#pragma unroll
        for (int i = 0; i < V; i++) t[i] = from_float<T>(f[i]);
        WordOf<T, V> w;
        memcpy(&w, t, sizeof w);
        *reinterpret_cast<WordOf<T, V> *>(p) = w;
    } else {
        constexpr int H = 16 / (int) sizeof(T);
#pragma unroll
        for (int h = 0; h < V / H; h++) {
            float g[H];
#pragma unroll
            for (int i = 0; i < H; i++) g[i] = f[h * H + i];
            store<T, H>(p + h * H, g);
        }
    }
}

template<typename T, int V>
__device__ __forceinline__ void load(const T *p, float (&f)[V]) {
    if constexpr (sizeof(T) * V <= 16) {
        unpack<T, V>(*reinterpret_cast<const WordOf<T, V> *>(p), f);
    } else {
        constexpr int H = 16 / (int) sizeof(T);
#pragma unroll
        for (int h = 0; h < V / H; h++) {
            float g[H];
            load<T, H>(p + h * H, g);
#pragma unroll
            for (int i = 0; i < H; i++) f[h * H + i] = g[i];
        }
    }
}

// Quotient by a number that is the same for a whole launch, by a multiplication (Granlund and Montgomery, 1994): exact for
// dividends below 2^31.
struct Div {
    uint32_t d, m, s;
    explicit Div(uint32_t by) : d(by), s(0) {
        while ((1ull << s) < by) s++;
        m = (uint32_t) ((((1ull << s) - by) << 32) / by + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return (__umulhi(m, x) + x) >> s; }
};

// ---- lookup -------------------------------------------------------------------------------------------------
// out[t] = scale * table[ids[t]], zeros for ids beyond the table (0xffffffff among them). A thread owns U words of the output, a
// CTA's width apart, so that U loads are in flight once the ids (which a CTA shares through L1) have come.
template<typename T, typename O, int V, int U>
__global__ void __launch_bounds__(256) lookup_kernel(const T *__restrict__ table, uint64_t table_stride, uint32_t n,
                                                     const uint32_t *__restrict__ ids, uint32_t units, Div words, float scale,
                                                     O *__restrict__ out, uint64_t out_stride) {
    const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t row[U], at[U], id[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t x = min(first + u * 256, units - 1);
        row[u] = words.of(x);
        at[u] = (x - row[u] * words.d) * V;
        id[u] = ids[row[u]];
    }
    float f[U][V];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (id[u] < n) {
            load<T, V>(table + (uint64_t) id[u] * table_stride + at[u], f[u]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) f[u][i] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (first + u * 256 >= units) break;
#pragma unroll
        for (int i = 0; i < V; i++) f[u][i] = id[u] < n ? f[u][i] * scale : 0.0f;
        store<O, V>(out + (uint64_t) row[u] * out_stride + at[u], f[u]);
    }
}

// ---- stable counting sort -------------------------------------------------------------------------------------
// One pass places every item behind all items of a smaller digit and behind the items of its own digit that came before it.
// count: a CTA takes kTile consecutive items, each of its warps a run of them 32 at a time; a lane's rank among the items of
// its digit is the warp's running count plus the equal digits at lower lanes, and a scan over the warps' counts makes it the
// rank in the CTA. scan: the counts of all CTAs become, digit by digit, counts of the CTAs before. No atomics: the order
// depends on nothing but the keys.
struct Digit {
    uint32_t limit, shift, mask;   // keys beyond limit count as limit
    __device__ __forceinline__ uint32_t of(uint32_t key) const { return (min(key, limit) >> shift) & mask; }
};

__global__ void __launch_bounds__(kSortThreads) bucket_count_kernel(const uint32_t *__restrict__ keys, uint32_t items, Digit digit,
                                                                    uint32_t buckets, uint32_t *__restrict__ counts,
                                                                    uint16_t *__restrict__ ranks) {
    extern __shared__ uint16_t warp_counts[];   // kSortWarps x buckets
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    for (uint32_t i = threadIdx.x; i < kSortWarps * buckets; i += kSortThreads) warp_counts[i] = 0;
    __syncthreads();
    uint16_t *mine = warp_counts + warp * buckets;
    const uint32_t first = blockIdx.x * kTile + warp * kWarpItems;
    uint32_t d[kWarpItems / 32], rank[kWarpItems / 32];
#pragma unroll
    for (uint32_t r = 0; r < kWarpItems / 32; r++) {
        const uint32_t i = first + r * 32 + lane;
        d[r] = i < items ? digit.of(keys[i]) : kNone;
    }
#pragma unroll
    for (uint32_t r = 0; r < kWarpItems / 32; r++) {
        const uint32_t same = __match_any_sync(0xffffffffu, d[r]);
        const bool there = d[r] != kNone;
        const uint32_t before = there ? mine[d[r]] : 0;
        rank[r] = before + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (there && (same >> lane) == 1u) mine[d[r]] = (uint16_t) (before + __popc(same));
        __syncwarp();
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += kSortThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSortWarps; w++) {
            const uint32_t c = warp_counts[w * buckets + b];
            warp_counts[w * buckets + b] = (uint16_t) sum;
            sum += c;
        }
        counts[(uint64_t) blockIdx.x * buckets + b] = sum;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kWarpItems / 32; r++) {
        const uint32_t i = first + r * 32 + lane;
        if (i < items) ranks[i] = (uint16_t) (mine[d[r]] + rank[r]);
    }
}

__global__ void __launch_bounds__(1024) bucket_scan_kernel(uint32_t *__restrict__ counts, uint32_t tiles, uint32_t buckets,
                                                           uint32_t *__restrict__ totals) {
    __shared__ uint32_t part[32][33];
    const uint32_t x = threadIdx.x & 31u, y = threadIdx.x >> 5;
    const uint32_t b = blockIdx.x * 32 + x;
    const uint32_t each = (tiles + 31) / 32, t0 = min(y * each, tiles), t1 = min(t0 + each, tiles);
    uint32_t sum = 0;
    if (b < buckets)
        for (uint32_t t = t0; t < t1; t++) sum += counts[(uint64_t) t * buckets + b];
    part[y][x] = sum;
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t i = 0; i < y; i++) run += part[i][x];
    if (b < buckets) {
        for (uint32_t t = t0; t < t1; t++) {
            const uint32_t c = counts[(uint64_t) t * buckets + b];
            counts[(uint64_t) t * buckets + b] = run;
            run += c;
        }
        if (y == 31) totals[b] = run;
    }
}

// The first place of every bucket, from the buckets' totals, into shared memory; every thread of the CTA calls it.
template<uint32_t kThreads>
__device__ __forceinline__ void bucket_starts(const uint32_t *__restrict__ totals, uint32_t buckets, uint32_t *starts) {
    __shared__ uint32_t warp_sum[kThreads / 32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t each = (buckets + kThreads - 1) / kThreads, b0 = min(threadIdx.x * each, buckets), b1 = min(b0 + each, buckets);
    uint32_t sum = 0;
    for (uint32_t b = b0; b < b1; b++) sum += totals[b];
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= (uint32_t) off) incl += o;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    uint32_t run = incl - sum;
    for (uint32_t w = 0; w < warp; w++) run += warp_sum[w];
    for (uint32_t b = b0; b < b1; b++) {
        starts[b] = run;
        run += totals[b];
    }
    __syncthreads();
}

// The items of one pass in their new places. values == nullptr: an item's value is its index.
__global__ void __launch_bounds__(kSortThreads) bucket_scatter_kernel(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ values,
                                                                      uint32_t items, Digit digit, uint32_t buckets,
                                                                      const uint32_t *__restrict__ before, const uint32_t *__restrict__ totals,
                                                                      const uint16_t *__restrict__ ranks, uint32_t *__restrict__ keys_out,
                                                                      uint32_t *__restrict__ values_out) {
    extern __shared__ uint32_t starts[];
    bucket_starts<kSortThreads>(totals, buckets, starts);
#pragma unroll
    for (uint32_t r = 0; r < kTile / kSortThreads; r++) {
        const uint32_t i = blockIdx.x * kTile + r * kSortThreads + threadIdx.x;
        if (i >= items) break;
        const uint32_t key = min(keys[i], digit.limit), d = digit.of(key);
        const uint32_t p = starts[d] + before[(uint64_t) blockIdx.x * buckets + d] + ranks[i];
        keys_out[p] = key;
        values_out[p] = values ? values[i] : i;
    }
}

// ---- gradient of a lookup ---------------------------------------------------------------------------------------
struct GradArgs {
    const uint32_t *keys, *values;   // sorted by id: the id, and the row of grad_out
    uint32_t items, n, dim, words, lanes, slabs;
    float scale;
    uint64_t in_stride, out_stride;
    int accumulate;
    float *partial;                  // (2 * chunk + which) * dim: sums of runs that leave their chunk
};

template<typename O, int V>
__device__ __forceinline__ void put_grad(O *out, const GradArgs &a, uint32_t id, uint32_t at, float (&acc)[V]) {
    O *p = out + (uint64_t) id * a.out_stride + at;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] *= a.scale;
    if (a.accumulate) {
        float old[V];
        load<O, V>(p, old);
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += old[i];
    }
    store<O, V>(p, acc);
}

// A group of lanes joins kChunk sorted items over a slab of the row: the sum of a run of equal ids goes to the id's row, or,
// where the run goes on in another chunk, to the chunk's partial sums (first: it came from the chunk before).
template<typename T, typename O, int V>
__global__ void __launch_bounds__(256) grad_join_kernel(const T *__restrict__ grad, O *__restrict__ out, GradArgs a) {
    constexpr int U = 8;
    const uint32_t group = (blockIdx.x * 256 + threadIdx.x) / a.lanes, lane = threadIdx.x & (a.lanes - 1);
    const uint32_t chunk = group / a.slabs, word = (group - chunk * a.slabs) * a.lanes + lane;
    const uint32_t c0 = chunk * kChunk;
    if (c0 >= a.items || word >= a.words) return;
    const uint32_t c1 = min(c0 + kChunk, a.items), at = word * V;
    uint32_t id = a.keys[c0];
    bool from_left = c0 > 0 && a.keys[c0 - 1] == id;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    auto put = [&](bool to_right) {
        if (id >= a.n) return;
        if (from_left || to_right) store<float, V>(a.partial + (uint64_t) (2 * chunk + (from_left ? 0 : 1)) * a.dim + at, acc);
        else put_grad<O, V>(out, a, id, at, acc);
    };
    for (uint32_t c = c0; c < c1; c += U) {
        uint32_t key[U];
        float f[U][V];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = min(c + u, c1 - 1);
            key[u] = a.keys[i];
            if (key[u] < a.n) load<T, V>(grad + (uint64_t) a.values[i] * a.in_stride + at, f[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c + u >= c1) break;
            if (key[u] != id) {
                put(false);
                id = key[u];
                from_left = false;
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] = 0.0f;
            }
            if (id < a.n) {
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += f[u][i];
            }
        }
    }
    put(c1 < a.items && a.keys[c1] == id);
}

// Runs over several chunks: whoever holds the chunk that a run starts in adds the partial sums in order.
template<typename O, int V>
__global__ void __launch_bounds__(256) grad_fix_kernel(O *__restrict__ out, GradArgs a) {
    const uint32_t group = (blockIdx.x * 256 + threadIdx.x) / a.lanes, lane = threadIdx.x & (a.lanes - 1);
    const uint32_t chunk = group / a.slabs, word = (group - chunk * a.slabs) * a.lanes + lane;
    const uint32_t c0 = chunk * kChunk, c1 = c0 + kChunk;
    if (c1 >= a.items || word >= a.words) return;
    const uint32_t id = a.keys[c1 - 1], at = word * V;
    if (id >= a.n || a.keys[c1] != id || (a.keys[c0] == id && c0 > 0 && a.keys[c0 - 1] == id)) return;
    float acc[V];
    load<float, V>(a.partial + (uint64_t) (2 * chunk + 1) * a.dim + at, acc);
    for (uint32_t c = chunk + 1;; c++) {
        float f[V];
        load<float, V>(a.partial + (uint64_t) (2 * c) * a.dim + at, f);
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += f[i];
        if ((c + 1) * kChunk >= a.items || a.keys[(c + 1) * kChunk] != id) break;
    }
    put_grad<O, V>(out, a, id, at, acc);
}

// ---- dispatch ---------------------------------------------------------------------------------------------------
// A CTA places the pairs of a few rows (place = start of the partition + pairs of earlier tiles + rank in the tile), then copies
// each of its rows, read once, to the places of its pairs.
template<int B>
__global__ void __launch_bounds__(256) dispatch_kernel(const uint8_t *__restrict__ rows, uint64_t stride, uint32_t count, uint32_t words,
                                                       const uint32_t *__restrict__ choice, uint32_t choices, uint32_t partitions,
                                                       const uint32_t *__restrict__ before, const uint32_t *__restrict__ totals,
                                                       const uint16_t *__restrict__ ranks, uint32_t rows_each, uint8_t *__restrict__ sorted,
                                                       uint64_t sorted_stride, uint32_t *__restrict__ position, uint32_t *__restrict__ map,
                                                       uint32_t *__restrict__ segment_start) {
    using W = typename Word<B>::type;
    extern __shared__ uint32_t smem[];
    uint32_t *starts = smem, *place = smem + partitions + 1;
    bucket_starts<256>(totals, partitions + 1, starts);
    if (blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i <= partitions; i += 256) segment_start[i] = starts[i];
    const uint32_t r0 = blockIdx.x * rows_each, nr = min(rows_each, count - r0);
    for (uint32_t i = threadIdx.x; i < nr * choices; i += 256) {
        const uint32_t pair = r0 * choices + i, e = min(choice[pair], partitions);
        const uint32_t p = starts[e] + before[(uint64_t) (pair / kTile) * (partitions + 1) + e] + ranks[pair];
        const bool there = e < partitions;
        place[i] = there ? p : kNone;
        position[pair] = there ? p : kNone;
        map[p] = there ? pair / choices : kNone;   // pairs without a partition come last: their places are the tail
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < nr * words; x += 256) {
        const uint32_t r = x / words, c = x - r * words;
        const W w = *reinterpret_cast<const W *>(rows + (uint64_t) (r0 + r) * stride + (uint64_t) c * B);
        for (uint32_t j = 0; j < choices; j++) {
            const uint32_t p = place[r * choices + j];
            if (p != kNone) *reinterpret_cast<W *>(sorted + (uint64_t) p * sorted_stride + (uint64_t) c * B) = w;
        }
    }
}

// ---- combine ----------------------------------------------------------------------------------------------------
// out[t] = sum over j, ascending, of weight[t,j] * sorted[position[t,j]]; K pairs' words are in flight for each word of a row.
template<typename T, int V, int K>
__global__ void __launch_bounds__(256) combine_kernel(const T *__restrict__ sorted, uint64_t stride, uint32_t sorted_rows,
                                                      const uint32_t *__restrict__ position, uint32_t choices,
                                                      const float *__restrict__ weights, uint32_t units, Div words, T *__restrict__ out,
                                                      uint64_t out_stride) {
    const uint32_t x = blockIdx.x * 256 + threadIdx.x;
    if (x >= units) return;
    const uint32_t row = words.of(x), at = (x - row * words.d) * V;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    for (uint32_t j0 = 0; j0 < choices; j0 += K) {
        uint32_t p[K];
        float w[K], f[K][V];
#pragma unroll
        for (int j = 0; j < K; j++) {
            const uint64_t pair = (uint64_t) row * choices + j0 + j;
            p[j] = j0 + j < choices ? position[pair] : kNone;
            w[j] = weights && j0 + j < choices ? weights[pair] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < K; j++)
            if (p[j] < sorted_rows) load<T, V>(sorted + (uint64_t) p[j] * stride + at, f[j]);
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (p[j] >= sorted_rows) continue;
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] = fmaf(w[j], f[j][i], acc[i]);
        }
    }
    store<T, V>(out + (uint64_t) row * out_stride + at, acc);
}

// grad_sorted[position[t,j]] = weight[t,j] * grad[t] and grad_weights[t,j] = <grad[t], sorted[position[t,j]]>: G lanes own a row.
template<typename T, int V, int K, int G>
__global__ void __launch_bounds__(256) combine_grad_kernel(const T *__restrict__ grad, uint64_t grad_stride, uint32_t count, uint32_t words,
                                                           const T *__restrict__ sorted, uint64_t stride, uint32_t sorted_rows,
                                                           const uint32_t *__restrict__ position, uint32_t choices,
                                                           const float *__restrict__ weights, T *__restrict__ grad_sorted,
                                                           uint64_t grad_sorted_stride, float *__restrict__ grad_weights) {
    __shared__ float part[8][K];
    const uint32_t row = blockIdx.x * (256 / G) + threadIdx.x / G, l = threadIdx.x % G;
    if (G == 32 && row >= count) return;
    for (uint32_t j0 = 0; j0 < choices; j0 += K) {
        uint32_t p[K];
        float w[K], dot[K];
#pragma unroll
        for (int j = 0; j < K; j++) {
            const uint64_t pair = (uint64_t) row * choices + j0 + j;
            p[j] = j0 + j < choices ? position[pair] : kNone;
            w[j] = weights && j0 + j < choices ? weights[pair] : 1.0f;
            dot[j] = 0.0f;
        }
        for (uint32_t c = l; c < words; c += G) {
            float g[V], f[K][V];
            load<T, V>(grad + (uint64_t) row * grad_stride + (uint64_t) c * V, g);
#pragma unroll
            for (int j = 0; j < K; j++)
                if (p[j] < sorted_rows) load<T, V>(sorted + (uint64_t) p[j] * stride + (uint64_t) c * V, f[j]);
#pragma unroll
            for (int j = 0; j < K; j++) {
                if (p[j] >= sorted_rows) continue;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    dot[j] = fmaf(g[i], f[j][i], dot[j]);
                    o[i] = w[j] * g[i];
                }
                store<T, V>(grad_sorted + (uint64_t) p[j] * grad_sorted_stride + (uint64_t) c * V, o);
            }
        }
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
        if (G == 32) {
            if (grad_weights && l < K && j0 + l < choices) {
                float v = dot[0];
#pragma unroll
                for (int j = 1; j < K; j++) v = l == (uint32_t) j ? dot[j] : v;
                grad_weights[(uint64_t) row * choices + j0 + l] = v;
            }
        } else {
            if ((l & 31u) == 0) {
#pragma unroll
                for (int j = 0; j < K; j++) part[l >> 5][j] = dot[j];
            }
            __syncthreads();
            if (grad_weights && l < K && j0 + l < choices) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) v += part[i][l];
                grad_weights[(uint64_t) row * choices + j0 + l] = v;
            }
            __syncthreads();
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------
int fail(glide_ctx *ctx, int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    if (ctx) {
        try { ctx->error = buf; } catch (...) {}
    }
    return code;
}

#define ROWS_REQUIRE(cond, code, ...)                        \
    do {                                                      \
        if (!(cond)) return fail(ctx, code, __VA_ARGS__);     \
    } while (0)

// The context's device for the length of a call; the caller's comes back.
struct OnDevice {
    int before = -1;
    cudaError_t status;
    explicit OnDevice(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

#define ROWS_CUDA(call)                                                                                      \
    do {                                                                                                     \
        const cudaError_t e_ = (call);                                                                       \
        if (e_ != cudaSuccess) return fail(ctx, GLIDE_ERR_CUDA, "%s: %s", __func__, cudaGetErrorString(e_)); \
    } while (0)

uint32_t bytes_of(int type) { return type == GLIDE_ROW_F32 ? 4 : type == GLIDE_ROW_U8 ? 1 : 2; }
bool is_float_type(int type) { return type == GLIDE_ROW_F32 || type == GLIDE_ROW_F16 || type == GLIDE_ROW_BF16; }

// A matrix of rows as an argument.
struct Matrix {
    const void *p;
    uint64_t rows, stride;   // in values
    uint32_t dim;
    int type;
    uint64_t bytes() const { return rows == 0 ? 0 : ((rows - 1) * stride + dim) * bytes_of(type); }
    bool sized() const { return stride <= (1ull << 40) && rows <= (1ull << 32); }
    // The most values (a power of two up to `most`) that a word may hold so that every word of every row is aligned.
    uint32_t width(uint32_t most) const {
        const uint32_t e = bytes_of(type);
        uint32_t v = most;
        while (v > 1 && (reinterpret_cast<uintptr_t>(p) % (v * e) || (rows > 1 && stride % v) || dim % v)) v >>= 1;
        return v;
    }
};

bool aligned(const Matrix &m) { return reinterpret_cast<uintptr_t>(m.p) % bytes_of(m.type) == 0; }
bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na && nb && x < y + nb && y < x + na;
}
bool overlap(const Matrix &a, const Matrix &b) { return overlap(a.p, a.bytes(), b.p, b.bytes()); }

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t) 255; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// f(width as a constant) for a width of 1, 2, 4 or 8 values
template<int V> struct Width { static constexpr int value = V; };
template<int kMost, typename F> cudaError_t with_width(uint32_t v, F f) {
    if constexpr (kMost >= 8) if (v >= 8) return f(Width<8>{});
    if constexpr (kMost >= 4) if (v >= 4) return f(Width<4>{});
    if (v >= 2) return f(Width<2>{});
    return f(Width<1>{});
}

// f(a value of the type, Width) for rows of floating types
template<typename F> cudaError_t with_rows(int type, uint32_t v, F f) {
    if (type == GLIDE_ROW_F32) return with_width<4>(v, [&](auto w) { return f(float{}, w); });
    if (type == GLIDE_ROW_F16) return with_width<8>(v, [&](auto w) { return f(__half{}, w); });
    return with_width<8>(v, [&](auto w) { return f(__nv_bfloat16{}, w); });
}
uint32_t most_of(int type) { return type == GLIDE_ROW_F32 || type == GLIDE_ROW_U8 ? 4 : 8; }

template<typename T, typename O, int V>
cudaError_t launch_lookup(const void *table, uint64_t table_stride, uint32_t n, const uint32_t *ids, uint64_t count, uint32_t dim, float scale,
                          void *out, uint64_t out_stride, cudaStream_t stream) {
    const uint32_t words = dim / V;
    const uint64_t most = 0x7fff0000u / words;   // rows of a launch: its words are counted in 31 bits
    for (uint64_t r0 = 0; r0 < count; r0 += most) {
        const uint32_t rows = (uint32_t) (count - r0 < most ? count - r0 : most), units = rows * words;
        O *to = static_cast<O *>(out) + r0 * out_stride;
        if (units <= 256 * 1024)
            lookup_kernel<T, O, V, 1><<<(uint32_t) ceil_div(units, 256), 256, 0, stream>>>(static_cast<const T *>(table), table_stride, n, ids + r0, units, Div(words), scale, to, out_stride);
        else
            lookup_kernel<T, O, V, 4><<<(uint32_t) ceil_div(units, 1024), 256, 0, stream>>>(static_cast<const T *>(table), table_stride, n, ids + r0, units, Div(words), scale, to, out_stride);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Shared memory of the counting kernel: above the 48 KB that need no word from the launcher for many buckets.
cudaError_t launch_count(const uint32_t *keys, uint32_t items, Digit digit, uint32_t buckets, uint32_t *counts, uint16_t *ranks,
                         uint32_t *totals, cudaStream_t stream) {
    const uint32_t tiles = (uint32_t) ceil_div(items, kTile), smem = kSortWarps * buckets * 2;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(bucket_count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem);
        if (e != cudaSuccess) return e;
    }
    bucket_count_kernel<<<tiles, kSortThreads, smem, stream>>>(keys, items, digit, buckets, counts, ranks);
    bucket_scan_kernel<<<(uint32_t) ceil_div(buckets, 32), 1024, 0, stream>>>(counts, tiles, buckets, totals);
    return cudaGetLastError();
}

// Scratch of the gradient: two copies of the sorted items, the counts of a pass, the partial sums of its chunks.
struct GradScratch {
    uint32_t *keys[2], *values[2], *counts, *totals;
    uint16_t *ranks;
    float *partial;
    uint32_t bits, passes, pass_bits;
    uint64_t bytes;
    GradScratch(void *base, uint64_t n, uint64_t items, uint32_t dim) {
        bits = 1;
        while ((1ull << bits) <= n) bits++;             // ids 0 .. n - 1, and n for none
        passes = (bits + 10) / 11;
        pass_bits = (bits + passes - 1) / passes;
        uint64_t at = 0;
        auto take = [&](uint64_t size) {
            const uint64_t here = at;
            at += align256(size);
            return static_cast<char *>(base) + here;
        };
        const uint64_t tiles = ceil_div(items, kTile);
        for (int i = 0; i < 2; i++) {
            keys[i] = reinterpret_cast<uint32_t *>(take(items * 4));
            values[i] = reinterpret_cast<uint32_t *>(take(items * 4));
        }
        ranks = reinterpret_cast<uint16_t *>(take(items * 2));
        counts = reinterpret_cast<uint32_t *>(take((tiles << pass_bits) * 4));
        totals = reinterpret_cast<uint32_t *>(take(4ull << pass_bits));
        partial = reinterpret_cast<float *>(take(2 * ceil_div(items, kChunk) * dim * 4));
        bytes = at;
    }
};

struct DispatchScratch {
    uint32_t *counts, *totals;
    uint16_t *ranks;
    uint64_t bytes;
    DispatchScratch(void *base, uint64_t pairs, uint32_t partitions) {
        uint64_t at = 0;
        auto take = [&](uint64_t size) {
            const uint64_t here = at;
            at += align256(size);
            return static_cast<char *>(base) + here;
        };
        ranks = reinterpret_cast<uint16_t *>(take(pairs * 2));
        counts = reinterpret_cast<uint32_t *>(take(ceil_div(pairs, kTile) * (partitions + 1) * 4));
        totals = reinterpret_cast<uint32_t *>(take((partitions + 1) * 4ull));
        bytes = at;
    }
};

}  // namespace
}  // namespace glide

using namespace glide;

extern "C" {

int glide_lookup_rows(glide_ctx *ctx, const void *d_table, int row_type, uint64_t n, uint32_t dim, uint64_t table_stride,
                      const uint32_t *d_ids, uint64_t count, float scale, void *d_out, uint64_t out_stride, void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "lookup_rows: null context");
    ROWS_REQUIRE(is_float_type(row_type) || row_type == GLIDE_ROW_U8, GLIDE_ERR_UNSUPPORTED, "lookup_rows: unsupported row type %d", row_type);
    const Matrix table{d_table, n, table_stride, dim, row_type};
    const Matrix out{d_out, count, out_stride, dim, row_type == GLIDE_ROW_U8 ? (int) GLIDE_ROW_F32 : row_type};
    ROWS_REQUIRE(dim >= 1 && n >= 1 && n <= kNone, GLIDE_ERR_BAD_ARG, "lookup_rows: a table has 1 to 2^32 - 1 rows of at least one value");
    ROWS_REQUIRE(dim <= kMaxDim && count <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "lookup_rows: rows of more than 2^20 values or more than 2^31 - 1 ids");
    if (count == 0) return GLIDE_OK;
    ROWS_REQUIRE(d_table && d_ids && d_out, GLIDE_ERR_BAD_ARG, "lookup_rows: null pointer");
    ROWS_REQUIRE(table.sized() && out.sized() && (out_stride >= dim || count == 1), GLIDE_ERR_BAD_ARG, "lookup_rows: rows of the result overlap, or a stride is beyond 2^40");
    ROWS_REQUIRE(aligned(table) && aligned(out) && reinterpret_cast<uintptr_t>(d_ids) % 4 == 0, GLIDE_ERR_BAD_ARG, "lookup_rows: a pointer is not aligned to its type");
    ROWS_REQUIRE(!overlap(out, table) && !overlap(d_out, out.bytes(), d_ids, count * 4), GLIDE_ERR_BAD_ARG, "lookup_rows: the result overlaps an input");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    const uint32_t most = most_of(row_type), v0 = table.width(most), v1 = out.width(most), v = v0 < v1 ? v0 : v1;
    auto s = static_cast<cudaStream_t>(stream);
    if (row_type == GLIDE_ROW_U8)
        ROWS_CUDA(with_width<4>(v, [&](auto w) { return launch_lookup<uint8_t, float, decltype(w)::value>(d_table, table_stride, (uint32_t) n, d_ids, count, dim, scale, d_out, out_stride, s); }));
    else
        ROWS_CUDA(with_rows(row_type, v, [&](auto t, auto w) { return launch_lookup<decltype(t), decltype(t), decltype(w)::value>(d_table, table_stride, (uint32_t) n, d_ids, count, dim, scale, d_out, out_stride, s); }));
    return GLIDE_OK;
}

size_t glide_lookup_rows_grad_workspace(uint64_t n, uint32_t dim, uint64_t count) {
    if (n > kNone || dim > kMaxDim || count > 0x7fffffffu) return 0;
    return count == 0 ? 0 : (size_t) GradScratch(nullptr, n, count, dim).bytes;
}

int glide_lookup_rows_grad(glide_ctx *ctx, const void *d_grad, int row_type, uint64_t grad_stride, const uint32_t *d_ids, uint64_t count,
                           float scale, void *d_table_grad, int grad_type, uint64_t n, uint32_t dim, uint64_t table_grad_stride, int accumulate,
                           void *d_workspace, size_t workspace_bytes, void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "lookup_rows_grad: null context");
    ROWS_REQUIRE(is_float_type(row_type) && (grad_type == row_type || grad_type == GLIDE_ROW_F32), GLIDE_ERR_UNSUPPORTED, "lookup_rows_grad: unsupported types %d, %d (the table's gradient has the rows' type or fp32)", row_type, grad_type);
    const Matrix in{d_grad, count, grad_stride, dim, row_type}, out{d_table_grad, n, table_grad_stride, dim, grad_type};
    ROWS_REQUIRE(dim >= 1 && n >= 1 && n <= kNone, GLIDE_ERR_BAD_ARG, "lookup_rows_grad: a table has 1 to 2^32 - 1 rows of at least one value");
    ROWS_REQUIRE(dim <= kMaxDim && count <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "lookup_rows_grad: rows of more than 2^20 values or more than 2^31 - 1 ids");
    ROWS_REQUIRE(d_table_grad && (count == 0 || (d_grad && d_ids)), GLIDE_ERR_BAD_ARG, "lookup_rows_grad: null pointer");
    ROWS_REQUIRE(in.sized() && out.sized() && (table_grad_stride >= dim || n == 1), GLIDE_ERR_BAD_ARG, "lookup_rows_grad: rows of the result overlap, or a stride is beyond 2^40");
    ROWS_REQUIRE(aligned(in) && aligned(out) && reinterpret_cast<uintptr_t>(d_ids) % 4 == 0, GLIDE_ERR_BAD_ARG, "lookup_rows_grad: a pointer is not aligned to its type");
    const size_t need = glide_lookup_rows_grad_workspace(n, dim, count);
    ROWS_REQUIRE(workspace_bytes >= need && (need == 0 || d_workspace), GLIDE_ERR_BAD_ARG, "lookup_rows_grad: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    ROWS_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0, GLIDE_ERR_BAD_ARG, "lookup_rows_grad: the workspace is not aligned to 256 bytes");
    ROWS_REQUIRE(!overlap(out, in) && !overlap(d_table_grad, out.bytes(), d_ids, count * 4) && !overlap(d_workspace, need, d_grad, in.bytes()) &&
                 !overlap(d_workspace, need, d_table_grad, out.bytes()) && !overlap(d_workspace, need, d_ids, count * 4),
                 GLIDE_ERR_BAD_ARG, "lookup_rows_grad: the result or the workspace overlaps another argument");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    if (!accumulate)
        ROWS_CUDA(cudaMemset2DAsync(d_table_grad, table_grad_stride * bytes_of(grad_type), 0, (size_t) dim * bytes_of(grad_type), n, s));
    if (count == 0) return GLIDE_OK;
    const GradScratch w(d_workspace, n, count, dim);
    const uint32_t items = (uint32_t) count;
    const uint32_t *keys = d_ids, *values = nullptr;
    for (uint32_t pass = 0; pass < w.passes; pass++) {
        const uint32_t left = w.bits - pass * w.pass_bits, here = left < w.pass_bits ? left : w.pass_bits, buckets = 1u << here;
        const Digit digit{(uint32_t) n, pass * w.pass_bits, buckets - 1};
        ROWS_CUDA(launch_count(keys, items, digit, buckets, w.counts, w.ranks, w.totals, s));
        bucket_scatter_kernel<<<(uint32_t) ceil_div(items, kTile), kSortThreads, buckets * 4, s>>>(keys, values, items, digit, buckets, w.counts, w.totals, w.ranks, w.keys[pass & 1], w.values[pass & 1]);
        ROWS_CUDA(cudaGetLastError());
        keys = w.keys[pass & 1];
        values = w.values[pass & 1];
    }
    const uint32_t most = most_of(row_type), v0 = in.width(most), v1 = out.width(most), v = v0 < v1 ? v0 : v1;
    GradArgs a{keys, values, items, (uint32_t) n, dim, dim / v, 32, 1, scale, grad_stride, table_grad_stride, accumulate, w.partial};
    while (a.lanes > 1 && a.lanes / 2 >= a.words) a.lanes /= 2;
    a.slabs = (uint32_t) ceil_div(a.words, a.lanes);
    const uint64_t grid = ceil_div(ceil_div(items, kChunk) * a.slabs * a.lanes, 256);
    ROWS_REQUIRE(grid <= 0xffffffu, GLIDE_ERR_UNSUPPORTED, "lookup_rows_grad: too many values in one call");   // threads are counted in 32 bits
    auto run = [&](auto t, auto o, auto wd) {
        using T = decltype(t);
        using O = decltype(o);
        constexpr int V = decltype(wd)::value;
        grad_join_kernel<T, O, V><<<(uint32_t) grid, 256, 0, s>>>(static_cast<const T *>(d_grad), static_cast<O *>(d_table_grad), a);
        grad_fix_kernel<O, V><<<(uint32_t) grid, 256, 0, s>>>(static_cast<O *>(d_table_grad), a);
        return cudaGetLastError();
    };
    ROWS_CUDA(with_rows(row_type, v, [&](auto t, auto wd) { return grad_type == GLIDE_ROW_F32 ? run(t, float{}, wd) : run(t, t, wd); }));
    return GLIDE_OK;
}

size_t glide_dispatch_rows_workspace(uint64_t count, uint32_t choices, uint32_t partitions) {
    if (count == 0 || choices == 0 || choices > kMaxChoices || partitions > kMaxPartitions || count > 0x7fffffffu / choices) return 0;
    return (size_t) DispatchScratch(nullptr, count * choices, partitions).bytes;
}

int glide_dispatch_rows(glide_ctx *ctx, const void *d_rows, int row_type, uint64_t count, uint32_t dim, uint64_t row_stride,
                        const uint32_t *d_choice, uint32_t choices, uint32_t partitions, void *d_sorted, uint64_t sorted_stride,
                        uint32_t *d_position, uint32_t *d_map, uint32_t *d_segment_start, void *d_workspace, size_t workspace_bytes, void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "dispatch_rows: null context");
    ROWS_REQUIRE(is_float_type(row_type), GLIDE_ERR_UNSUPPORTED, "dispatch_rows: unsupported row type %d", row_type);
    ROWS_REQUIRE(dim >= 1 && choices >= 1 && partitions >= 1, GLIDE_ERR_BAD_ARG, "dispatch_rows: no values, choices or partitions");
    ROWS_REQUIRE(dim <= kMaxDim && choices <= kMaxChoices && partitions <= kMaxPartitions && count <= 0x7fffffffu / choices, GLIDE_ERR_UNSUPPORTED, "dispatch_rows: more than 128 choices, 4096 partitions, 2^20 values or 2^31 - 1 pairs");
    const uint64_t pairs = count * choices;
    const Matrix in{d_rows, count, row_stride, dim, row_type}, out{d_sorted, pairs, sorted_stride, dim, row_type};
    ROWS_REQUIRE(d_segment_start && (count == 0 || (d_rows && d_choice && d_sorted && d_position && d_map)), GLIDE_ERR_BAD_ARG, "dispatch_rows: null pointer");
    ROWS_REQUIRE(in.sized() && out.sized() && (sorted_stride >= dim || pairs <= 1), GLIDE_ERR_BAD_ARG, "dispatch_rows: rows of the result overlap, or a stride is beyond 2^40");
    ROWS_REQUIRE(aligned(in) && aligned(out) && (reinterpret_cast<uintptr_t>(d_choice) | reinterpret_cast<uintptr_t>(d_position) | reinterpret_cast<uintptr_t>(d_map) | reinterpret_cast<uintptr_t>(d_segment_start)) % 4 == 0, GLIDE_ERR_BAD_ARG, "dispatch_rows: a pointer is not aligned to its type");
    const size_t need = glide_dispatch_rows_workspace(count, choices, partitions);
    ROWS_REQUIRE(workspace_bytes >= need && (need == 0 || d_workspace), GLIDE_ERR_BAD_ARG, "dispatch_rows: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    ROWS_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0, GLIDE_ERR_BAD_ARG, "dispatch_rows: the workspace is not aligned to 256 bytes");
    {
        struct Range { const void *p; uint64_t n; } r[] = {{d_rows, in.bytes()}, {d_choice, pairs * 4}, {d_sorted, out.bytes()}, {d_position, pairs * 4}, {d_map, pairs * 4},
                                                           {d_segment_start, (partitions + 1) * 4ull}, {d_workspace, need}};
        for (int i = 2; i < 7; i++)
            for (int j = 0; j < i; j++)
                ROWS_REQUIRE(!overlap(r[i].p, r[i].n, r[j].p, r[j].n), GLIDE_ERR_BAD_ARG, "dispatch_rows: a result or the workspace overlaps another argument");
    }
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    if (count == 0) {
        ROWS_CUDA(cudaMemsetAsync(d_segment_start, 0, (partitions + 1) * 4ull, s));
        return GLIDE_OK;
    }
    const DispatchScratch w(d_workspace, pairs, partitions);
    ROWS_CUDA(launch_count(d_choice, (uint32_t) pairs, Digit{partitions, 0, kNone}, partitions + 1, w.counts, w.ranks, w.totals, s));
    const uint32_t e = bytes_of(row_type), most = 16 / e, v0 = in.width(most), v1 = out.width(most), v = v0 < v1 ? v0 : v1, words = dim / v;
    uint32_t each = 2048 / words;   // rows of a CTA: some 2,048 words to copy, and as many pairs at most
    if (each > 2048 / choices) each = 2048 / choices;
    if (each < 1) each = 1;
    if (each > count) each = (uint32_t) count;
    const uint32_t grid = (uint32_t) ceil_div(count, each), smem = (partitions + 1 + each * choices) * 4;
    auto run = [&](auto b) {
        dispatch_kernel<decltype(b)::value><<<grid, 256, smem, s>>>(static_cast<const uint8_t *>(d_rows), row_stride * e, (uint32_t) count, words, d_choice, choices, partitions, w.counts, w.totals, w.ranks, each,
                                                                   static_cast<uint8_t *>(d_sorted), sorted_stride * e, d_position, d_map, d_segment_start);
        return cudaGetLastError();
    };
    switch (v * e) {
        case 16: ROWS_CUDA(run(Width<16>{})); break;
        case 8: ROWS_CUDA(run(Width<8>{})); break;
        case 4: ROWS_CUDA(run(Width<4>{})); break;
        default: ROWS_CUDA(run(Width<2>{})); break;
    }
    return GLIDE_OK;
}

int glide_combine_rows(glide_ctx *ctx, const void *d_sorted, int row_type, uint64_t sorted_rows, uint32_t dim, uint64_t sorted_stride,
                       const uint32_t *d_position, uint64_t count, uint32_t choices, const float *d_weights_or_null, void *d_out,
                       uint64_t out_stride, void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "combine_rows: null context");
    ROWS_REQUIRE(is_float_type(row_type), GLIDE_ERR_UNSUPPORTED, "combine_rows: unsupported row type %d", row_type);
    ROWS_REQUIRE(dim >= 1 && choices >= 1, GLIDE_ERR_BAD_ARG, "combine_rows: no values or choices");
    ROWS_REQUIRE(dim <= kMaxDim && choices <= kMaxChoices && count <= 0x7fffffffu / choices && sorted_rows <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "combine_rows: more than 128 choices, 2^20 values or 2^31 - 1 pairs or rows");
    if (count == 0) return GLIDE_OK;
    const Matrix in{d_sorted, sorted_rows, sorted_stride, dim, row_type}, out{d_out, count, out_stride, dim, row_type};
    ROWS_REQUIRE((d_sorted || sorted_rows == 0) && d_position && d_out, GLIDE_ERR_BAD_ARG, "combine_rows: null pointer");
    ROWS_REQUIRE(in.sized() && out.sized() && (out_stride >= dim || count == 1), GLIDE_ERR_BAD_ARG, "combine_rows: rows of the result overlap, or a stride is beyond 2^40");
    ROWS_REQUIRE(aligned(in) && aligned(out) && (reinterpret_cast<uintptr_t>(d_position) | reinterpret_cast<uintptr_t>(d_weights_or_null)) % 4 == 0, GLIDE_ERR_BAD_ARG, "combine_rows: a pointer is not aligned to its type");
    ROWS_REQUIRE(!overlap(out, in) && !overlap(d_out, out.bytes(), d_position, count * choices * 4) && !overlap(d_out, out.bytes(), d_weights_or_null, d_weights_or_null ? count * choices * 4 : 0), GLIDE_ERR_BAD_ARG, "combine_rows: the result overlaps an input");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    const uint32_t most = most_of(row_type), v0 = in.width(most), v1 = out.width(most), v = v0 < v1 ? v0 : v1, words = dim / v;
    const uint64_t each = 0x7fff0000u / words;   // rows of a launch: its words are counted in 31 bits
    for (uint64_t r0 = 0; r0 < count; r0 += each) {
        const uint32_t rows = (uint32_t) (count - r0 < each ? count - r0 : each), units = rows * words, grid = (uint32_t) ceil_div(units, 256);
        const uint32_t *position = d_position + r0 * choices;
        const float *weights = d_weights_or_null ? d_weights_or_null + r0 * choices : nullptr;
        ROWS_CUDA(with_rows(row_type, v, [&](auto t, auto wd) {
            using T = decltype(t);
            constexpr int V = decltype(wd)::value;
            const T *from = static_cast<const T *>(d_sorted);
            T *to = static_cast<T *>(d_out) + r0 * out_stride;
            if (choices <= 2) combine_kernel<T, V, 2><<<grid, 256, 0, s>>>(from, sorted_stride, (uint32_t) sorted_rows, position, choices, weights, units, Div(words), to, out_stride);
            else combine_kernel<T, V, 8><<<grid, 256, 0, s>>>(from, sorted_stride, (uint32_t) sorted_rows, position, choices, weights, units, Div(words), to, out_stride);
            return cudaGetLastError();
        }));
    }
    return GLIDE_OK;
}

int glide_combine_rows_grad(glide_ctx *ctx, const void *d_grad, int row_type, uint64_t count, uint32_t dim, uint64_t grad_stride,
                            const void *d_sorted, uint64_t sorted_rows, uint64_t sorted_stride, const uint32_t *d_position, uint32_t choices,
                            const float *d_weights_or_null, void *d_grad_sorted, uint64_t grad_sorted_stride, float *d_grad_weights_or_null,
                            void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "combine_rows_grad: null context");
    ROWS_REQUIRE(is_float_type(row_type), GLIDE_ERR_UNSUPPORTED, "combine_rows_grad: unsupported row type %d", row_type);
    ROWS_REQUIRE(dim >= 1 && choices >= 1, GLIDE_ERR_BAD_ARG, "combine_rows_grad: no values or choices");
    ROWS_REQUIRE(dim <= kMaxDim && choices <= kMaxChoices && count <= 0x7fffffffu / choices && sorted_rows <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "combine_rows_grad: more than 128 choices, 2^20 values or 2^31 - 1 pairs or rows");
    if (count == 0) return GLIDE_OK;
    const uint64_t pairs = count * choices;
    const Matrix grad{d_grad, count, grad_stride, dim, row_type}, in{d_sorted, sorted_rows, sorted_stride, dim, row_type}, out{d_grad_sorted, sorted_rows, grad_sorted_stride, dim, row_type};
    ROWS_REQUIRE(d_grad && d_position && (sorted_rows == 0 || (d_sorted && d_grad_sorted)), GLIDE_ERR_BAD_ARG, "combine_rows_grad: null pointer");
    ROWS_REQUIRE(grad.sized() && in.sized() && out.sized() && (grad_sorted_stride >= dim || sorted_rows <= 1), GLIDE_ERR_BAD_ARG, "combine_rows_grad: rows of the result overlap, or a stride is beyond 2^40");
    ROWS_REQUIRE(aligned(grad) && aligned(in) && aligned(out) && (reinterpret_cast<uintptr_t>(d_position) | reinterpret_cast<uintptr_t>(d_weights_or_null) | reinterpret_cast<uintptr_t>(d_grad_weights_or_null)) % 4 == 0, GLIDE_ERR_BAD_ARG, "combine_rows_grad: a pointer is not aligned to its type");
    {
        struct Range { const void *p; uint64_t n; } r[] = {{d_grad, grad.bytes()}, {d_sorted, in.bytes()}, {d_position, pairs * 4}, {d_weights_or_null, d_weights_or_null ? pairs * 4 : 0},
                                                           {d_grad_sorted, out.bytes()}, {d_grad_weights_or_null, d_grad_weights_or_null ? pairs * 4 : 0}};
        for (int i = 4; i < 6; i++)
            for (int j = 0; j < i; j++)
                ROWS_REQUIRE(!overlap(r[i].p, r[i].n, r[j].p, r[j].n), GLIDE_ERR_BAD_ARG, "combine_rows_grad: a result overlaps another argument");
    }
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    const uint32_t most = most_of(row_type), v0 = grad.width(most), v1 = in.width(most), v2 = out.width(most);
    const uint32_t v01 = v0 < v1 ? v0 : v1, v = v01 < v2 ? v01 : v2, words = dim / v;
    ROWS_CUDA(with_rows(row_type, v, [&](auto t, auto wd) {
        using T = decltype(t);
        constexpr int V = decltype(wd)::value;
        auto go = [&](auto kk, auto gg) {
            constexpr int K = decltype(kk)::value, G = decltype(gg)::value;
            combine_grad_kernel<T, V, K, G><<<(uint32_t) ceil_div(count, 256 / G), 256, 0, s>>>(
                static_cast<const T *>(d_grad), grad_stride, (uint32_t) count, words, static_cast<const T *>(d_sorted), sorted_stride, (uint32_t) sorted_rows, d_position, choices,
                d_weights_or_null, static_cast<T *>(d_grad_sorted), grad_sorted_stride, d_grad_weights_or_null);
            return cudaGetLastError();
        };
        if (choices <= 2) return words > 64 ? go(Width<2>{}, Width<256>{}) : go(Width<2>{}, Width<32>{});
        return words > 64 ? go(Width<8>{}, Width<256>{}) : go(Width<8>{}, Width<32>{});
    }));
    return GLIDE_OK;
}

}  // extern "C"
