// Operators on the rows of a table: rows looked up by ids and the gradient of the table, rows sorted by the
// partitions (experts) they chose, brought back with weights, and the gradients of that. They follow a search (ids to
// rows) or an assignment (partitions to rows) and precede an index (the table it is built over); the reference has
// no counterpart. All calls enqueue on the caller's stream and return; scratch is the caller's.
//
// Everything here is bound by bytes, or by launches where rows are few. Rows are read and written in the widest words their
// addresses allow (16 bytes where base, stride and length are multiples of it), sums are fp32 in an order that the arguments
// alone determine, and each value is rounded once, when it is stored. Times in the comments are of one call in a captured graph on
// inputs larger than L2, shares are of the measured copy rate (6.55 TB/s).
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
constexpr uint32_t kRounds = 8;             // items of a thread in the counting sort
constexpr uint32_t kTileThreads = 256, kTile = kTileThreads * kRounds;
constexpr uint32_t kFew = 4096;             // items that are sorted by comparing each with all (the gradient of 4,000 ids of 64 bf16: 15 us, of 4,097 in tiles: 20)
constexpr uint32_t kFewPairs = 2048;        // pairs that dispatch_rows places and copies in one launch (2,000: 6 to 8 us, in tiles 8; 4,000: 14 to 19, in tiles 8 to 10)
// Ids whose gradient takes one launch (see grad_few_kernel), whatever they are: 1,024 different ones, added to a table of 64, 512 and 4,096 bf16 a row, 7,
// 8 and 10 us, by the sort 10, 10 and 11. The other side: one CTA adds up an id, so that 1,024 equal ones take 7, 27 and 187 us, by the sort 13, 14 and 15.
constexpr uint32_t kFewIds = 1024;
constexpr uint32_t kMaxPassBits = 11;       // bits of a pass's digit, at most
constexpr uint32_t kMaxFusedCounts = 16384; // counts (tiles x buckets) that every CTA of the second kernel adds up by itself (64 x 1,001 of them: 19.5 us, scanned by a launch of their own 13.9)
constexpr uint32_t kClearShare = 48u << 20; // bytes of a gradient that are cleared beside each launch of its sort (12 to 64 MB differ by 3 %)

// ---- rows as words ----------------------------------------------------------------------------------------
// A kernel handles a row in pieces of V values, a word of up to 16 bytes of its input: as many as the addresses, strides and lengths of
// all matrices are multiples of. Rows of an odd number of 16-bit values (or of bytes) would leave an access for each value. Where that
// costs most (lookup_kernel, combine_kernel) they have a second form, kWhole = false: a piece is what falls into a word of the row
// that is WRITTEN, so that full words are stored, and what is read lies in two words beside each other, which are shifted into one;
// words that would reach beyond the matrix are read value by value. 1,001 bf16 a row, value by value and shifted: 40,000 rows looked up
// 46 and 38 us, 20,000 x 4 combined 88 and 65; but dispatched 56 and 94, the gradient of combine 94 and 170: the shifting costs more.
template<int B> struct Word;
template<> struct Word<16> { using type = uint4; };
template<> struct Word<8> { using type = uint2; };
template<> struct Word<4> { using type = uint32_t; };
template<> struct Word<2> { using type = uint16_t; };
template<typename T, int V> using WordOf = typename Word<(int) sizeof(T) * V>::type;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(uint8_t x) { return (float) x; }
template<typename T> __device__ __forceinline__ T from_float(float x);
template<> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template<> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Rows of a matrix in device memory, and its first and last address.
template<typename T>
struct Rows {
    T *p;
    uint64_t stride;   // in values
    uint64_t begin, end;
    __device__ __forceinline__ T *row(uint64_t r) const { return p + r * stride; }
};

// A piece that has been asked for. Nothing may look at it before all pieces that are to be in flight have been: a conversion beside a
// load makes the load be waited for before the next (combine_kernel: 1.9 of 6.5 TB/s).
template<typename T, int V, bool kWhole>
struct Piece {
    WordOf<T, V> a;
    __device__ __forceinline__ WordOf<T, V> word() const { return a; }
};
template<typename T, int V>
struct Piece<T, V, false> {
    WordOf<T, V> a, b;
    uint32_t shift;   // bytes of a that come before the piece
    __device__ __forceinline__ WordOf<T, V> word() const {
        if constexpr (sizeof(a) == 4) {
            return __funnelshift_r(a, b, shift * 8);
        } else {
            uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 6; i++) w[i] = shift & 8u ? w[i + 2] : w[i];
#pragma unroll
            for (int i = 0; i < 5; i++) w[i] = shift & 4u ? w[i + 1] : w[i];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(w[i], w[i + 1], (shift & 3u) * 8);
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// Values start .. start + V - 1 of a row of m; zeros where the piece is not wanted. Values outside of the row are anything.
// One access a word: a plain dereference is split into values by the compiler when they are taken apart next.
template<int V, bool kWhole, typename T>
__device__ __forceinline__ Piece<T, V, kWhole> fetch(const Rows<const T> &m, const T *row, int32_t start, uint32_t dim, bool wanted) {
    using W = WordOf<T, V>;
    Piece<T, V, kWhole> piece;
    memset(&piece, 0, sizeof piece);
    if constexpr (kWhole) {
        if (wanted) piece.a = __ldg(reinterpret_cast<const W *>(row + start));
    } else if (wanted) {
        const uint64_t at = reinterpret_cast<uintptr_t>(row) + (int64_t) start * (int64_t) sizeof(T), from = at & ~(uint64_t) (sizeof(W) - 1);
        const uint32_t shift = (uint32_t) (at - from);
        if (from >= m.begin && from + (shift ? 2 : 1) * sizeof(W) <= m.end) {
            piece.a = __ldg(reinterpret_cast<const W *>(from));
            if (shift) piece.b = __ldg(reinterpret_cast<const W *>(from) + 1);
            piece.shift = shift;
        } else {   // at either end of the matrix
            T t[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                memset(&t[i], 0, sizeof t[i]);
                if (start + i >= 0 && start + i < (int32_t) dim) t[i] = row[start + i];
            }
            memcpy(&piece.a, t, sizeof piece.a);
        }
    }
    return piece;
}

template<typename T, int V>
__device__ __forceinline__ void unpack(const WordOf<T, V> &w, float (&f)[V]) {
    T t[V];
    memcpy(t, &w, sizeof w);
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = to_float(t[i]);
}

// The first value of piece c of a row that is written.
template<int V, bool kWhole, typename O>
__device__ __forceinline__ int32_t piece_start(const O *row, uint32_t c) {
    if constexpr (kWhole) return (int32_t) (c * V);
    else return (int32_t) (c * V) - (int32_t) ((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(O));
}
// Pieces of such a row, at most.
template<int V, typename O> constexpr uint32_t pieces(bool whole, uint32_t dim) { return whole ? dim / V : (dim + V - 1 + 16 / (uint32_t) sizeof(O) - 1) / V; }

// V values in words of 16 bytes at most.
template<typename O, int V>
__device__ __forceinline__ void store(O *p, const float (&f)[V]) {
    constexpr int H = 16 / (int) sizeof(O) < V ? 16 / (int) sizeof(O) : V;
#pragma unroll
    for (int h = 0; h < V; h += H) {
        O t[H];
#pragma unroll
        for (int i = 0; i < H; i++) t[i] = from_float<O>(f[h + i]);
        WordOf<O, H> w;
        memcpy(&w, t, sizeof w);
        __stcg(reinterpret_cast<WordOf<O, H> *>(p + h), w);
    }
}
// Of memory that is written in the same launch, each word by the thread that reads it, or by a launch of the same call
template<typename O, int V>
__device__ __forceinline__ void load(const O *p, float (&f)[V]) {
    constexpr int H = 16 / (int) sizeof(O) < V ? 16 / (int) sizeof(O) : V;
#pragma unroll
    for (int h = 0; h < V; h += H) {
        const WordOf<O, H> w = __ldcg(reinterpret_cast<const WordOf<O, H> *>(p + h));
        O t[H];
        memcpy(t, &w, sizeof w);
#pragma unroll
        for (int i = 0; i < H; i++) f[h + i] = to_float(t[i]);
    }
}

// A piece of a row that is written: the values of it that the row has.
template<int V, bool kWhole, typename O>
__device__ __forceinline__ void put(O *row, int32_t start, uint32_t dim, const float (&f)[V]) {
    if (kWhole || (start >= 0 && start + V <= (int32_t) dim)) {
        store<O, V>(row + start, f);
    } else {
        const int32_t lo = -start, hi = (int32_t) dim - start;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= lo && i < hi) row[start + i] = from_float<O>(f[i]);
    }
}

// How many pieces of `each` bytes a lane keeps in flight to have `bytes` of them: narrow ones have to be many (40,500 rows of 2,463 fp32
// looked up one by one: 183 us with 4 in flight, 119 with 16).
__host__ __device__ constexpr int in_flight(int bytes, int each, int most) { return bytes / each < 1 ? 1 : bytes / each > most ? most : bytes / each; }

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
// out[t] = scale * table[ids[t]], zeros for ids beyond the table (0xffffffff among them). A thread owns U pieces of the output, a
// CTA's width apart, so that U loads are in flight once the ids (which a CTA shares through L1) have come: 2 for large calls (1 takes a
// quarter longer, 4 as long), 1 where 2 would leave SMs idle. 32,768 ids over 131,072 rows of 8 KB: 64 us, 87 % of the copy rate; bound by
// DRAM and, a little, by the wait for the ids.
template<typename T, typename O, int V, bool kWhole, int U>
__global__ void __launch_bounds__(256) lookup_kernel(Rows<const T> table, uint32_t n, uint32_t dim, const uint32_t *__restrict__ ids, uint32_t units, Div words,
                                                     float scale, Rows<O> out) {
    const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t id[U];
    int32_t at[U];
    O *to[U];
    Piece<T, V, kWhole> piece[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t x = min(first + u * 256, units - 1), row = words.of(x);
        to[u] = out.row(row);
        at[u] = piece_start<V, kWhole>(to[u], x - row * words.d);
        id[u] = ids[row];
    }
#pragma unroll
    for (int u = 0; u < U; u++) piece[u] = fetch<V, kWhole>(table, table.row(id[u]), at[u], dim, id[u] < n);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (first + u * 256 >= units) break;
        float f[V];
        unpack<T, V>(piece[u].word(), f);
#pragma unroll
        for (int i = 0; i < V; i++) f[i] *= id[u] < n ? scale : 0.0f;   // what was not fetched is 0
        put<V, kWhole>(to[u], at[u], dim, f);
    }
}

// The same with a warp a row: what belongs to the row is worked out once, not for every piece. Taken for many long rows of narrow pieces (long_rows).
template<typename T, typename O, int V, bool kWhole, int U>
__global__ void __launch_bounds__(256) lookup_long_kernel(Rows<const T> table, uint32_t n, uint32_t dim, const uint32_t *__restrict__ ids, uint32_t count, uint32_t words,
                                                          float scale, Rows<O> out) {
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= count) return;
    const uint32_t id = ids[row];
    const bool there = id < n;
    const T *from = table.row(id);
    O *to = out.row(row);
    const float by = there ? scale : 0.0f;   // what is not fetched is 0
    for (uint32_t c = threadIdx.x & 31u; c < words; c += 32 * U) {
        Piece<T, V, kWhole> piece[U];
#pragma unroll
        for (int u = 0; u < U; u++) piece[u] = fetch<V, kWhole>(table, from, piece_start<V, kWhole>(to, c + u * 32), dim, there && c + u * 32 < words);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c + u * 32 >= words) break;
            float f[V];
            unpack<T, V>(piece[u].word(), f);
#pragma unroll
            for (int i = 0; i < V; i++) f[i] *= by;
            put<V, kWhole>(to, piece_start<V, kWhole>(to, c + u * 32), dim, f);
        }
    }
}

// ---- launches that follow one another -----------------------------------------------------------------------------
// The kernels of one call are launched as programmatic dependents: the next one's CTAs become resident while the last one
// drains, and wait_for_previous() holds them until everything before is complete and visible. What the launch before wrote was not
// constant while this one ran, so it is never read through the read-only path (__ldg, const __restrict__): by plain loads or __ldcg.
// Before its wait a kernel reads the call's inputs and nothing that the call has made, however many launches ago: a wait is what makes that
// visible. CTAs that only clear rows of the result wait for nothing; every launch has others that do, so its end is the end of all before.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    let_next_start();
}

template<typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), uint64_t grid, uint32_t block, uint32_t smem, cudaStream_t stream, bool dependent, A... args) {
    if (smem > 40 * 1024) {   // with what the kernel declares (8 KB at most), more than the 48 KB that it gets unasked
        const cudaError_t e = allow_shared(kernel, smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((uint32_t) grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

// ---- stable counting sort -------------------------------------------------------------------------------------
// One pass places every item behind all items of a smaller digit and behind the items of its own digit that came before it.
// A CTA takes a tile of consecutive items, each of its warps a run of 256, 32 at a time: a lane's rank among the items of
// its digit is the warp's running count plus the equal digits at lower lanes, and a scan over the warps' counts makes it the
// rank in the tile. The order depends on nothing but the keys (atomics only add up counts, in shared memory). Few launches count most here (the data are 6 to 10
// bytes an item): up to kFew items are sorted by one launch that compares each with all, more by two launches a pass while every CTA
// of the second can add up the counts of all tiles, else by three. A launch takes 2 to 4 us of latency, whatever its size. Tiles are
// small because their items' scattered stores leave an SM at one sector a cycle: in tiles of 8,192 a pass over 100,000 ids took 31 us,
// in tiles of 2,048 it takes 10.
struct Digit {
    uint32_t limit, shift, bits;   // keys beyond limit count as limit; bits: of the digit
    __device__ __forceinline__ uint32_t of(uint32_t key) const { return (min(key, limit) >> shift) & ((1u << bits) - 1); }
};

// Keys alone, or in the first half of items that an earlier pass has placed (the second: an item's value).
struct Keys {
    const uint32_t *plain;
    const uint2 *items;
    __device__ __forceinline__ uint2 item(uint32_t i) const { return items ? items[i] : make_uint2(plain[i], i); }
    __device__ __forceinline__ uint32_t key(uint32_t i) const { return items ? items[i].x : plain[i]; }
};

// Bytes [lo, hi) from `at` on, multiples of 2, cleared by a CTA in words of 16 bytes but for the ends; `skip(first, last)` names words
// (by their first and last byte) that are left to the caller.
template<typename Skip>
__device__ __forceinline__ void clear_bytes(uint8_t *at, uint64_t lo, uint64_t hi, Skip skip) {
    const uint64_t base = reinterpret_cast<uintptr_t>(at);
    const uint64_t up = ((base + lo + 15) & ~(uint64_t) 15) - base, down = ((base + hi) & ~(uint64_t) 15) - base;
    const uint64_t first = up < hi ? up : hi, last = down > first && down <= hi ? down : first;
    for (uint64_t o = first + threadIdx.x * 16ull; o < last; o += blockDim.x * 16ull)
        if (!skip((uint32_t) (o - lo), (uint32_t) (o - lo) + 15)) __stcg(reinterpret_cast<uint4 *>(at + o), make_uint4(0, 0, 0, 0));
    const uint32_t head = (uint32_t) (first - lo) / 2, tail = (uint32_t) (hi - last) / 2;
    if (threadIdx.x < head + tail) {   // at most 7 halves each
        const uint64_t o = threadIdx.x < head ? lo + 2 * threadIdx.x : last + 2 * (threadIdx.x - head);
        if (!skip((uint32_t) (o - lo), (uint32_t) (o - lo) + 1)) *reinterpret_cast<uint16_t *>(at + o) = 0;
    }
}

// Rows that CTAs without a tile clear while the others sort (the memory is idle then).
struct Clear {
    uint8_t *at;
    uint64_t stride, bytes;    // of a row
    uint32_t rows, each;       // all rows, and those of a CTA
    __host__ __device__ uint32_t blocks() const { return rows == 0 ? 0 : (rows - 1) / each + 1; }
    // Touches nothing that the launches before it read or write, so it waits for none of them.
    __device__ __forceinline__ void block(uint32_t b) const {
        let_next_start();
        const uint64_t r0 = b * each, r1 = min((uint32_t) r0 + each, rows);
        const auto none = [](uint32_t, uint32_t) { return false; };
        if (stride == bytes) return clear_bytes(at, r0 * bytes, r1 * bytes, none);
        for (uint64_t r = r0; r < r1; r++) clear_bytes(at + r * stride, 0, bytes, none);
    }
};

__device__ __forceinline__ uint32_t tile_item(uint32_t r) {   // of this thread, from the tile's first
    return (threadIdx.x >> 5) * (kRounds * 32) + r * 32 + (threadIdx.x & 31u);
}

// Ranks in the tile of this thread's items by their digits (kNone: no item), and the tile's count of each bucket through `put`;
// warp_counts (a counter for each warp and bucket) has been zeroed by the CTA.
// Lanes of the same digit are found by a ballot for each bit of it.
template<typename Put>
__device__ __forceinline__ void rank_tile(const uint32_t (&d)[kRounds], uint32_t bits, uint32_t buckets, uint16_t *warp_counts, uint32_t (&rank)[kRounds], Put put) {
    const uint32_t warps = blockDim.x >> 5, lane = threadIdx.x & 31u;
    uint32_t same[kRounds];
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) same[r] = __ballot_sync(0xffffffffu, d[r] != kNone);
    for (uint32_t b = 0; b < bits; b++) {
#pragma unroll
        for (uint32_t r = 0; r < kRounds; r++) {
            const bool set = d[r] >> b & 1u;
            const uint32_t others = __ballot_sync(0xffffffffu, set);
            same[r] &= set ? others : ~others;
        }
    }
    __syncthreads();
    uint16_t *mine = warp_counts + (threadIdx.x >> 5) * buckets;
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) {
        const bool there = d[r] != kNone;
        const uint32_t before = there ? mine[d[r]] : 0;
        rank[r] = before + __popc(same[r] & ((1u << lane) - 1));
        __syncwarp();
        if (there && (same[r] >> lane) == 1u) mine[d[r]] = (uint16_t) (before + __popc(same[r]));
        __syncwarp();
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += blockDim.x) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < warps; w++) {
            const uint32_t c = warp_counts[w * buckets + b];
            warp_counts[w * buckets + b] = (uint16_t) sum;
            sum += c;
        }
        put(b, sum);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++)
        if (d[r] != kNone) rank[r] += mine[d[r]];
}

// Counts of a tile lie in whole words of four.
__host__ __device__ constexpr uint32_t count_stride(uint32_t buckets) { return (buckets + 3) & ~3u; }
__host__ __device__ constexpr uint32_t rank_smem(uint32_t warps, uint32_t buckets) { return (warps * buckets + 7) / 8 * 16; }

// Exclusive sums over `buckets` values, in place in shared memory, which the CTA has written.
__device__ __forceinline__ void scan_buckets(uint32_t *values, uint32_t buckets) {
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t all;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint32_t carry = 0;
    for (uint32_t b0 = 0; b0 < buckets; b0 += blockDim.x * 4) {
        __syncthreads();
        const uint32_t b = b0 + threadIdx.x * 4;
        uint32_t v[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = b + i < buckets ? values[b + i] : 0;
            sum += v[i];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= (uint32_t) off) incl += o;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        if (warp == 0) {
            uint32_t w = lane < warps ? warp_sum[lane] : 0, run = w;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, run, off);
                if (lane >= (uint32_t) off) run += o;
            }
            warp_sum[lane] = run - w;
            if (lane == 31) all = run;
        }
        __syncthreads();
        uint32_t run = carry + warp_sum[warp] + incl - sum;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (b + i < buckets) values[b + i] = run;
            run += v[i];
        }
        carry += all;
    }
    __syncthreads();
}

// Where a pass leaves its items. A radix sort: key and value in their new order.
struct ToSorted {
    uint2 *items;
    __device__ __forceinline__ void item(uint2 item, const Digit &digit, uint32_t place) const { items[place] = make_uint2(min(item.x, digit.limit), item.y); }
    __device__ __forceinline__ void start(uint32_t, uint32_t) const {}
};

// Dispatch: the place of every pair, the row at every place, the first place of every partition. Pairs without a partition are
// the last bucket, so that the tail of the map is theirs.
struct ToPlaces {
    uint32_t *position, *map, *segment_start;
    Div choices;
    __device__ __forceinline__ void item(uint2 item, const Digit &digit, uint32_t place) const {
        const bool there = item.x < digit.limit;
        position[item.y] = there ? place : kNone;
        map[place] = there ? choices.of(item.y) : kNone;
    }
    __device__ __forceinline__ void start(uint32_t bucket, uint32_t place) const { segment_start[bucket] = place; }
};

__global__ void __launch_bounds__(kTileThreads) bucket_count_kernel(Keys keys, uint32_t items, Digit digit, uint32_t buckets, uint32_t tiles,
                                                                    uint32_t *__restrict__ counts, uint16_t *__restrict__ ranks, Clear clear) {
    extern __shared__ __align__(16) uint16_t warp_counts[];
    if (blockIdx.x >= tiles) return clear.block(blockIdx.x - tiles);
    for (uint32_t i = threadIdx.x; i < rank_smem(kTileThreads / 32, buckets) / 16; i += kTileThreads) reinterpret_cast<uint4 *>(warp_counts)[i] = make_uint4(0, 0, 0, 0);
    wait_for_previous();
    const uint32_t first = blockIdx.x * kTile;
    uint32_t d[kRounds], rank[kRounds];
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) {
        const uint32_t i = first + tile_item(r);
        d[r] = i < items ? digit.of(keys.key(i)) : kNone;
    }
    const uint32_t stride = count_stride(buckets);
    uint32_t *mine = counts + (uint64_t) blockIdx.x * stride;
    if (threadIdx.x < stride - buckets) mine[buckets + threadIdx.x] = 0;
    rank_tile(d, digit.bits, buckets, warp_counts, rank, [&](uint32_t b, uint32_t sum) { mine[b] = sum; });
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) {
        const uint32_t i = first + tile_item(r);
        if (i < items) ranks[i] = (uint16_t) rank[r];
    }
}

// The counts of all tiles become, bucket by bucket, counts of the tiles before, and totals.
__global__ void __launch_bounds__(1024) bucket_scan_kernel(uint32_t *__restrict__ counts, uint32_t tiles, uint32_t buckets,
                                                           uint32_t *__restrict__ totals, Clear clear) {
    __shared__ uint32_t part[32][33];
    const uint32_t blocks = (buckets + 31) / 32;
    if (blockIdx.x >= blocks) return clear.block(blockIdx.x - blocks);
    wait_for_previous();
    const uint32_t stride = count_stride(buckets);
    const uint32_t x = threadIdx.x & 31u, y = threadIdx.x >> 5;
    const uint32_t b = blockIdx.x * 32 + x;
    const uint32_t each = (tiles + 31) / 32, t0 = min(y * each, tiles), t1 = min(t0 + each, tiles);
    uint32_t sum = 0;
    if (b < buckets) {
#pragma unroll 8
        for (uint32_t t = t0; t < t1; t++) sum += counts[(uint64_t) t * stride + b];
    }
    part[y][x] = sum;
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t i = 0; i < y; i++) run += part[i][x];
    if (b < buckets) {
#pragma unroll 8
        for (uint32_t t = t0; t < t1; t++) {
            const uint32_t c = counts[(uint64_t) t * stride + b];
            counts[(uint64_t) t * stride + b] = run;
            run += c;
        }
        if (y == 31) totals[b] = run;
    }
}

template<typename To, bool kScanned>
__global__ void __launch_bounds__(kTileThreads) bucket_place_kernel(Keys keys, uint32_t items, Digit digit, uint32_t buckets, uint32_t tiles,
                                                                    const uint32_t *counts, const uint32_t *totals, const uint16_t *ranks, To to, Clear clear) {
    extern __shared__ __align__(16) uint32_t base[];   // of each bucket: all items of smaller ones; then, behind, its items in the tiles before
    if (blockIdx.x >= tiles) return clear.block(blockIdx.x - tiles);
    const uint32_t stride = count_stride(buckets);
    uint32_t *before = base + stride;
    const uint32_t first = blockIdx.x * kTile;
    uint2 item[kRounds];
    uint32_t rank[kRounds];
    const bool given = keys.items == nullptr;   // by the caller: they need not wait, as items that an earlier pass has placed do
    if (given) {
#pragma unroll
        for (uint32_t r = 0; r < kRounds; r++) item[r] = keys.item(min(first + r * kTileThreads + threadIdx.x, items - 1));
    }
    if (!kScanned)
        for (uint32_t b = threadIdx.x; b < 2 * stride; b += kTileThreads) base[b] = 0;
    wait_for_previous();
    if (!given) {
#pragma unroll
        for (uint32_t r = 0; r < kRounds; r++) item[r] = __ldcg(keys.items + min(first + r * kTileThreads + threadIdx.x, items - 1));
    }
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) rank[r] = __ldcg(ranks + min(first + r * kTileThreads + threadIdx.x, items - 1));
    if constexpr (kScanned) {
        for (uint32_t b = threadIdx.x; b < buckets; b += kTileThreads) {
            base[b] = __ldcg(totals + b);
            before[b] = __ldcg(counts + (uint64_t) blockIdx.x * stride + b);
        }
    } else {
        // four buckets a thread; where that leaves threads over, groups of them share the tiles
        const uint32_t quads = stride / 4, across = min(quads, kTileThreads), groups = kTileThreads / across, group = threadIdx.x / across;
        __syncthreads();
        const uint32_t each = (tiles + groups - 1) / groups, t0 = group * each, t1 = min(t0 + each, tiles);
        if (group < groups)
            for (uint32_t q = threadIdx.x - group * across; q < quads; q += across) {
                uint4 all = make_uint4(0, 0, 0, 0), mine = all;
#pragma unroll 16
                for (uint32_t t = t0; t < t1; t++) {
                    const uint4 c = __ldcg(reinterpret_cast<const uint4 *>(counts + t * stride) + q);
                    all.x += c.x; all.y += c.y; all.z += c.z; all.w += c.w;
                    if (t < blockIdx.x) { mine.x += c.x; mine.y += c.y; mine.z += c.z; mine.w += c.w; }
                }
                atomicAdd(base + 4 * q, all.x); atomicAdd(base + 4 * q + 1, all.y); atomicAdd(base + 4 * q + 2, all.z); atomicAdd(base + 4 * q + 3, all.w);
                atomicAdd(before + 4 * q, mine.x); atomicAdd(before + 4 * q + 1, mine.y); atomicAdd(before + 4 * q + 2, mine.z); atomicAdd(before + 4 * q + 3, mine.w);
            }
    }
    scan_buckets(base, buckets);
    if (blockIdx.x == 0)
        for (uint32_t b = threadIdx.x; b < buckets; b += kTileThreads) to.start(b, base[b]);
#pragma unroll
    for (uint32_t r = 0; r < kRounds; r++) {
        const uint32_t d = digit.of(item[r].x);
        if (first + r * kTileThreads + threadIdx.x < items) to.item(item[r], digit, base[d] + before[d] + rank[r]);
    }
}

// Few items: an item's place is the number of smaller keys and of equal ones before it. A CTA holds all keys in shared memory, `few_keys`
// fills them; a warp counts for one item.
__device__ __forceinline__ void few_keys(const uint32_t *__restrict__ keys, uint32_t items, uint32_t limit, uint4 *all) {
    uint32_t *to = reinterpret_cast<uint32_t *>(all);
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < (items + 3) / 4 * 4; i += blockDim.x) to[i] = i < items ? min(keys[i], limit) : kNone;
}
__device__ __forceinline__ uint32_t few_place(const uint4 *all, uint32_t items, uint32_t item, uint32_t key) {
    // keys before the item count when they are not greater, those behind it when they are smaller
    const uint32_t lane = threadIdx.x & 31u, quads = (items + 3) / 4, own = item / 4;
    uint32_t before = 0, q = lane;
#pragma unroll 4
    for (; q < own; q += 32) {
        const uint4 k = all[q];
        before += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
    }
    if (q == own) {
        const uint4 k = all[q];
        const uint32_t in = item & 3u;
        before += (in > 0 ? k.x <= key : 0) + (in > 1 ? k.y <= key : k.y < key) + (in > 2 ? k.z <= key : k.z < key) + (k.w < key);
        q += 32;
    }
#pragma unroll 4
    for (; q < quads; q += 32) {
        const uint4 k = all[q];
        before += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    }
    return __reduce_add_sync(0xffffffffu, before);
}

__global__ void __launch_bounds__(256) few_sort_kernel(const uint32_t *__restrict__ keys, uint32_t items, uint32_t limit, uint2 *__restrict__ sorted, Clear clear) {
    __shared__ uint4 all[kFew / 4];
    const uint32_t blocks = (items + 7) / 8;
    if (blockIdx.x >= blocks) return clear.block(blockIdx.x - blocks);
    wait_for_previous();
    few_keys(keys, items, limit, all);
    __syncthreads();
    const uint32_t i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= items) return;
    const uint32_t key = reinterpret_cast<const uint32_t *>(all)[i], place = few_place(all, items, i, key);
    if ((threadIdx.x & 31u) == 0) sorted[place] = make_uint2(key, i);
}

// ---- gradient of a lookup ---------------------------------------------------------------------------------------
struct GradArgs {
    const uint2 *sorted;             // by id: the id, and the row of the gradient
    uint32_t items, n, dim, words, lanes, slabs, chunk;   // words: pieces of a row
    float scale;
    int accumulate;
    float *partial;                  // at (2 * chunk + which) * dim: sums of runs that leave their chunk
    Div by_row_bytes;                // of the table's gradient
    uint32_t join_blocks, clear_from, clear_rows;   // CTAs that join; the others clear clear_rows rows each, from row clear_from on
    __device__ __forceinline__ uint32_t key(uint64_t i) const { return sorted[i].x; }
};

template<int V, typename O>
__device__ __forceinline__ void put_grad(const Rows<O> &out, const GradArgs &a, uint32_t id, uint32_t word, float (&acc)[V]) {
    O *p = out.row(id) + word * V;
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

// The first of the sorted keys from `lo` on that is not below `key`; the CTA narrows the range by its width at each step.
__device__ __forceinline__ uint32_t first_not_below(const uint2 *sorted, uint32_t lo, uint32_t hi, uint32_t key) {
    while (lo < hi) {
        const uint32_t step = (hi - lo + blockDim.x - 1) / blockDim.x;
        const uint64_t i = lo + (uint64_t) threadIdx.x * step;
        const uint32_t below = __syncthreads_count(i < hi && sorted[i].x < key);
        if (below == 0) break;
        const uint64_t end = lo + (uint64_t) below * step;
        lo += (below - 1) * step + 1;
        if (end < hi) hi = (uint32_t) end;
    }
    return lo;
}

// Of rows [r0, r1), at most 256, those that an id names: by the sorted items.
__device__ __forceinline__ void name_rows(const GradArgs &a, uint32_t r0, uint32_t r1, uint32_t *named) {
    uint32_t at = first_not_below(a.sorted, 0, a.items, r0);
    bool more = at < a.items;
    for (int step = 0; step < 2 && more; step++) {   // mostly a few items: all of them are looked at
        const uint32_t i = at + threadIdx.x, key = i < a.items ? a.key(i) : kNone;
        if (key < r1) atomicOr(&named[(key - r0) >> 5], 1u << ((key - r0) & 31u));
        more = __syncthreads_count(key < r1) == blockDim.x;
        at += blockDim.x;
    }
    if (more && r0 + threadIdx.x < r1) {   // ids that come often: each row is searched for
        const uint32_t r = r0 + threadIdx.x;
        uint32_t lo = at, hi = a.items;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.key(mid) < r) lo = mid + 1;
            else hi = mid;
        }
        if (lo < a.items && a.key(lo) == r) atomicOr(&named[(r - r0) >> 5], 1u << ((r - r0) & 31u));
    }
}

// Rows [r0, r1) that `mark` does not name are cleared.
template<typename O, typename Mark>
__device__ __forceinline__ void clear_rows(const Rows<O> &out, uint32_t dim, const Div &by_row_bytes, uint32_t r0, uint32_t r1, Mark mark) {
    __shared__ uint32_t named[256 / 32];
    if (threadIdx.x < 8) named[threadIdx.x] = 0;
    __syncthreads();
    mark(named);
    __syncthreads();
    uint8_t *at = reinterpret_cast<uint8_t *>(out.row(r0));
    const uint64_t row_bytes = (uint64_t) dim * sizeof(O);
    if (out.stride == dim && row_bytes >= 16) {   // a word of 16 bytes lies in two rows at most; one that lies in a named and another one goes out in halves
        const auto is_named = [&](uint32_t byte) {
            const uint32_t r = by_row_bytes.of(byte);
            return (named[r >> 5] >> (r & 31u) & 1u) != 0;
        };
        clear_bytes(at, 0, (r1 - r0) * row_bytes, [&](uint32_t first, uint32_t last) {
            const bool x = is_named(first), y = is_named(last);
            if (x != y)
                for (uint32_t o = first; o < last; o += 2)
                    if (!is_named(o)) *reinterpret_cast<uint16_t *>(at + o) = 0;
            return x || y;
        });
    } else if (row_bytes >= 256) {
        for (uint32_t r = 0; r < r1 - r0; r++)
            if (!(named[r >> 5] >> (r & 31u) & 1u)) clear_bytes(at + r * out.stride * sizeof(O), 0, row_bytes, [](uint32_t, uint32_t) { return false; });
    } else {
        for (uint32_t x = threadIdx.x; x < (r1 - r0) * dim; x += blockDim.x) {
            const uint32_t r = x / dim;
            if (!(named[r >> 5] >> (r & 31u) & 1u)) out.row(r0 + r)[x - r * dim] = from_float<O>(0.0f);
        }
    }
}

// A group of lanes joins a chunk of sorted items over a slab of the row: the sum of a run of equal ids goes to the id's row, or,
// where the run goes on in another chunk, to the chunk's partial sums (first: it came from the chunk before). Consecutive items of a
// sorted list make equal shares of any distribution of ids, be it one id. The other CTAs clear the rows that no id names.
// 32,768 tokens over 131,072 rows of 8 KB (1.3 GB with the cleared rows): 221 us with its sort, 93 % of the copy rate; 100,000 ids over a
// million rows of 512 bytes: 105 us, 82 %, of which the sort's latency is the rest.
template<typename T, typename O, int V>
__global__ void __launch_bounds__(256, 4) grad_join_kernel(Rows<const T> grad, Rows<O> out, GradArgs a) {
    constexpr int U = in_flight(64, V * (int) sizeof(T), 8);
    wait_for_previous();
    if (blockIdx.x >= a.join_blocks) {
        const uint64_t r0 = a.clear_from + (uint64_t) (blockIdx.x - a.join_blocks) * a.clear_rows;
        const uint32_t r1 = (uint32_t) min((uint64_t) a.n, r0 + a.clear_rows);
        return clear_rows(out, a.dim, a.by_row_bytes, (uint32_t) r0, r1, [&](uint32_t *named) { name_rows(a, (uint32_t) r0, r1, named); });
    }
    const uint32_t group = (blockIdx.x * 256 + threadIdx.x) / a.lanes, lane = threadIdx.x & (a.lanes - 1);
    const uint32_t chunk = group / a.slabs, word = (group - chunk * a.slabs) * a.lanes + lane;
    const uint64_t c0 = (uint64_t) chunk * a.chunk;
    if (c0 >= a.items || word >= a.words) return;
    const uint32_t c1 = (uint32_t) min(c0 + a.chunk, (uint64_t) a.items);
    uint32_t id = a.key(c0);
    bool from_left = c0 > 0 && a.key(c0 - 1) == id;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    auto leave = [&](bool to_right) {
        if (id >= a.n) return;
        if (from_left || to_right) store<float, V>(a.partial + (2ull * chunk + (from_left ? 0 : 1)) * a.dim + word * V, acc);
        else put_grad<V>(out, a, id, word, acc);
    };
    uint2 next[U];   // items of the batch to come: their rows can be fetched without waiting for them
#pragma unroll
    for (int u = 0; u < U; u++) next[u] = a.sorted[min((uint32_t) c0 + u, c1 - 1)];
    for (uint32_t c = (uint32_t) c0; c < c1; c += U) {
        uint32_t key[U];
        Piece<T, V, true> piece[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            key[u] = next[u].x;
            piece[u] = fetch<V, true>(grad, grad.row(next[u].y), (int32_t) (word * V), a.dim, key[u] < a.n && c + u < c1);
        }
#pragma unroll
        for (int u = 0; u < U; u++) next[u] = a.sorted[min(c + U + u, c1 - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c + u >= c1) break;
            if (key[u] != id) {
                leave(false);
                id = key[u];
                from_left = false;
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] = 0.0f;
            }
            if (id < a.n) {
                float f[V];
                unpack<T, V>(piece[u].word(), f);
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += f[i];
            }
        }
    }
    leave(c1 < a.items && a.key(c1) == id);
}

// Few ids: everything in one launch. A CTA owns one id, unless an earlier one is equal: it lists the equal ones in order, its groups of
// lanes add consecutive parts of the list and the groups' sums are added in order. The other CTAs clear the rows that no id names.
// Rows of 64 bf16: 10 ids 3.0 us, 1,000 ids 7.5, against 7.3 and 10.5 by three launches.
template<typename T, typename O, int V>
__global__ void __launch_bounds__(256) grad_few_kernel(Rows<const T> grad, Rows<O> out, const uint32_t *__restrict__ ids, GradArgs a) {
    constexpr int U = 8;
    __shared__ uint32_t keys[kFewIds], counts[8];
    __shared__ uint16_t list[kFewIds];
    __shared__ float part[256][V];
    for (uint32_t i = threadIdx.x; i < a.items; i += 256) keys[i] = ids[i];
    __syncthreads();
    if (blockIdx.x >= a.items) {
        const uint64_t r0 = (uint64_t) (blockIdx.x - a.items) * a.clear_rows;
        const uint32_t r1 = (uint32_t) min((uint64_t) a.n, r0 + a.clear_rows);
        return clear_rows(out, a.dim, a.by_row_bytes, (uint32_t) r0, r1, [&](uint32_t *named) {
            for (uint32_t i = threadIdx.x; i < a.items; i += 256)
                if (keys[i] >= r0 && keys[i] < r1) atomicOr(&named[(keys[i] - (uint32_t) r0) >> 5], 1u << ((keys[i] - (uint32_t) r0) & 31u));
        });
    }
    const uint32_t id = keys[blockIdx.x], warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    bool earlier = id >= a.n;
    for (uint32_t i = threadIdx.x; i < blockIdx.x; i += 256) earlier |= keys[i] == id;
    if (__syncthreads_or(earlier)) return;
    const uint32_t segment = (a.items + 7) / 8, i0 = min(warp * segment, a.items), i1 = min(i0 + segment, a.items);
    uint32_t found = 0;
    for (uint32_t i = i0; i < i1; i += 32) found += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && keys[i + lane] == id));
    if (lane == 0) counts[warp] = found;
    __syncthreads();
    uint32_t all = 0, at = 0;
#pragma unroll
    for (uint32_t w = 0; w < 8; w++) {
        at += w < warp ? counts[w] : 0;
        all += counts[w];
    }
    for (uint32_t i = i0; i < i1; i += 32) {
        const bool equal = i + lane < i1 && keys[i + lane] == id;
        const uint32_t lanes = __ballot_sync(0xffffffffu, equal);
        if (equal) list[at + __popc(lanes & ((1u << lane) - 1))] = (uint16_t) (i + lane);
        at += __popc(lanes);
    }
    __syncthreads();
    const uint32_t group = threadIdx.x / a.lanes, groups = 256 / a.lanes, each = (all + groups - 1) / groups;
    const uint32_t s0 = min(group * each, all), s1 = min(s0 + each, all);
    for (uint32_t word = threadIdx.x & (a.lanes - 1); word < a.words; word += a.lanes) {   // more than once only where one group has the row
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = 0.0f;
        for (uint32_t s = s0; s < s1; s += U) {
            Piece<T, V, true> piece[U];
#pragma unroll
            for (int u = 0; u < U; u++) piece[u] = fetch<V, true>(grad, grad.row(list[min(s + u, s1 - 1)]), (int32_t) (word * V), a.dim, s + u < s1);
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (s + u >= s1) break;
                float f[V];
                unpack<T, V>(piece[u].word(), f);
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += f[i];
            }
        }
        if (groups == 1) {
            put_grad<V>(out, a, id, word, acc);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) part[threadIdx.x][i] = acc[i];
        }
    }
    if (groups == 1) return;
    __syncthreads();
    if (threadIdx.x >= a.words) return;   // fewer than a group's lanes: the first group
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = part[threadIdx.x][i];
    const uint32_t used = (all + each - 1) / each;
    for (uint32_t g = 1; g < used; g++)
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += part[g * a.lanes + threadIdx.x][i];
    put_grad<V>(out, a, id, threadIdx.x, acc);
}

// Runs over several chunks, whose first chunk's unit (a chunk and a slab) adds their partial sums and writes the row. A warp owns a unit and
// adds short runs by itself, in order; the CTA's warps share the runs with more partial sums than kLongRun, each takes consecutive ones,
// and the warps' sums are added in order.
constexpr uint32_t kLongRun = 16;
template<typename O, int V>
__global__ void __launch_bounds__(256) grad_fix_kernel(Rows<O> out, GradArgs a, uint32_t units) {
    __shared__ float part[8][32][V];
    __shared__ uint32_t long_last[8];
    wait_for_previous();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    auto add = [&](uint32_t chunk, uint32_t word, uint32_t s0, uint32_t s1, float (&acc)[V]) {   // partial sums s0 .. s1 - 1 of the run that starts in chunk
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = 0.0f;
        constexpr int U = in_flight(128, 4 * V, 8);
        for (uint32_t s = s0; s < s1; s += U) {
            float f[U][V];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t i = min(s + u, s1 - 1);
                load<float, V>(a.partial + (2ull * (chunk + i) + (i == 0 ? 1 : 0)) * a.dim + word * V, f[u]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (s + u >= s1) break;
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += f[u][i];
            }
        }
    };
    const uint32_t unit = blockIdx.x * 8 + warp, starts = units / a.slabs;   // chunk by chunk, so that the slabs of a long run fall to several CTAs
    uint32_t last = 0;   // the run's last chunk; 0: no run starts here and goes on
    if (unit < units) {
        const uint32_t slab = unit / starts, chunk = unit - slab * starts, word = slab * a.lanes + lane;
        const uint64_t c0 = (uint64_t) chunk * a.chunk, c1 = c0 + a.chunk;   // below a.items, as the last chunk has no unit
        const uint32_t id = a.key(c1 - 1);
        if (id < a.n && a.key(c1) == id && !(a.key(c0) == id && c0 > 0 && a.key(c0 - 1) == id)) {
            // the first chunk boundary that the run does not cross, among the next 32 at a time
            uint32_t c = chunk + 1;
            while (true) {
                const uint64_t end = (uint64_t) (c + lane + 1) * a.chunk;
                const uint32_t beyond = __ballot_sync(0xffffffffu, end >= a.items || a.key(end < a.items ? end : 0) != id);
                if (beyond) {
                    last = c + __ffs(beyond) - 1;
                    break;
                }
                c += 32;
            }
            if (last - chunk < kLongRun && lane < a.lanes && word < a.words) {
                float acc[V];
                add(chunk, word, 0, last - chunk + 1, acc);
                put_grad<V>(out, a, id, word, acc);
            }
            if (last - chunk < kLongRun) last = 0;
        }
    }
    if (lane == 0) long_last[warp] = last;
    if (!__syncthreads_or(last)) return;
    // the CTA's long runs, one after another or, two or four, at once: `each` warps to a run
    uint32_t found = 0, units_of[8];
#pragma unroll
    for (uint32_t u = 0; u < 8; u++)
        if (long_last[u] != 0) units_of[found++] = u;
    const uint32_t at_once = found >= 4 ? 4 : found >= 2 ? 2 : 1, each = 8 / at_once, share = warp & (each - 1);
    for (uint32_t f = 0; f < found; f += at_once) {
        const bool there = f + warp / each < found;
        const uint32_t u = units_of[there ? f + warp / each : 0];
        const uint32_t slab = (blockIdx.x * 8 + u) / starts, chunk = blockIdx.x * 8 + u - slab * starts, word = slab * a.lanes + lane;
        const uint32_t sums = long_last[u] - chunk + 1, part_sums = (sums + each - 1) / each, s0 = min(share * part_sums, sums), s1 = min(s0 + part_sums, sums);
        const bool mine = there && lane < a.lanes && word < a.words;
        float acc[V];
        if (mine) {
            add(chunk, word, s0, s1, acc);
#pragma unroll
            for (int i = 0; i < V; i++) part[warp][lane][i] = acc[i];
        }
        __syncthreads();
        if (share == 0 && mine) {
            for (uint32_t w = 1; w < each; w++)
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += part[warp + w][lane][i];
            put_grad<V>(out, a, a.key((uint64_t) (chunk + 1) * a.chunk - 1), word, acc);
        }
        __syncthreads();
    }
}

// ---- dispatch ---------------------------------------------------------------------------------------------------
// Each row, read once, is copied to the places of its pairs. A thread has U words of rows in flight. 16,384 x 8 rows of 4 KB: 93 us
// of 104 with the sort, bound by the writes (5.6 TB/s). The other way round, sorted rows fetched by the map and written one behind the
// other, takes 138: each row is read eight times.
template<typename T, int V, int U>
__global__ void __launch_bounds__(256) dispatch_kernel(Rows<const T> rows, uint32_t dim, uint32_t units, Div words, uint32_t choices,
                                                       const uint32_t *position, Rows<T> sorted) {
    constexpr int K = 8;   // places that are fetched before a piece goes to any of them
    const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t row[U], at[U];
    Piece<T, V, true> piece[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t x = min(first + u * 256, units - 1);
        row[u] = words.of(x);
        at[u] = (x - row[u] * words.d) * V;
        piece[u] = fetch<V, true>(rows, rows.row(row[u]), (int32_t) at[u], dim, true);
    }
    wait_for_previous();   // the places come from the launch before, the rows do not
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (first + u * 256 >= units) break;
        for (uint32_t j0 = 0; j0 < choices; j0 += K) {
            uint32_t p[K];
#pragma unroll
            for (int j = 0; j < K; j++) p[j] = j0 + j < choices ? position[(uint64_t) row[u] * choices + j0 + j] : kNone;
#pragma unroll
            for (int j = 0; j < K; j++)
                if (p[j] != kNone) __stcg(reinterpret_cast<WordOf<T, V> *>(sorted.row(p[j]) + at[u]), piece[u].a);
        }
    }
}

// The same with a warp a row, for many long rows.
template<typename T, int V, int U>
__global__ void __launch_bounds__(256) dispatch_long_kernel(Rows<const T> rows, uint32_t dim, uint32_t count, uint32_t words, uint32_t choices,
                                                            const uint32_t *position, Rows<T> sorted) {
    constexpr int K = 4;
    wait_for_previous();
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= count) return;
    const T *from = rows.row(row);
    position += (uint64_t) row * choices;
    for (uint32_t c = threadIdx.x & 31u; c < words; c += 32 * U) {
        Piece<T, V, true> piece[U];
#pragma unroll
        for (int u = 0; u < U; u++) piece[u] = fetch<V, true>(rows, from, (int32_t) ((c + u * 32) * V), dim, c + u * 32 < words);
        for (uint32_t j0 = 0; j0 < choices; j0 += K) {
            uint32_t p[K];
#pragma unroll
            for (int j = 0; j < K; j++) p[j] = j0 + j < choices ? position[j0 + j] : kNone;
#pragma unroll
            for (int j = 0; j < K; j++) {
                if (p[j] == kNone) continue;
                T *to = sorted.row(p[j]) + c * V;
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (c + u * 32 < words) __stcg(reinterpret_cast<WordOf<T, V> *>(to + u * 32 * V), piece[u].a);
            }
        }
    }
}

// Few pairs: everything in one launch. A CTA owns one row; a warp finds a pair's place by comparing it with all pairs, then the CTA
// copies the row. One CTA more counts the partitions.
template<typename T, int V>
__global__ void __launch_bounds__(256) dispatch_small_kernel(Rows<const T> rows, uint32_t dim, uint32_t count, uint32_t words,
                                                             const uint32_t *__restrict__ choice, uint32_t choices, uint32_t partitions, Rows<T> sorted,
                                                             uint32_t *__restrict__ position, uint32_t *__restrict__ map, uint32_t *__restrict__ segment_start) {
    __shared__ uint4 all[kFewPairs / 4];
    __shared__ uint32_t place[kMaxChoices];
    extern __shared__ __align__(16) uint32_t counts[];
    const uint32_t pairs = count * choices, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, row = blockIdx.x;
    if (row == count) {
        for (uint32_t b = threadIdx.x; b <= partitions; b += 256) counts[b] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < pairs; i += 256) {
            const uint32_t e = choice[i];
            if (e < partitions) atomicAdd(counts + e, 1u);
        }
        scan_buckets(counts, partitions + 1);
        for (uint32_t b = threadIdx.x; b <= partitions; b += 256) segment_start[b] = counts[b];
        return;
    }
    few_keys(choice, pairs, partitions, all);
    const T *from = rows.row(row);
    Piece<T, V, true> piece{};   // fetched before the places are known
    if (threadIdx.x < words) piece = fetch<V, true>(rows, from, (int32_t) (threadIdx.x * V), dim, true);
    __syncthreads();
    for (uint32_t j = warp; j < choices; j += 8) {
        const uint32_t pair = row * choices + j, key = reinterpret_cast<const uint32_t *>(all)[pair], before = few_place(all, pairs, pair, key);
        if (lane == 0) {
            const bool there = key < partitions;
            place[j] = position[pair] = there ? before : kNone;
            map[before] = there ? row : kNone;
        }
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < words; c += 256) {
        if (c != threadIdx.x) piece = fetch<V, true>(rows, from, (int32_t) (c * V), dim, true);
        for (uint32_t j = 0; j < choices; j++)
            if (place[j] != kNone) __stcg(reinterpret_cast<WordOf<T, V> *>(sorted.row(place[j]) + c * V), piece.a);
    }
}

// ---- combine ----------------------------------------------------------------------------------------------------
// out[t] = sum over j, ascending, of weight[t,j] * sorted[position[t,j]]; K pairs' pieces are in flight for each piece of a row: as many
// as there are choices, up to 8. 16,384 x 8 rows of 4 KB: 96 us, 94 % of the copy rate.
template<typename T, int V, bool kWhole, int K>
__global__ void __launch_bounds__(256) combine_kernel(Rows<const T> sorted, uint32_t sorted_rows, uint32_t dim, const uint32_t *__restrict__ position,
                                                      uint32_t choices, const float *__restrict__ weights, uint32_t units, Div words, Rows<T> out) {
    const uint32_t x = blockIdx.x * 256 + threadIdx.x;
    if (x >= units) return;
    const uint32_t row = words.of(x);
    T *to = out.row(row);
    const int32_t at = piece_start<V, kWhole>(to, x - row * words.d);
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    for (uint32_t j0 = 0; j0 < choices; j0 += K) {
        uint32_t p[K];
        float w[K];
        Piece<T, V, kWhole> y[K];
#pragma unroll
        for (int j = 0; j < K; j++) {
            const uint64_t pair = (uint64_t) row * choices + j0 + j;
            p[j] = j0 + j < choices ? position[pair] : kNone;
            w[j] = weights && j0 + j < choices ? weights[pair] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < K; j++) y[j] = fetch<V, kWhole>(sorted, sorted.row(p[j]), at, dim, p[j] < sorted_rows);
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (p[j] >= sorted_rows) continue;
            float f[V];
            unpack<T, V>(y[j].word(), f);
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] = fmaf(w[j], f[i], acc[i]);
        }
    }
    put<V, kWhole>(to, at, dim, acc);
}

// The same with a warp a row, for many long rows: U of its pieces and those of K of its places are in flight.
template<typename T, int V, int K, int U>
__global__ void __launch_bounds__(256) combine_long_kernel(Rows<const T> sorted, uint32_t sorted_rows, uint32_t dim, const uint32_t *__restrict__ position,
                                                           uint32_t choices, const float *__restrict__ weights, uint32_t count, uint32_t words, Rows<T> out) {
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= count) return;
    T *to = out.row(row);
    position += (uint64_t) row * choices;
    uint32_t p[K];
    float w[K];
    auto places = [&](uint32_t j0) {
#pragma unroll
        for (int j = 0; j < K; j++) {
            p[j] = j0 + j < choices ? position[j0 + j] : kNone;
            w[j] = weights && j0 + j < choices ? weights[(uint64_t) row * choices + j0 + j] : 1.0f;
        }
    };
    places(0);
    for (uint32_t c = threadIdx.x & 31u; c < words; c += 32 * U) {
        float acc[U][V];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < V; i++) acc[u][i] = 0.0f;
        for (uint32_t j0 = 0; j0 < choices; j0 += K) {
            if (choices > K) places(j0);
            Piece<T, V, true> y[U][K];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < K; j++)
                    y[u][j] = fetch<V, true>(sorted, sorted.row(p[j]), (int32_t) ((c + u * 32) * V), dim, p[j] < sorted_rows && c + u * 32 < words);
#pragma unroll
            for (int j = 0; j < K; j++) {
                if (p[j] >= sorted_rows) continue;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float f[V];
                    unpack<T, V>(y[u][j].word(), f);
#pragma unroll
                    for (int i = 0; i < V; i++) acc[u][i] = fmaf(w[j], f[i], acc[u][i]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c + u * 32 < words) store<T, V>(to + (c + u * 32) * V, acc[u]);
    }
}

// grad_sorted[position[t,j]] = weight[t,j] * grad[t] and grad_weights[t,j] = <grad[t], sorted[position[t,j]]>: G lanes own a row,
// and have U of its pieces and those of K of its places in flight. A warp a row beats a CTA a row (16,384 x 8 rows of 4 KB: 180 against
// 205 us, 95 % of the copy rate; 39,047 x 4 of 5 KB: 278 against 340) but where rows are few (64 x 8: 9.1 against 3.3; 1,000 x 4 of 8 KB:
// 22 against 16). grad is read once for K places.
template<typename T, int V, int K, int U, int G>
__global__ void __launch_bounds__(256) combine_grad_kernel(Rows<const T> grad, uint32_t count, uint32_t dim, uint32_t words, Rows<const T> sorted, uint32_t sorted_rows,
                                                           const uint32_t *__restrict__ position, uint32_t choices, const float *__restrict__ weights,
                                                           Rows<T> grad_sorted, float *__restrict__ grad_weights) {
    __shared__ float part[8][K];
    const uint32_t row = blockIdx.x * (256 / G) + threadIdx.x / G, l = threadIdx.x % G;
    if (G <= 32 && row >= count) return;
    const T *from = grad.row(row);
    const uint32_t team = G < 32 ? ((1u << G) - 1) << (threadIdx.x & 31u & ~(G - 1u)) : 0xffffffffu;   // the lanes of this row, or of this warp
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
        for (uint32_t c0 = l; c0 < words; c0 += G * U) {
            Piece<T, V, true> x[U], y[U][K];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t c = c0 + u * G;
                const bool in = u == 0 || c < words;
                x[u] = fetch<V, true>(grad, from, (int32_t) (c * V), dim, in);
#pragma unroll
                for (int j = 0; j < K; j++) y[u][j] = fetch<V, true>(sorted, sorted.row(p[j]), (int32_t) (c * V), dim, in && p[j] < sorted_rows);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t c = c0 + u * G;
                if (u > 0 && c >= words) break;
                float g[V];
                unpack<T, V>(x[u].word(), g);
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (p[j] >= sorted_rows) continue;
                    float f[V], o[V];
                    unpack<T, V>(y[u][j].word(), f);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        dot[j] = fmaf(g[i], f[i], dot[j]);
                        o[i] = w[j] * g[i];
                    }
                    store<T, V>(grad_sorted.row(p[j]) + c * V, o);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int off = G < 32 ? G / 2 : 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(team, dot[j], off);
        if (G <= 32) {
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

// ---- rows without a place -------------------------------------------------------------------------------------------
// A bit for each row that a position names, then a CTA looks at the bits of `each` rows (32 to 256, some 128 KB) and clears those without one. Rows
// that are named cost a bit each: 131,072 rows of 4 KB, 2 % of them without a place, take 15 us, as zeros for all of them before take 140.
__global__ void __launch_bounds__(256) mark_places_kernel(const uint32_t *__restrict__ position, uint32_t pairs, uint32_t rows, uint32_t *marks) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    const uint32_t p = i < pairs ? position[i] : kNone;
    if (p < rows) atomicOr(marks + (p >> 5), 1u << (p & 31u));
    let_next_start();
}
template<typename O>
__global__ void __launch_bounds__(256) clear_unplaced_kernel(Rows<O> out, uint32_t rows, uint32_t dim, Div by_row_bytes, uint32_t each, const uint32_t *marks) {
    wait_for_previous();
    const uint32_t r0 = blockIdx.x * each, r1 = r0 + min(each, rows - r0), words = (r1 - r0 + 31) / 32;
    const uint32_t mine = threadIdx.x < words ? __ldcg(marks + r0 / 32 + threadIdx.x) : 0xffffffffu;
    const uint32_t there = threadIdx.x + 1 == words && (r1 & 31u) ? (1u << (r1 & 31u)) - 1 : 0xffffffffu;   // bits of rows that there are
    if (__syncthreads_and((mine & there) == there)) return;
    clear_rows(out, dim, by_row_bytes, r0, r1, [&](uint32_t *named) {
        if (threadIdx.x < words) named[threadIdx.x] = mine;
    });
}

// ---- host side ----------------------------------------------------------------------------------------------------
int fail(glide_ctx *ctx, int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    if (code == GLIDE_ERR_CUDA || code == GLIDE_ERR_NO_MEMORY) cudaGetLastError();   // reported here, not by whoever asks next
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

#define ROWS_CUDA(...)                                                                                       \
    do {                                                                                                     \
        const cudaError_t e_ = (__VA_ARGS__);                                                                \
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
    bool sized() const { return rows == 0 || stride <= (1ull << 60) / rows; }   // its bytes fit 64 bits
    // The most values (1, 2, 4 or 8) that a word may hold so that every word of every row is aligned, words of 16 bytes at most.
    uint32_t width(uint32_t most) const {
        const uint64_t e = bytes_of(type);
        uint32_t v = most;
        for (; v > 1; v >>= 1) {
            const uint64_t word = v * e < 16 ? v * e : 16;
            if (reinterpret_cast<uintptr_t>(p) % word == 0 && (rows <= 1 || stride * e % word == 0) && dim % v == 0) break;
        }
        return v;
    }
    template<typename T> Rows<T> as() const { return Rows<T>{static_cast<T *>(const_cast<void *>(p)), stride, reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes()}; }
    Matrix from(uint64_t r) const { return Matrix{static_cast<const char *>(p) + r * stride * bytes_of(type), rows - r, stride, dim, type}; }
};

bool aligned(const Matrix &m) { return reinterpret_cast<uintptr_t>(m.p) % bytes_of(m.type) == 0; }
bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na && nb && x < y + nb && y < x + na;
}
bool overlap(const Matrix &a, const Matrix &b) { return overlap(a.p, a.bytes(), b.p, b.bytes()); }

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t) 255; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

template<int N> struct Number { static constexpr int value = N; };

uint32_t values_of(int type) { return type == GLIDE_ROW_F32 || type == GLIDE_ROW_U8 ? 4 : 8; }   // of a piece, at most
uint32_t min_of(uint32_t a, uint32_t b) { return a < b ? a : b; }

// f(the width as a constant)
template<int kMost, typename F> cudaError_t with_width(uint32_t v, F f) {
    if constexpr (kMost >= 8) if (v >= 8) return f(Number<8>{});
    if (v >= 4) return f(Number<4>{});
    if (v >= 2) return f(Number<2>{});
    return f(Number<1>{});
}
// f(a value of the type, the width) for rows of floating types
template<typename F> cudaError_t with_rows(int type, uint32_t v, F f) {
    if (type == GLIDE_ROW_F32) return with_width<4>(v, [&](auto w) { return f(float{}, w); });
    if (type == GLIDE_ROW_F16) return with_width<8>(v, [&](auto w) { return f(__half{}, w); });
    return with_width<8>(v, [&](auto w) { return f(__nv_bfloat16{}, w); });
}
// f(a value of the type, the width, whether rows are whole words): 16-bit values that would go one by one are shifted instead
template<typename F> cudaError_t with_rows_or_shifted(int type, uint32_t v, F f) {
    return with_rows(type, type != GLIDE_ROW_F32 && v == 1 ? 8 : v, [&](auto t, auto w) {
        if constexpr (sizeof t == 2 && decltype(w)::value == 8)
            if (v == 1) return f(t, w, Number<0>{});
        if constexpr (sizeof t == 2 && decltype(w)::value == 1) return cudaErrorInvalidValue;   // the shifted form takes these
        else return f(t, w, Number<1>{});
    });
}

// f(first row, rows) for parts of a call whose pieces a launch can count in 31 bits
template<typename F> cudaError_t in_parts(uint64_t count, uint32_t words, F f) {
    const uint64_t each = 0x7fff0000u / words;
    for (uint64_t r0 = 0; r0 < count; r0 += each) {
        const cudaError_t e = f(r0, (uint32_t) (count - r0 < each ? count - r0 : each));
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Whether a warp a row is taken, rather than a thread a piece: rows of two pieces a lane at least, enough of them for 16 warps an SM, and
// pieces so narrow that the work around each of them tells.
bool long_rows(uint64_t rows, uint32_t words, uint32_t piece_bytes) { return piece_bytes < 16 && words >= 64 && rows >= 148 * 16; }

template<typename T, typename O, int V, bool kWhole>
cudaError_t launch_lookup(const Matrix &table, const uint32_t *ids, float scale, const Matrix &out, cudaStream_t stream) {
    const uint32_t words = pieces<V, O>(kWhole, out.dim);
    return in_parts(out.rows, words, [&](uint64_t r0, uint32_t rows) {
        const uint32_t units = rows * words;
        if (long_rows(rows, words, kWhole ? V * sizeof(T) : 8))   // shifted pieces have more work around them, too
            return launch(lookup_long_kernel<T, O, V, kWhole, kWhole ? in_flight(64, V * (int) sizeof(T), 16) : 4>, ceil_div(rows, 8), 256, 0, stream, false, table.as<const T>(), (uint32_t) table.rows, out.dim, ids + r0, rows, words, scale,
                          out.from(r0).as<O>());
        auto go = [&](auto u) {
            return launch(lookup_kernel<T, O, V, kWhole, decltype(u)::value>, ceil_div(units, 256 * decltype(u)::value), 256, 0, stream, false, table.as<const T>(), (uint32_t) table.rows,
                          out.dim, ids + r0, units, Div(words), scale, out.from(r0).as<O>());
        };
        return units <= 256 * 1024 ? go(Number<1>{}) : go(Number<2>{});
    });
}

uint32_t bits_for(uint64_t values) {   // to write 0 .. values - 1
    uint32_t bits = 1;
    while ((1ull << bits) < values) bits++;
    return bits;
}

// One pass over more than one tile; `clear` gives the next rows to clear to each launch that has room for it.
template<typename To, typename C>
cudaError_t sort_pass(const Keys &keys, uint32_t items, const Digit &digit, uint32_t buckets, uint32_t *counts, uint32_t *totals, uint16_t *ranks,
                      const To &to, bool dependent, cudaStream_t stream, C clear) {
    const uint32_t tiles = (uint32_t) ceil_div(items, kTile);
    Clear c = clear();
    cudaError_t e = launch(bucket_count_kernel, tiles + c.blocks(), kTileThreads, rank_smem(kTileThreads / 32, buckets), stream, dependent, keys, items, digit, buckets, tiles, counts, ranks, c);
    if (e != cudaSuccess) return e;
    c = clear();
    if ((uint64_t) tiles * count_stride(buckets) <= kMaxFusedCounts)
        return launch(bucket_place_kernel<To, false>, tiles + c.blocks(), kTileThreads, count_stride(buckets) * 8, stream, true, keys, items, digit, buckets, tiles, counts, totals, ranks, to, c);
    e = launch(bucket_scan_kernel, ceil_div(buckets, 32) + c.blocks(), 1024, 0, stream, true, counts, tiles, buckets, totals, c);
    if (e != cudaSuccess) return e;
    c = clear();
    return launch(bucket_place_kernel<To, true>, tiles + c.blocks(), kTileThreads, count_stride(buckets) * 8, stream, true, keys, items, digit, buckets, tiles, counts, totals, ranks, to, c);
}

// Scratch of the gradient: two copies of the sorted items, the counts of a pass, the partial sums of its chunks.
struct GradScratch {
    uint2 *items[2];
    uint32_t *counts, *totals;
    uint16_t *ranks;
    float *partial;
    uint32_t bits, passes, pass_bits, chunk;
    uint64_t bytes;
    GradScratch(void *base, uint64_t n, uint64_t count, uint32_t dim) {
        bits = bits_for(n + 1);             // ids 0 .. n - 1, and n for none
        passes = (bits + kMaxPassBits - 1) / kMaxPassBits;
        pass_bits = (bits + passes - 1) / passes;
        // Long chunks leave few partial sums, short ones many groups of lanes to work: as long as some 16 warps an SM remain
        // (counted for words of 16 bytes of bf16), 8 to 128.
        chunk = 8;
        while (chunk < 128 && count * dim / 256 / chunk >= 2 * 148 * 16) chunk *= 2;
        uint64_t at = 0;
        auto take = [&](uint64_t size) {
            const uint64_t here = at;
            at += align256(size);
            return static_cast<char *>(base) + here;
        };
        for (int i = 0; i < 2; i++) items[i] = reinterpret_cast<uint2 *>(take(count * 8));
        ranks = reinterpret_cast<uint16_t *>(take(count * 2));
        counts = reinterpret_cast<uint32_t *>(take(ceil_div(count, kTile) * count_stride(1u << pass_bits) * 4));
        totals = reinterpret_cast<uint32_t *>(take(4ull << pass_bits));
        partial = reinterpret_cast<float *>(take(2 * ceil_div(count, chunk) * dim * 4));
        bytes = at;
    }
};

struct DispatchScratch {
    uint32_t *counts = nullptr, *totals = nullptr;
    uint16_t *ranks = nullptr;
    uint64_t bytes = 0;
    DispatchScratch(void *base, uint64_t pairs, uint32_t partitions) {
        if (pairs <= kFewPairs) return;
        auto take = [&](uint64_t size) {
            const uint64_t here = bytes;
            bytes += align256(size);
            return static_cast<char *>(base) + here;
        };
        ranks = reinterpret_cast<uint16_t *>(take(pairs * 2));
        counts = reinterpret_cast<uint32_t *>(take(ceil_div(pairs, kTile) * count_stride(partitions + 1) * 4));
        totals = reinterpret_cast<uint32_t *>(take((partitions + 1) * 4ull));
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
    ROWS_REQUIRE(table.sized() && out.sized() && (out_stride >= dim || count == 1), GLIDE_ERR_BAD_ARG, "lookup_rows: rows of the result overlap, or it is beyond 2^60 values");
    ROWS_REQUIRE(aligned(table) && aligned(out) && reinterpret_cast<uintptr_t>(d_ids) % 4 == 0, GLIDE_ERR_BAD_ARG, "lookup_rows: a pointer is not aligned to its type");
    ROWS_REQUIRE(!overlap(out, table) && !overlap(d_out, out.bytes(), d_ids, count * 4), GLIDE_ERR_BAD_ARG, "lookup_rows: the result overlaps an input");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    const uint32_t most = values_of(row_type), v = min_of(table.width(most), out.width(most));
    auto s = static_cast<cudaStream_t>(stream);
    if (row_type == GLIDE_ROW_U8) ROWS_CUDA(v == 4 ? launch_lookup<uint8_t, float, 4, true>(table, d_ids, scale, out, s) : launch_lookup<uint8_t, float, 4, false>(table, d_ids, scale, out, s));
    else ROWS_CUDA(with_rows_or_shifted(row_type, v, [&](auto t, auto w, auto wh) {
        return launch_lookup<decltype(t), decltype(t), decltype(w)::value, decltype(wh)::value != 0>(table, d_ids, scale, out, s);
    }));
    return GLIDE_OK;
}

size_t glide_lookup_rows_grad_workspace(uint64_t n, uint32_t dim, uint64_t count) {
    if (n > kNone || dim > kMaxDim || count > 0x7fffffffu) return 0;
    return count <= kFewIds ? 0 : (size_t) GradScratch(nullptr, n, count, dim).bytes;
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
    ROWS_REQUIRE(in.sized() && out.sized() && (table_grad_stride >= dim || n == 1), GLIDE_ERR_BAD_ARG, "lookup_rows_grad: rows of the result overlap, or it is beyond 2^60 values");
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
    const uint32_t most = values_of(row_type), v = min_of(count ? in.width(most) : most, out.width(most));
    const GradScratch w(d_workspace, n, count, dim);
    const uint32_t items = (uint32_t) count, row_bytes = dim * bytes_of(grad_type);
    // Rows are cleared where the memory is idle: a share with each launch of the sort, whether an id names them or not, as long as ids are
    // few beside rows; the rest by the kernel that joins, which by then knows the rows that no id names.
    uint32_t clear_each = (128u << 10) / row_bytes, cleared = 0;   // a CTA clears up to 128 KB
    clear_each = clear_each < 1 ? 1 : clear_each > 256 ? 256 : clear_each;
    GradArgs a{nullptr, items, (uint32_t) n, dim, dim / v, 32, 1, w.chunk, scale, accumulate, w.partial, Div(row_bytes), 0, 0, clear_each};
    // f(a value of the rows' type, one of the result's, the width)
    auto with_types = [&](auto f) {
        return with_rows(row_type, v, [&](auto t, auto wd) { return grad_type == GLIDE_ROW_F32 ? f(t, float{}, wd) : f(t, t, wd); });
    };
    auto lanes_up_to = [&](uint32_t most) {
        a.lanes = most;
        while (a.lanes > 1 && a.lanes / 2 >= a.words) a.lanes /= 2;
    };
    if (count <= kFewIds) {
        const uint64_t grid = count + (accumulate ? 0 : ceil_div(n, clear_each));
        if (grid == 0) return GLIDE_OK;
        lanes_up_to(256);
        ROWS_CUDA(with_types([&](auto t, auto o, auto wd) {
            using T = decltype(t);
            using O = decltype(o);
            return launch(grad_few_kernel<T, O, decltype(wd)::value>, grid, 256, 0, s, false, in.as<const T>(), out.as<O>(), d_ids, a);
        }));
        return GLIDE_OK;
    }
    lanes_up_to(32);
    a.slabs = (uint32_t) ceil_div(a.words, a.lanes);
    const uint64_t chunks = ceil_div(items, a.chunk), join = ceil_div(chunks * a.slabs * a.lanes, 256), units = (chunks - 1) * a.slabs;
    // threads are counted in 32 bits, CTAs in 31; nothing has been launched yet
    ROWS_REQUIRE(join <= 0xffffffu && units <= 0x7fffffffu && join + ceil_div(n, clear_each) <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "lookup_rows_grad: too many values in one call");
    a.join_blocks = (uint32_t) join;
    const uint64_t share = accumulate || count >= n / 2 ? 0 : kClearShare / row_bytes;
    auto clear = [&]() {
        const Clear c{static_cast<uint8_t *>(d_table_grad) + (uint64_t) cleared * table_grad_stride * bytes_of(grad_type), table_grad_stride * bytes_of(grad_type), row_bytes,
                      (uint32_t) (share < n - cleared ? share : n - cleared), clear_each};
        cleared += c.rows;
        return c;
    };
    const uint2 *sorted = nullptr;
    if (count <= kFew) {
        const Clear c = clear();
        ROWS_CUDA(launch(few_sort_kernel, ceil_div(items, 8) + c.blocks(), 256, 0, s, false, d_ids, items, (uint32_t) n, w.items[0], c));
        sorted = w.items[0];
    } else {
        for (uint32_t pass = 0; pass < w.passes; pass++) {
            const uint32_t left = w.bits - pass * w.pass_bits, here = left < w.pass_bits ? left : w.pass_bits;
            ROWS_CUDA(sort_pass(Keys{d_ids, sorted}, items, Digit{(uint32_t) n, pass * w.pass_bits, here}, 1u << here, w.counts, w.totals, w.ranks, ToSorted{w.items[pass & 1]}, pass > 0, s, clear));
            sorted = w.items[pass & 1];
        }
    }
    a.sorted = sorted;
    a.clear_from = cleared;
    const uint64_t zero = accumulate ? 0 : ceil_div(n - cleared, clear_each);
    ROWS_CUDA(with_types([&](auto t, auto o, auto wd) {
        using T = decltype(t);
        using O = decltype(o);
        constexpr int V = decltype(wd)::value;
        const cudaError_t e = launch(grad_join_kernel<T, O, V>, join + zero, 256, 0, s, true, in.as<const T>(), out.as<O>(), a);
        if (e != cudaSuccess) return e;   // more than kFewIds ids are more than one chunk, so that units is not 0
        return launch(grad_fix_kernel<O, V>, ceil_div(units, 8), 256, 0, s, true, out.as<O>(), a, (uint32_t) units);
    }));
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
    ROWS_REQUIRE(in.sized() && out.sized() && (sorted_stride >= dim || pairs <= 1), GLIDE_ERR_BAD_ARG, "dispatch_rows: rows of the result overlap, or it is beyond 2^60 values");
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
    const uint32_t most = values_of(row_type), v = min_of(in.width(most), out.width(most)), words = dim / v;
    // rows are copied as bits: f(a value as wide as theirs, the width)
    auto with_bits = [&](auto f) {
        if (row_type == GLIDE_ROW_F32) return with_width<4>(v, [&](auto wd) { return f(uint32_t{}, wd); });
        return with_width<8>(v, [&](auto wd) { return f(uint16_t{}, wd); });
    };
    if (pairs <= kFewPairs) {
        ROWS_CUDA(with_bits([&](auto t, auto wd) {
            using T = decltype(t);
            return launch(dispatch_small_kernel<T, decltype(wd)::value>, count + 1, 256, (partitions + 1) * 4, s, false, in.as<const T>(), dim, (uint32_t) count, words, d_choice, choices, partitions,
                          out.as<T>(), d_position, d_map, d_segment_start);
        }));
        return GLIDE_OK;
    }
    const DispatchScratch w(d_workspace, pairs, partitions);
    const Digit digit{partitions, 0, bits_for(partitions + 1)};
    const ToPlaces places{d_position, d_map, d_segment_start, Div(choices)};
    ROWS_CUDA(sort_pass(Keys{d_choice, nullptr}, (uint32_t) pairs, digit, partitions + 1, w.counts, w.totals, w.ranks, places, false, s, [] { return Clear{}; }));
    ROWS_CUDA(with_bits([&](auto t, auto wd) {
        using T = decltype(t);
        return in_parts(count, words, [&](uint64_t r0, uint32_t rows) {
            const uint32_t units = rows * words;
            if (long_rows(rows, words, decltype(wd)::value * sizeof t))
                return launch(dispatch_long_kernel<T, decltype(wd)::value, in_flight(64, decltype(wd)::value * (int) sizeof(T), 16)>, ceil_div(rows, 8), 256, 0, s, r0 == 0, in.from(r0).as<const T>(), dim, rows, words, choices, d_position + r0 * choices,
                              out.as<T>());
            auto go = [&](auto u) {
                return launch(dispatch_kernel<T, decltype(wd)::value, decltype(u)::value>, ceil_div(units, 256 * decltype(u)::value), 256, 0, s, r0 == 0, in.from(r0).as<const T>(), dim, units,
                              Div(words), choices, d_position + r0 * choices, out.as<T>());
            };
            return units <= 256 * 1024 ? go(Number<1>{}) : go(Number<2>{});
        });
    }));
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
    ROWS_REQUIRE(in.sized() && out.sized() && (out_stride >= dim || count == 1), GLIDE_ERR_BAD_ARG, "combine_rows: rows of the result overlap, or it is beyond 2^60 values");
    ROWS_REQUIRE(aligned(in) && aligned(out) && (reinterpret_cast<uintptr_t>(d_position) | reinterpret_cast<uintptr_t>(d_weights_or_null)) % 4 == 0, GLIDE_ERR_BAD_ARG, "combine_rows: a pointer is not aligned to its type");
    ROWS_REQUIRE(!overlap(out, in) && !overlap(d_out, out.bytes(), d_position, count * choices * 4) && !overlap(d_out, out.bytes(), d_weights_or_null, d_weights_or_null ? count * choices * 4 : 0), GLIDE_ERR_BAD_ARG, "combine_rows: the result overlaps an input");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    const uint32_t most = values_of(row_type), v = min_of(in.width(most), out.width(most));
    ROWS_CUDA(with_rows_or_shifted(row_type, v, [&](auto t, auto wd, auto wh) {
        using T = decltype(t);
        constexpr int V = decltype(wd)::value;
        constexpr bool kWhole = decltype(wh)::value != 0;
        const uint32_t words = pieces<V, T>(kWhole, dim);
        return in_parts(count, words, [&](uint64_t r0, uint32_t rows) {
            const uint32_t units = rows * words;
            auto go = [&](auto k) {
                constexpr int K = decltype(k)::value;
                // With one choice, or a few of which many may be missing, a thread a piece has too little in flight, whatever the width: 21,701 x 6
                // rows of 3 KB, two thirds of them missing, 61 us, by a warp a row 48; one choice, 32,081 rows of 4.5 KB, 76 and 56; but
                // 39,047 x 4 of 5 KB, all there, 143 and 153. Shifted pieces: a thread a piece 65, a warp a row 70 (20,000 x 4 of 2 KB).
                if constexpr (kWhole)
                    if (long_rows(rows, words, K == 4 || choices == 1 ? 8 : V * sizeof t))
                        return launch(combine_long_kernel<T, V, K, in_flight((K <= 2 ? 64 : 128) / K, V * (int) sizeof(T), 8)>, ceil_div(rows, 8), 256, 0, s, false, in.as<const T>(), (uint32_t) sorted_rows,
                                      dim, d_position + r0 * choices, choices, d_weights_or_null ? d_weights_or_null + r0 * choices : nullptr, rows, words, out.from(r0).as<T>());
                return launch(combine_kernel<T, V, kWhole, K>, ceil_div(units, 256), 256, 0, s, false, in.as<const T>(), (uint32_t) sorted_rows, dim, d_position + r0 * choices, choices,
                              d_weights_or_null ? d_weights_or_null + r0 * choices : nullptr, units, Div(words), out.from(r0).as<T>());
            };
            if (choices == 1) return go(Number<1>{});
            if (choices == 2) return go(Number<2>{});
            if constexpr (kWhole) if (choices >= 8) return go(Number<8>{});
            return go(Number<4>{});
        });
    }));
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
    ROWS_REQUIRE(grad.sized() && in.sized() && out.sized() && (grad_sorted_stride >= dim || sorted_rows <= 1), GLIDE_ERR_BAD_ARG, "combine_rows_grad: rows of the result overlap, or it is beyond 2^60 values");
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
    const uint32_t most = values_of(row_type), v = min_of(grad.width(most), min_of(in.width(most), out.width(most))), words = dim / v;
    ROWS_CUDA(with_rows(row_type, v, [&](auto t, auto wd) {
        using T = decltype(t);
        auto go = [&](auto k, auto g) {
            constexpr int V = decltype(wd)::value, K = decltype(k)::value, G = decltype(g)::value, U = in_flight(64 / K, V * (int) sizeof(T), 8);
            return launch(combine_grad_kernel<T, V, K, U, G>, ceil_div(count, 256 / G), 256, 0, s, false, grad.as<const T>(), (uint32_t) count, dim, words, in.as<const T>(), (uint32_t) sorted_rows,
                          d_position, choices, d_weights_or_null, out.as<T>(), d_grad_weights_or_null);
        };
        if (count <= 148 * 8 && words > 64) return choices <= 4 ? go(Number<4>{}, Number<256>{}) : go(Number<8>{}, Number<256>{});
        auto lanes = [&](auto g) { return choices <= 2 ? go(Number<2>{}, g) : choices < 8 ? go(Number<4>{}, g) : go(Number<8>{}, g); };
        // eight lanes a row of up to 32 pieces: 92,324 x 3 rows of 64 bytes 33 against 15 us, 100,000 x 2 of 512 bytes 50 against 43
        return words <= 32 ? lanes(Number<8>{}) : lanes(Number<32>{});
    }));
    return GLIDE_OK;
}

size_t glide_clear_rows_without_place_workspace(uint64_t rows) { return rows > 0x7fffffffu ? 0 : (size_t) align256(ceil_div(rows, 32) * 4); }

int glide_clear_rows_without_place(glide_ctx *ctx, void *d_rows, int row_type, uint64_t rows, uint32_t dim, uint64_t row_stride, const uint32_t *d_position,
                                   uint64_t pairs, void *d_workspace, size_t workspace_bytes, void *stream) {
    ROWS_REQUIRE(ctx, GLIDE_ERR_BAD_ARG, "clear_rows_without_place: null context");
    ROWS_REQUIRE(is_float_type(row_type), GLIDE_ERR_UNSUPPORTED, "clear_rows_without_place: unsupported row type %d", row_type);
    ROWS_REQUIRE(dim >= 1, GLIDE_ERR_BAD_ARG, "clear_rows_without_place: no values");
    ROWS_REQUIRE(dim <= kMaxDim && rows <= 0x7fffffffu && pairs <= 0x7fffffffu, GLIDE_ERR_UNSUPPORTED, "clear_rows_without_place: more than 2^20 values or 2^31 - 1 pairs or rows");
    if (rows == 0) return GLIDE_OK;
    const Matrix out{d_rows, rows, row_stride, dim, row_type};
    ROWS_REQUIRE(d_rows && (d_position || pairs == 0), GLIDE_ERR_BAD_ARG, "clear_rows_without_place: null pointer");
    ROWS_REQUIRE(out.sized() && (row_stride >= dim || rows == 1), GLIDE_ERR_BAD_ARG, "clear_rows_without_place: rows overlap, or are beyond 2^60 values");
    ROWS_REQUIRE(aligned(out) && reinterpret_cast<uintptr_t>(d_position) % 4 == 0, GLIDE_ERR_BAD_ARG, "clear_rows_without_place: a pointer is not aligned to its type");
    const size_t need = glide_clear_rows_without_place_workspace(rows);
    ROWS_REQUIRE(workspace_bytes >= need && d_workspace, GLIDE_ERR_BAD_ARG, "clear_rows_without_place: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    ROWS_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0, GLIDE_ERR_BAD_ARG, "clear_rows_without_place: the workspace is not aligned to 256 bytes");
    ROWS_REQUIRE(!overlap(d_rows, out.bytes(), d_position, pairs * 4) && !overlap(d_workspace, need, d_rows, out.bytes()) && !overlap(d_workspace, need, d_position, pairs * 4),
                 GLIDE_ERR_BAD_ARG, "clear_rows_without_place: the rows or the workspace overlap another argument");
    const OnDevice guard(ctx->device);
    ROWS_CUDA(guard.status);
    auto s = static_cast<cudaStream_t>(stream);
    uint32_t *marks = static_cast<uint32_t *>(d_workspace);
    ROWS_CUDA(cudaMemsetAsync(marks, 0, ceil_div(rows, 32) * 4, s));
    if (pairs) ROWS_CUDA(launch(mark_places_kernel, ceil_div(pairs, 256), 256, 0, s, false, d_position, (uint32_t) pairs, (uint32_t) rows, marks));
    const uint32_t row_bytes = dim * bytes_of(row_type);
    uint32_t each = (128u << 10) / row_bytes / 32 * 32;
    each = each < 32 ? 32 : each > 256 ? 256 : each;
    auto clear = [&](auto o) {   // zeros have the same bits in both types of 16 bits
        using O = decltype(o);
        return launch(clear_unplaced_kernel<O>, ceil_div(rows, each), 256, 0, s, pairs != 0, out.as<O>(), (uint32_t) rows, dim, Div(row_bytes), each, marks);
    };
    ROWS_CUDA(bytes_of(row_type) == 4 ? clear(float{}) : clear(__half{}));
    return GLIDE_OK;
}

}  // extern "C"
