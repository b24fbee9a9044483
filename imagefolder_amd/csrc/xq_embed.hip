// xq_embed.hip — embedding lookup with a scale, and its gradient by tokens sorted by row (gfx950).
//
// forward:  y[n] = scale * w[idx[n]].
// gradient: dw[v] = scale * sum of g[n] over the tokens n with idx[n] = v — no floating-point atomics: the tokens are sorted by row (stable: ascending n
// inside a row) and every row of dw is one fp32 chain, written once (rows without a token with zeros: no clearing pass).
//
// The sort is two launches, not a radix sort's pass per digit: (1) `embed_bin_kernel` — every block sorts its slice of the tokens by the row's high
// bits (the bucket: up to 1024 buckets of 2^shift rows) in LDS and writes the slice's sorted list and its bucket starts; (2) `embed_sort_kernel` —
// one block per bucket gathers its pieces of every slice's list (they follow each other in token order) and places them by the row's low bits.  The
// position of a bucket in the sorted whole needs no scan over buckets: it is the sum of the slices' starts of that bucket.
// The sums are two more: (3) `embed_sum_kernel` — rows of up to `chunk` tokens whole, and of the longer ones (a frequent word, a padding id) the pieces
// that lie in each `chunk` of sorted positions, so that one row's tokens are read by many blocks; (4) `embed_long_kernel` adds a long row's pieces in order.
#include "xq_common.hpp"
#include "xq_internal.hpp"
#include "xq_vec.hpp"
#include "../../include/xq_ops.h"
#include <algorithm>

namespace {

constexpr int BIN_THREADS = 256, BIN_WAVES = BIN_THREADS / 64, BIN_ROUNDS = 8, BIN_TILE = BIN_THREADS * BIN_ROUNDS;
constexpr int MAX_BUCKETS = 1024, MAX_LOCAL = 1024;      // rows <= 2^20

// ---- forward ------------------------------------------------------------------------------------------------------------------------------

template <typename TW, typename TY, typename TI, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const TI *__restrict__ idx, const TW *__restrict__ w, long N, long V, int D, int lanes, float scale,
                                                        TY *__restrict__ y) {
    const int rows = 256 / lanes, lane = threadIdx.x % lanes;
    for (long n = (long)blockIdx.x * rows + threadIdx.x / lanes; n < N; n += (long)gridDim.x * rows) {
        const long v = (long)idx[n];
        const bool ok = v >= 0 && v < V;
        const TW *src = w + (ok ? v : 0) * (long)D;
        TY *dst = y + n * (long)D;
        for (int c = lane * VEC; c < D; c += lanes * VEC) {
            float a[VEC];
            load_vec<TW, VEC>(src + c, a);
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = ok ? a[j] * scale : __uint_as_float(0x7fc00000u);   // an index outside the table reads nothing of it
            store_vec<TY, VEC>(dst + c, a);
        }
    }
}

// ---- gradient: the sort ---------------------------------------------------------------------------------------------------------------------

// lanes of the wave whose `digit` (bits bits) equals this lane's; dead lanes carry a digit of their own class through `live`
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool live) {
    uint64_t m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1u);
        m &= ((digit >> b) & 1u) ? set : ~set;
    }
    return m;
}

// exclusive scan of count[0 .. n) in place by the whole block; `part` holds one value a wave.  Returns the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t *count, int n, uint32_t *part) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (n + BIN_THREADS - 1) / BIN_THREADS;
    const int lo = min(tid * per, n), hi = min(lo + per, n);
    uint32_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += count[i];
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (int w = 0; w < BIN_WAVES; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    uint32_t at = before + incl - mine;
    for (int i = lo; i < hi; ++i) {
        const uint32_t c = count[i];
        count[i] = at;
        at += c;
    }
    __syncthreads();
    return total;
}

// The stable ranks of one tile of BIN_TILE items: wave w owns items [w * 512, (w + 1) * 512) of the tile in rounds of 64; at[w][digit] counts what the
// wave has seen (own region of LDS: no two waves meet).  rank[r] = items of the same digit before this one in the wave.
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[ROUNDS], const bool (&live)[ROUNDS], int bits, uint32_t *at, uint32_t (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint64_t same = same_digit(digit[r], bits, live[r]);
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1));
        uint32_t seen = 0;
        if (live[r]) seen = at[digit[r]];
        rank[r] = seen + before;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // every lane has read before the last one of the digit writes, and reads again after it
        if (live[r] && (same >> lane) == 1ull) at[digit[r]] = seen + before + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// slices of `tiles` tiles; list (row low bits | token) in bucket order, starts[slice][bucket] relative to the slice, buckets + 1 entries
template <typename TI>
__global__ __launch_bounds__(BIN_THREADS) void embed_bin_kernel(const TI *__restrict__ idx, long N, long V, long skip, int shift, int buckets, int bits,
                                                                int tiles, uint2 *__restrict__ list, uint32_t *__restrict__ starts) {
    __shared__ uint32_t at[BIN_WAVES][MAX_BUCKETS];
    __shared__ uint32_t base[MAX_BUCKETS];
    __shared__ uint32_t part[BIN_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long first = (long)blockIdx.x * tiles * BIN_TILE, end = min(N, first + (long)tiles * BIN_TILE);
    // the slice's bucket counts (a slice of one tile gets them from the ranking below)
    for (int i = tid; i < buckets; i += BIN_THREADS) base[i] = 0;
    __syncthreads();
    for (long n = first + tid; n < end; n += BIN_THREADS) {
        const long v = (long)idx[n];
        if (v >= 0 && v < V && v != skip) atomicAdd(&base[v >> shift], 1u);      // whole numbers: the order of the adds does not matter
    }
    __syncthreads();
    const uint32_t total = block_scan(base, buckets, part);
    uint32_t *st = starts + (long)blockIdx.x * (buckets + 1);
    for (int i = tid; i < buckets; i += BIN_THREADS) st[i] = base[i];
    if (tid == 0) st[buckets] = total;
    for (long t0 = first; t0 < end; t0 += BIN_TILE) {
        for (int i = lane; i < buckets; i += 64) at[wave][i] = 0;
        __syncthreads();
        uint32_t digit[BIN_ROUNDS], low[BIN_ROUNDS], rank[BIN_ROUNDS];
        bool live[BIN_ROUNDS];
#pragma unroll
        for (int r = 0; r < BIN_ROUNDS; ++r) {
            const long n = t0 + wave * (64 * BIN_ROUNDS) + r * 64 + lane;
            long v = -1;
            if (n < end) v = (long)idx[n];
            live[r] = v >= 0 && v < V && v != skip;
            digit[r] = live[r] ? (uint32_t)(v >> shift) : 0u;
            low[r] = (uint32_t)v & ((1u << shift) - 1);
        }
        wave_ranks<BIN_ROUNDS>(digit, live, bits, at[wave], rank);
        __syncthreads();
        for (int i = tid; i < buckets; i += BIN_THREADS) {      // where each wave's items of bucket i begin; base moves on to the next tile
            uint32_t b = base[i];
#pragma unroll
            for (int w = 0; w < BIN_WAVES; ++w) {
                const uint32_t c = at[w][i];
                at[w][i] = b;
                b += c;
            }
            base[i] = b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < BIN_ROUNDS; ++r) {
            const long n = t0 + wave * (64 * BIN_ROUNDS) + r * 64 + lane;
            if (live[r]) list[first + at[wave][digit[r]] + rank[r]] = make_uint2(low[r], (uint32_t)n);
        }
        __syncthreads();
    }
}

// one block per bucket: row starts of the bucket's rows, its tokens in row order, and the rows of every chunk's first and last position
__global__ __launch_bounds__(BIN_THREADS) void embed_sort_kernel(const uint2 *__restrict__ list, const uint32_t *__restrict__ starts, long V, int shift,
                                                                 int buckets, int bits, int slices, long slice_tokens, uint32_t *__restrict__ row_start,
                                                                 uint32_t *__restrict__ order, int chunk_bits, uint32_t *__restrict__ edge) {
    extern __shared__ uint32_t lds[];
    uint32_t *piece = lds;                       // [slices + 1] where a slice's piece begins in the bucket
    __shared__ uint32_t at[BIN_WAVES][MAX_LOCAL];
    __shared__ uint32_t base[MAX_LOCAL];
    __shared__ uint32_t part[BIN_WAVES];
    __shared__ uint32_t before;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bucket = blockIdx.x;
    const int rows = 1 << shift;
    if (tid == 0) before = 0;
    __syncthreads();
    uint32_t ahead = 0;
    for (int s = tid; s < slices; s += BIN_THREADS) {
        const uint32_t *st = starts + (long)s * (buckets + 1) + bucket;
        const uint32_t b = st[0];
        ahead += b;
        piece[s] = st[1] - b;
    }
    if (ahead) atomicAdd(&before, ahead);
    for (int i = tid; i < rows; i += BIN_THREADS) base[i] = 0;
    __syncthreads();
    const uint32_t total = block_scan(piece, slices, part);
    if (tid == 0) piece[slices] = total;
    __syncthreads();
    const uint32_t start = before;
    // the item at position i of the bucket: the slice whose piece holds it
    auto item = [&](uint32_t i) {
        int lo = 0, hi = slices;                 // piece[lo] <= i < piece[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (piece[mid] <= i) lo = mid; else hi = mid;
        }
        return list[(long)lo * slice_tokens + starts[(long)lo * (buckets + 1) + bucket] + (i - piece[lo])];
    };
    for (uint32_t i = tid; i < total; i += BIN_THREADS) atomicAdd(&base[item(i).x], 1u);
    __syncthreads();
    block_scan(base, rows, part);
    const long v0 = (long)bucket << shift;
    for (int i = tid; i < rows; i += BIN_THREADS)
        if (v0 + i < V) row_start[v0 + i] = start + base[i];
    if (bucket == buckets - 1 && tid == 0) row_start[V] = start + total;
    for (uint32_t t0 = 0; t0 < total; t0 += BIN_TILE) {
        for (int i = lane; i < rows; i += 64) at[wave][i] = 0;
        __syncthreads();
        uint32_t digit[BIN_ROUNDS], tok[BIN_ROUNDS], rank[BIN_ROUNDS];
        bool live[BIN_ROUNDS];
#pragma unroll
        for (int r = 0; r < BIN_ROUNDS; ++r) {
            const uint32_t i = t0 + wave * (64 * BIN_ROUNDS) + r * 64 + lane;
            live[r] = i < total;
            uint2 it = make_uint2(0u, 0u);
            if (live[r]) it = item(i);
            digit[r] = it.x;
            tok[r] = it.y;
        }
        wave_ranks<BIN_ROUNDS>(digit, live, bits, at[wave], rank);
        __syncthreads();
        for (int i = tid; i < rows; i += BIN_THREADS) {
            uint32_t b = base[i];
#pragma unroll
            for (int w = 0; w < BIN_WAVES; ++w) {
                const uint32_t c = at[w][i];
                at[w][i] = b;
                b += c;
            }
            base[i] = b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < BIN_ROUNDS; ++r) {
            if (!live[r]) continue;
            const uint32_t pos = start + at[wave][digit[r]] + rank[r], in = pos & ((1u << chunk_bits) - 1);
            order[pos] = tok[r];
            if (in == 0) edge[2 * (pos >> chunk_bits)] = (uint32_t)v0 + digit[r];
            if (in == (1u << chunk_bits) - 1) edge[2 * (pos >> chunk_bits) + 1] = (uint32_t)v0 + digit[r];
        }
        __syncthreads();
    }
}

// ---- gradient: the sums ---------------------------------------------------------------------------------------------------------------------

// sum of g over the sorted positions [lo, hi) at columns c .. c + VEC
template <typename TG, int VEC>
__device__ __forceinline__ void sum_rows(const TG *__restrict__ g, const uint32_t *__restrict__ order, uint32_t lo, uint32_t hi, int D, int c, float (&acc)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    uint32_t i = lo;
    for (; i + 4 <= hi; i += 4) {
        float a[4][VEC];
#pragma unroll
        for (int k = 0; k < 4; ++k) load_vec<TG, VEC>(g + (long)order[i + k] * D + c, a[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += a[k][j];
    }
    for (; i < hi; ++i) {
        float a[VEC];
        load_vec<TG, VEC>(g + (long)order[i] * D + c, a);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += a[j];
    }
}

// blocks [0, row_blocks): rows of at most `chunk` tokens; the others: chunk `b` of the sorted positions, pieces of longer rows -> part[b][head | tail][D]
template <typename TG, typename TW, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const TG *__restrict__ g, const uint32_t *__restrict__ order, const uint32_t *__restrict__ row_start,
                                                        const uint32_t *__restrict__ edge, long V, int D, int lanes, float scale, uint32_t chunk, long row_blocks, TW *__restrict__ dw,
                                                        float *__restrict__ part) {
    const int lane = threadIdx.x % lanes, sub = threadIdx.x / lanes, rows = 256 / lanes;
    if ((long)blockIdx.x < row_blocks) {
        const long v = (long)blockIdx.x * rows + sub;
        if (v >= V) return;
        const uint32_t lo = row_start[v], hi = row_start[v + 1];
        if (hi - lo > chunk) return;
        for (int c = lane * VEC; c < D; c += lanes * VEC) {
            float acc[VEC];
            sum_rows<TG, VEC>(g, order, lo, hi, D, c, acc);
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] *= scale;
            store_vec<TW, VEC>(dw + v * D + c, acc);
        }
        return;
    }
    const uint32_t valid = row_start[V];
    const long b = (long)blockIdx.x - row_blocks;
    const uint64_t p0_ = (uint64_t)b * chunk;
    if (p0_ >= valid) return;
    const bool full = p0_ + chunk <= valid;
    const uint32_t p0 = (uint32_t)p0_, p1 = full ? p0 + chunk : valid;
    const uint32_t vh = edge[2 * b], vt = full ? edge[2 * b + 1] : vh;
    const uint32_t hs = row_start[vh], he = row_start[vh + 1], ts = row_start[vt], te = row_start[vt + 1];
    if (sub >= 2) return;
    // head: a long row that began in an earlier chunk; tail: one that begins here and goes on behind the chunk's end
    uint32_t lo, hi;
    if (sub == 0) {
        if (!(he - hs > chunk && hs < p0)) return;
        lo = p0; hi = min(he, p1);
    } else {
        if (!(full && te - ts > chunk && ts >= p0)) return;
        lo = ts; hi = p1;
    }
    float *dst = part + (2 * b + sub) * (long)D;
    for (int c = lane * VEC; c < D; c += lanes * VEC) {
        float acc[VEC];
        sum_rows<TG, VEC>(g, order, lo, hi, D, c, acc);
        store_vec<float, VEC>(dst + c, acc);
    }
}

// block b: the long row that begins in chunk b (there is at most one: it goes on behind the chunk's end), its pieces in order
template <typename TW>
__global__ __launch_bounds__(256) void embed_long_kernel(const float *__restrict__ part, const uint32_t *__restrict__ row_start,
                                                         const uint32_t *__restrict__ edge, long V, int D, float scale, uint32_t chunk,
                                                         TW *__restrict__ dw) {
    const uint32_t valid = row_start[V];
    const uint64_t p0 = (uint64_t)blockIdx.x * chunk;
    if (p0 + chunk >= valid) return;             // nothing goes on behind the last chunk
    const long lo = edge[2 * (long)blockIdx.x + 1];
    const uint32_t s = row_start[lo], e = row_start[lo + 1];
    if (!(e - s > chunk && s >= p0)) return;
    const long b0 = blockIdx.x, b1 = (long)((e - 1) / chunk);
    for (int c = blockIdx.y * 256 + threadIdx.x; c < D; c += 256 * gridDim.y) {
        float acc = part[(2 * b0 + 1) * (long)D + c];
#pragma unroll 4
        for (long b = b0 + 1; b <= b1; ++b) acc += part[2 * b * (long)D + c];
        dw[lo * D + c] = from_f<TW>(acc * scale);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------

int log2_up(long x) { int b = 0; while ((1L << b) < x) ++b; return b; }
int pow2_lanes(int D, int vec) { int l = 1; while (l < 256 && l * vec < D) l <<= 1; return l; }

struct Plan {
    int shift, buckets, bucket_bits, tiles, slices;
    int chunk_bits;
    long chunks;
    size_t o_list, o_starts, o_rows, o_order, o_edge, o_part, bytes;
};

Plan make_plan(long N, long V, int D) {
    Plan p;
    const int bits = log2_up(V);
    // a table of up to 256 rows: one row a bucket; above, 512 or 1024 buckets of few rows (a codebook of 16384: 1024 of 16)
    p.shift = bits <= 8 ? 0 : std::max(bits - 10, (bits - 7) / 2);
    p.buckets = (int)((V + (1L << p.shift) - 1) >> p.shift);
    p.bucket_bits = log2_up(p.buckets);
    const long tiles = (N + BIN_TILE - 1) / BIN_TILE;
    p.tiles = (int)((tiles + 511) / 512);
    p.slices = (int)((tiles + p.tiles - 1) / p.tiles);
    // pieces long enough that a row's own sum (one fp32 each) is little work, short enough that the rows' longest chain stays near the mean's cost
    p.chunk_bits = std::max(7, log2_up((N + 2047) / 2048));
    p.chunks = (N + (1L << p.chunk_bits) - 1) >> p.chunk_bits;
    size_t off = 0;
    auto take = [&](size_t b) { size_t o = off; off = xq::align_up(off + b, 256); return o; };
    p.o_list = take((size_t)N * 8);
    p.o_starts = take((size_t)p.slices * (p.buckets + 1) * 4);
    p.o_rows = take((size_t)(V + 1) * 4);
    p.o_order = take((size_t)N * 4);
    p.o_edge = take((size_t)p.chunks * 2 * 4);
    p.o_part = take((size_t)p.chunks * 2 * D * 4);
    p.bytes = off;
    return p;
}

int check(const char *fn, int64_t N, int64_t V, int D) {
    if (N < 0 || V < 1 || D < 1) return xq_set_error(XQ_EINVAL, "%s: bad sizes (V=%ld, D=%ld)", fn, (long)V, (long)D);
    if (N > 0x7fffffffL) return xq_set_error(XQ_EINVAL, "%s: more than 2^31 - 1 tokens (%ld)", fn, (long)N);
    if (V > (1L << 20)) return xq_set_error(XQ_EINVAL, "%s: more than 2^20 rows (%ld)", fn, (long)V);
    return XQ_OK;
}

template <typename TW, typename TY, typename TI>
void launch_fwd(const void *idx, const void *w, long N, long V, int D, float scale, void *y, hipStream_t s) {
    const bool a16 = (((uintptr_t)w | (uintptr_t)y) & 15) == 0;
#define XQ_EMB(VEC)                                                                                                                          \
    {                                                                                                                                        \
        const int lanes = pow2_lanes(D, VEC);                                                                                                \
        const long blocks = std::min<long>((N + 256 / lanes - 1) / (256 / lanes), (long)num_cus() * 32);                                     \
        hipLaunchKernelGGL((embed_fwd_kernel<TW, TY, TI, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, (const TI *)idx, (const TW *)w, N, V, D, \
                           lanes, scale, (TY *)y);                                                                                           \
    }
    if (a16 && D % 8 == 0) XQ_EMB(8)
    else if (a16 && D % 4 == 0 && sizeof(TW) == 4 && sizeof(TY) == 4) XQ_EMB(4)
    else XQ_EMB(1)
#undef XQ_EMB
}

template <typename TG, typename TW>
void launch_sums(const void *g, long V, int D, float scale, const Plan &p, const uint32_t *order, const uint32_t *rows, const uint32_t *edge, float *part, void *dw,
                 hipStream_t s) {
    const bool a16 = (((uintptr_t)g | (uintptr_t)dw) & 15) == 0;
#define XQ_SUM(VEC)                                                                                                                          \
    {                                                                                                                                        \
        const int lanes = std::min(128, pow2_lanes(D, VEC));                                                                                 \
        const long rb = (V + 256 / lanes - 1) / (256 / lanes);                                                                               \
        hipLaunchKernelGGL((embed_sum_kernel<TG, TW, VEC>), dim3((unsigned)(rb + p.chunks)), dim3(256), 0, s, (const TG *)g, order, rows, edge, V, D, lanes, \
                           scale, 1u << p.chunk_bits, rb, (TW *)dw, part);                                                                              \
    }
    if (a16 && D % 8 == 0 && sizeof(TG) == 2) XQ_SUM(8)
    else if (a16 && D % 4 == 0 && sizeof(TG) == 4) XQ_SUM(4)
    else XQ_SUM(1)
#undef XQ_SUM
    hipLaunchKernelGGL((embed_long_kernel<TW>), dim3((unsigned)p.chunks, (unsigned)std::min(8, (D + 255) / 256)), dim3(256), 0, s, part, rows, edge, V, D,
                       scale, 1u << p.chunk_bits, (TW *)dw);
}

template <typename TW>
__global__ __launch_bounds__(256) void embed_zero_kernel(TW *__restrict__ dw, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) dw[i] = from_f<TW>(0.0f);
}

}  // namespace

extern "C" int xq_embedding_forward(const void *idx, int idx_i64, const void *w, int w_bf16, int64_t N, int64_t V, int D, float scale, void *y, int y_bf16,
                                    xq_stream_t stream) {
    const char *fn = "xq_embedding_forward";
    if (int rc = check(fn, N, V, D)) return rc;
    if (N == 0) return XQ_OK;
    if (!idx || !w || !y) return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    hipStream_t s = (hipStream_t)stream;
#define XQ_GO(TW, TY)                                                                      \
    {                                                                                      \
        if (idx_i64) launch_fwd<TW, TY, int64_t>(idx, w, N, V, D, scale, y, s);            \
        else launch_fwd<TW, TY, int32_t>(idx, w, N, V, D, scale, y, s);                    \
    }
    if (w_bf16 && y_bf16) XQ_GO(bf16, bf16)
    else if (w_bf16) XQ_GO(bf16, float)
    else if (y_bf16) XQ_GO(float, bf16)
    else XQ_GO(float, float)
#undef XQ_GO
    return xq_check_launch(fn);
}

extern "C" size_t xq_embedding_backward_workspace_bytes(int64_t N, int64_t V, int D) {
    if (N < 1 || V < 1 || D < 1 || N > 0x7fffffffL || V > (1L << 20)) return 0;
    return make_plan((long)N, (long)V, D).bytes;
}

extern "C" int xq_embedding_backward(const void *idx, int idx_i64, const void *g, int g_bf16, int64_t N, int64_t V, int D, float scale, int64_t skip, void *dw,
                                     int dw_bf16, void *workspace, size_t workspace_bytes, xq_stream_t stream) {
    const char *fn = "xq_embedding_backward";
    if (int rc = check(fn, N, V, D)) return rc;
    if (!dw) return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    hipStream_t s = (hipStream_t)stream;
    if (N == 0) {
        const long n = (long)V * D;
        const unsigned blocks = (unsigned)std::min<long>((n + 255) / 256, (long)num_cus() * 16);
        if (dw_bf16) hipLaunchKernelGGL((embed_zero_kernel<bf16>), dim3(blocks), dim3(256), 0, s, (bf16 *)dw, n);
        else hipLaunchKernelGGL((embed_zero_kernel<float>), dim3(blocks), dim3(256), 0, s, (float *)dw, n);
        return xq_check_launch(fn);
    }
    if (!idx || !g || !workspace) return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    const Plan p = make_plan((long)N, (long)V, D);
    if (workspace_bytes < p.bytes)
        return xq_set_error(XQ_ENOSPACE, "%s: workspace too small (need %ld bytes, got %ld)", fn, (long)p.bytes, (long)workspace_bytes);
    char *ws = (char *)workspace;
    uint2 *list = (uint2 *)(ws + p.o_list);
    uint32_t *starts = (uint32_t *)(ws + p.o_starts), *rows = (uint32_t *)(ws + p.o_rows), *order = (uint32_t *)(ws + p.o_order),
             *edge = (uint32_t *)(ws + p.o_edge);
    float *part = (float *)(ws + p.o_part);
    if (idx_i64)
        hipLaunchKernelGGL((embed_bin_kernel<int64_t>), dim3(p.slices), dim3(BIN_THREADS), 0, s, (const int64_t *)idx, (long)N, (long)V, (long)skip, p.shift,
                           p.buckets, p.bucket_bits, p.tiles, list, starts);
    else
        hipLaunchKernelGGL((embed_bin_kernel<int32_t>), dim3(p.slices), dim3(BIN_THREADS), 0, s, (const int32_t *)idx, (long)N, (long)V, (long)skip, p.shift,
                           p.buckets, p.bucket_bits, p.tiles, list, starts);
    hipLaunchKernelGGL(embed_sort_kernel, dim3(p.buckets), dim3(BIN_THREADS), (size_t)(p.slices + 1) * 4, s, list, starts, (long)V, p.shift, p.buckets, p.shift,
                       p.slices, (long)p.tiles * BIN_TILE, rows, order, p.chunk_bits, edge);
    if (g_bf16 && dw_bf16) launch_sums<bf16, bf16>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else if (g_bf16) launch_sums<bf16, float>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else if (dw_bf16) launch_sums<float, bf16>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else launch_sums<float, float>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    return xq_check_launch(fn);
}
