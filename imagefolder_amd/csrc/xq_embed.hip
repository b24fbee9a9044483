// xq_embed.hip — embedding lookup with a scale, and its gradient by tokens sorted by row (gfx950).
//
// forward:  y[n] = scale * w[idx[n]].
// gradient: dw[v] = scale * sum of g[n] over the tokens n with idx[n] = v — no floating-point atomics: the tokens are sorted by row (stable: ascending n
// inside a row) and every row of dw is one fp32 chain, written once (rows without a token with zeros: no clearing pass).
//
// The sort is two launches, not a radix sort's pass per digit: (1) `embed_bin_kernel` — every block sorts a slice of 1024 tokens by row in LDS and writes the
// sorted list and where each bucket (256 or up to 1024 buckets of 2^shift rows) begins in it; (2) `embed_sort_kernel` — one block per bucket gathers its pieces of
// every slice's list (they follow each other in token order).  The position of a bucket in the sorted whole needs no scan over buckets: it is the sum of the slices'
// starts of that bucket.  A slice is sorted by row whole, and not by bucket alone, for 2 us more of the first launch (9 us instead of 7): it leaves the second
// one no ranking, so that a bucket with a frequent row (14000 of 100000 tokens) takes it 20 us instead of 40, a table read at one row only 96 instead of 250 (100000
// tokens), and 6 to 7 as before where no row is frequent.
// The sums are two more: (3) `embed_sum_kernel` — rows of up to `chunk` tokens whole, and of the longer ones (a frequent word, a padding id) the pieces
// that lie in each `chunk` of sorted positions, so that one row's tokens are read by many blocks; (4) `embed_long_kernel` adds a long row's pieces in order.
#include "xq_common.hpp"
#include "xq_internal.hpp"
#include "xq_vec.hpp"
#include "../../include/xq_ops.h"
#include <algorithm>

namespace {

constexpr int TILE = 1024, BIN_THREADS = 512;            // tokens and threads of a block of the first launch (2048 and 1024: 11 us instead of 9)

// ---- forward ------------------------------------------------------------------------------------------------------------------------------

// a / per_row from the host's floor(2^64 / per_row) + 1 (exact for whole numbers below 2^32; 0 stands for a divisor of one)
__device__ __forceinline__ uint32_t quotient(uint32_t a, uint64_t reciprocal) { return reciprocal ? (uint32_t)__umul64hi((uint64_t)a, reciprocal) : a; }

// One thread per VEC columns; `per_row` threads a row, a quotient by the host's reciprocal (a block of threads per row would idle a quarter of them at
// a width of 768).  split = 8: XCD x (blocks go round-robin over the eight) takes the x-th eighth of the columns of every token, so that a table of up to
// 32 MB, which no 4 MB L2 holds, is held by the eight together; the rows that many tokens share then come out of L2 (32768 tokens of an fp32 table of 8192 x 768
// -> bf16: 17 us, without it 23).  Bound by the rows of y written: 99991 x 512 bf16 30 us, 5.1 TB/s with what it reads.
template <typename TW, typename TY, typename TI, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const TI *__restrict__ idx, const TW *__restrict__ w, long V, int D, int split, uint32_t per_row, uint32_t total,
                                                        uint64_t reciprocal, float scale, TY *__restrict__ y) {
    constexpr int U = 4;
    const uint32_t part = split == 1 ? 0 : blockIdx.x & 7, block = split == 1 ? blockIdx.x : blockIdx.x >> 3;
    const uint32_t step = gridDim.x / split * 256u;
    uint32_t at[U];
    long v[U];
    float a[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        at[u] = block * 256u + threadIdx.x + u * step;
        v[u] = -1;
        if (at[u] < total) v[u] = (long)idx[quotient(at[u], reciprocal)];
    }
    uint32_t n[U], c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        n[u] = quotient(at[u], reciprocal);
        c[u] = at[u] < total ? (at[u] - n[u] * per_row + part * per_row) * VEC : 0;
        const long row = v[u] >= 0 && v[u] < V ? v[u] : 0;
        load_vec<TW, VEC>(w + row * D + c[u], a[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool ok = v[u] >= 0 && v[u] < V;
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[u][j] = ok ? a[u][j] * scale : __uint_as_float(0x7fc00000u);   // an index outside the table reads nothing of it
        if (at[u] < total) store_vec<TY, VEC>(y + (long)n[u] * D + c[u], a[u]);
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
template <int THREADS>
__device__ __forceinline__ uint32_t block_scan(uint32_t *count, int n, uint32_t *part) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (n + THREADS - 1) / THREADS;
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
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
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

// A stable counting sort of one tile by a whole block.  Every wave holds ROUNDS x 64 items that follow each other in token order, round r's digit in
// digit[r] (NONE: no item); at[digit] counts what the wave has met (no two waves share a counter, and the additions of one wave are in order).
constexpr uint32_t NONE = 0xffffffffu;

template <int ROUNDS>
__device__ __forceinline__ void tile_ranks(const uint32_t (&digit)[ROUNDS], int bits, int digits, uint32_t *at, uint32_t (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < digits; i += 64) at[i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool live = digit[r] != NONE;
        const uint64_t same = same_digit(digit[r], bits, live);
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1));
        uint32_t met = 0;
        if (live) met = at[digit[r]];
        rank[r] = met + before;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // every lane has read before the last one of a digit writes, and reads again after it
        if (live && (same >> lane) == 1ull) at[digit[r]] = met + before + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
}

// the tile's count of every digit -> count
template <int WAVES>
__device__ __forceinline__ void tile_counts(const uint32_t *seen, int pitch, int digits, uint32_t *count) {
    for (int i = threadIdx.x; i < digits; i += WAVES * 64) {
        uint32_t c = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) c += seen[w * pitch + i];
        count[i] = c;
    }
    __syncthreads();
}

// base: where each digit's first item goes -> seen[wave][digit]: where the wave's first one goes
template <int WAVES>
__device__ __forceinline__ void tile_places(uint32_t *seen, int pitch, int digits, const uint32_t *base) {
    for (int i = threadIdx.x; i < digits; i += WAVES * 64) {
        uint32_t b = base[i];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t c = seen[w * pitch + i];
            seen[w * pitch + i] = b;
            b += c;
        }
    }
    __syncthreads();
}

// A slice is one tile.  Its tokens are sorted by row in LDS — by the row's low bits, then, stable, by its bucket — and written with what the second launch needs to
// place them without ranking them again: low bits | place in the slice's run of the row << 10 | last of the run << 21, token.  starts[slice][bucket], buckets + 1.
template <typename TI>
__global__ __launch_bounds__(BIN_THREADS) void embed_bin_kernel(const TI *__restrict__ idx, long N, long V, long skip, int shift, int buckets, int bits,
                                                                int pitch, uint2 *__restrict__ list, uint32_t *__restrict__ starts) {
    constexpr int WAVES = BIN_THREADS / 64, ROUNDS = TILE / BIN_THREADS;
    extern __shared__ uint32_t lds[];             // the waves' counters, and the block's: pitch each
    uint32_t *seen = lds, *base = seen + WAVES * pitch;
    __shared__ uint32_t part[WAVES];
    __shared__ uint32_t sorted[TILE + 1];         // row << 11 | token's place in the tile
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long first = (long)blockIdx.x * TILE;
    const uint32_t at0 = wave * (64 * ROUNDS) + lane;        // this thread's places: at0 + 64 r
    uint32_t x[ROUNDS], digit[ROUNDS], rank[ROUNDS], total = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const long n = first + at0 + 64 * r;
        long v = -1;
        if (n < N) v = (long)idx[n];
        x[r] = v >= 0 && v < V && v != skip ? (uint32_t)v << 11 | (at0 + 64 * r) : NONE;
    }
    auto pass = [&](int digits, int nbits, bool publish) {
        tile_ranks<ROUNDS>(digit, nbits, digits, seen + wave * pitch, rank);
        tile_counts<WAVES>(seen, pitch, digits, base);
        total = block_scan<BIN_THREADS>(base, digits, part);
        if (publish) {
            uint32_t *st = starts + (long)blockIdx.x * (buckets + 1);
            for (int i = tid; i < digits; i += BIN_THREADS) st[i] = base[i];
            if (tid == 0) st[buckets] = total;
        }
        tile_places<WAVES>(seen, pitch, digits, base);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (digit[r] != NONE) sorted[seen[wave * pitch + digit[r]] + rank[r]] = x[r];
        __syncthreads();
    };
    if (shift > 0) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) digit[r] = x[r] == NONE ? NONE : x[r] >> 11 & ((1u << shift) - 1);
        pass(1 << shift, shift, false);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) x[r] = at0 + 64 * r < total ? sorted[at0 + 64 * r] : NONE;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) digit[r] = x[r] == NONE ? NONE : x[r] >> (11 + shift);
    pass(buckets, bits, true);
    // where the run of the same row begins: the first place not below row << 11
    uint32_t lo[ROUNDS], key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        x[r] = at0 + 64 * r < total ? sorted[at0 + 64 * r] : NONE;
        key[r] = x[r] & ~2047u;
        lo[r] = 0;
    }
    for (int h = TILE / 2; h > 0; h >>= 1) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (lo[r] + h <= total && sorted[lo[r] + h - 1] < key[r]) lo[r] += h;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t at = at0 + 64 * r;
        if (at >= total) continue;
        const bool last = at + 1 == total || (sorted[at + 1] & ~2047u) != key[r];
        const uint32_t low = x[r] >> 11 & ((1u << shift) - 1);
        list[first + at] = make_uint2(low | (at - lo[r]) << 10 | (last ? 1u << 21 : 0u), (uint32_t)first + (x[r] & 2047u));
    }
}

// One block per bucket: row starts of the bucket's rows, its tokens in row order, and the rows of every chunk's first and last position.  Every wave takes its
// share of the slices, 64 at a time (their pieces end to end, 64 tokens a round, U rounds' loads abreast): it counts its rows from the runs' last tokens; then, the waves' counts
// known, a token's position is its row's next one plus its place in the run.  Slices that meet in one round take turns, so that a row's runs stay in order.
template <int SORT_THREADS>
__global__ __launch_bounds__(SORT_THREADS) void embed_sort_kernel(const uint2 *__restrict__ list, const uint32_t *__restrict__ starts, long V, int shift,
                                                                  int buckets, int slices, uint32_t *__restrict__ row_start,
                                                                  uint32_t *__restrict__ order, int chunk_bits, uint32_t *__restrict__ edge) {
    constexpr int WAVES = SORT_THREADS / 64, U = 4;
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t part[WAVES];
    __shared__ uint32_t ahead[WAVES];
    __shared__ uint32_t pieces[WAVES][64], froms[WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bucket = blockIdx.x;
    const int rows = 1 << shift;
    uint32_t *seen = lds, *base = seen + (WAVES << shift), *at = seen + (wave << shift);
    uint32_t *piece = pieces[wave], *from = froms[wave];          // a wave's own: where a slice's piece begins in the 64 slices' tokens, and in the slice's list
    const int s0 = (int)((long)slices * wave / WAVES), s1 = (int)((long)slices * (wave + 1) / WAVES);
    for (int i = lane; i < rows; i += 64) at[i] = 0;
    // the pieces of slices s .. s + 63 (below s1) -> their tokens' number; `mine`: this lane's slice's tokens ahead of the bucket
    auto take = [&](int s, uint32_t &mine) {
        uint32_t b = 0, n = 0;
        if (s + lane < s1) {
            const uint32_t *st = starts + (long)(s + lane) * (buckets + 1) + bucket;
            b = st[0];
            n = st[1] - b;
        }
        mine = b;
        uint32_t incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(incl, o);
            if (lane >= o) incl += up;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        piece[lane] = incl - n;
        from[lane] = b;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return (uint32_t)__shfl(incl, 63);
    };
    // the tokens at places i + 64 r (+ lane) of those pieces, and the slice (0 .. 63) of each; NONE behind the end
    auto items = [&](int s, uint32_t i, uint32_t total, uint2 (&it)[U], int (&lo)[U]) {
#pragma unroll
        for (int r = 0; r < U; ++r) lo[r] = 0;
#pragma unroll
        for (int h = 32; h > 0; h >>= 1) {
#pragma unroll
            for (int r = 0; r < U; ++r)
                if (piece[lo[r] + h] <= i + 64 * r + lane) lo[r] += h;          // (lo + h <= 63; the last slice that begins not behind the place: the one that holds it)
        }
#pragma unroll
        for (int r = 0; r < U; ++r) {
            const uint32_t p = i + 64 * r + lane;
            it[r] = make_uint2(NONE, 0u);
            if (p < total) it[r] = list[(long)(s + lo[r]) * TILE + from[lo[r]] + (p - piece[lo[r]])];
        }
    };
    uint32_t tokens = 0, before = 0;
    uint2 it[U];
    int lo[U];
    for (int s = s0; s < s1; s += 64) {
        uint32_t mine;
        const uint32_t total = take(s, mine);
        before += mine;
        tokens += total;
        for (uint32_t i = 0; i < total; i += 64 * U) {
            items(s, i, total, it, lo);
#pragma unroll
            for (int r = 0; r < U; ++r)
                if (it[r].x != NONE && it[r].x >> 21) atomicAdd(&at[it[r].x & 1023u], (it[r].x >> 10 & 2047u) + 1);      // a run's tokens (whole numbers: any order)
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
    if (lane == 0) ahead[wave] = before;
    __syncthreads();
    tile_counts<WAVES>(seen, rows, rows, base);
    const uint32_t total_rows = block_scan<SORT_THREADS>(base, rows, part);
    uint32_t start = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) start += ahead[w];
    const long v0 = (long)bucket << shift;
    for (int i = tid; i < rows; i += SORT_THREADS)
        if (v0 + i < V) row_start[v0 + i] = start + base[i];
    if (bucket == buckets - 1 && tid == 0) row_start[V] = start + total_rows;
    tile_places<WAVES>(seen, rows, rows, base);
    const bool here = s1 - s0 <= 64 && tokens <= 64 * U;          // all of the wave's tokens are in registers
    for (int s = s0; s < s1; s += 64) {
        uint32_t mine, total = tokens;
        if (!here) total = take(s, mine);
        for (uint32_t i = 0; i < total; i += 64 * U) {
            if (!here) items(s, i, total, it, lo);
#pragma unroll
            for (int r = 0; r < U; ++r) {
                const uint64_t live = __ballot(it[r].x != NONE);
                if (!live) break;
                const uint32_t low = it[r].x & 1023u, place = it[r].x >> 10 & 2047u;
                const int s_first = __builtin_amdgcn_readlane(lo[r], 0), s_last = __builtin_amdgcn_readlane(lo[r], 63 - __builtin_clzll(live));
                for (int turn = s_first; turn <= s_last; ++turn) {
                    if (it[r].x == NONE || lo[r] != turn) continue;
                    const uint32_t next = at[low];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");           // every token of the run has read before its last one moves the row on
                    if (it[r].x >> 21) at[low] = next + place + 1;
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    const uint32_t pos = start + next + place, in = pos & ((1u << chunk_bits) - 1);
                    order[pos] = it[r].y;
                    if (in == 0) edge[2 * (pos >> chunk_bits)] = (uint32_t)v0 + low;
                    if (in == (1u << chunk_bits) - 1) edge[2 * (pos >> chunk_bits) + 1] = (uint32_t)v0 + low;
                }
            }
        }
    }
}

// ---- gradient: the sums ---------------------------------------------------------------------------------------------------------------------

// Sum of g over the sorted positions [lo, hi) at columns c .. c + VEC.  Eight rows of g in flight, the next eight tokens' numbers fetched behind them: what a
// row takes are its trips to memory.  The last ones in pieces of four, two and one, so that a short row (four tokens, at a codebook's sizes) loads no more than it has.
template <typename TG, int VEC>
__device__ __forceinline__ void sum_rows(const TG *__restrict__ g, const uint32_t *__restrict__ order, uint32_t lo, uint32_t hi, int D, int c, float (&acc)[VEC]) {
    constexpr int U = 8;
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    if (lo >= hi) return;
    const uint32_t last = hi - 1;
    uint32_t n[U];
#pragma unroll
    for (int k = 0; k < U; ++k) n[k] = order[min(lo + k, last)];
    uint32_t i = lo;
    for (; i + U <= hi; i += U) {
        float a[U][VEC];
#pragma unroll
        for (int k = 0; k < U; ++k) load_vec<TG, VEC>(g + (long)n[k] * D + c, a[k]);
#pragma unroll
        for (int k = 0; k < U; ++k) n[k] = order[min(i + U + k, last)];
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += a[k][j];
    }
    const uint32_t left = hi - i;
#define XQ_PIECE(COUNT, FROM)                                                                                     \
    {                                                                                                             \
        float a[COUNT][VEC];                                                                                      \
        _Pragma("unroll") for (int k = 0; k < COUNT; ++k) load_vec<TG, VEC>(g + (long)(FROM)[k] * D + c, a[k]);   \
        _Pragma("unroll") for (int k = 0; k < COUNT; ++k)                                                         \
            _Pragma("unroll") for (int j = 0; j < VEC; ++j) acc[j] += a[k][j];                                    \
    }
    if (left & 4) {
        XQ_PIECE(4, n)
#pragma unroll
        for (int k = 0; k < 3; ++k) n[k] = n[k + 4];
    }
    if (left & 2) {
        XQ_PIECE(2, n)
        n[0] = n[2];
    }
    if (left & 1) XQ_PIECE(1, n)
#undef XQ_PIECE
}

// Groups of `lanes` threads.  Blocks [0, piece_blocks): pieces of long rows (the longest work: begun first), piece 2 b (+ 1) being the head (tail) of chunk b of
// the sorted positions -> part[piece][D]; the others: one row of at most `chunk` tokens each (two or four
// of them in turn: 40 us instead of 42 at 50021 rows of two tokens, 12 instead of 8 at 16384 of five).  Bound by the gathered rows: 32768 x 768 bf16 15 us at HBM's rate,
// 99991 x 512 bf16 into 50021 rows 43 us, 3.6 TB/s: the row's start, its tokens and their rows are three trips for two tokens.
template <typename TG, typename TW, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const TG *__restrict__ g, const uint32_t *__restrict__ order, const uint32_t *__restrict__ row_start,
                                                        const uint32_t *__restrict__ edge, long V, int D, int lanes, float scale, uint32_t chunk, long chunks,
                                                        long piece_blocks, TW *__restrict__ dw, float *__restrict__ part) {
    const int lane = threadIdx.x % lanes, sub = threadIdx.x / lanes, groups = 256 / lanes;
    if ((long)blockIdx.x < piece_blocks) {
        const long id = (long)blockIdx.x * groups + sub, b = id >> 1;
        if (b >= chunks) return;
        const uint32_t valid = row_start[V];
        const uint64_t p0_ = (uint64_t)b * chunk;
        if (p0_ >= valid) return;
        const bool full = p0_ + chunk <= valid, tail = id & 1;
        const uint32_t p0 = (uint32_t)p0_, p1 = full ? p0 + chunk : valid;
        if (tail && !full) return;                 // a tail goes on behind its chunk's end
        const uint32_t v = edge[2 * b + tail];
        const uint32_t s = row_start[v], e = row_start[v + 1];
        // a long row that began in an earlier chunk, or one that begins here and goes on behind the chunk's end
        if (!(e - s > chunk && (tail ? s >= p0 : s < p0))) return;
        const uint32_t lo = tail ? s : p0, hi = tail ? p1 : min(e, p1);
        float *dst = part + id * (long)D;
        for (int c = lane * VEC; c < D; c += lanes * VEC) {
            float acc[VEC];
            sum_rows<TG, VEC>(g, order, lo, hi, D, c, acc);
            store_vec<float, VEC>(dst + c, acc);
        }
        return;
    }
    const long v = ((long)blockIdx.x - piece_blocks) * groups + sub;
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
}

// Chunks 8 b .. 8 b + 7, one a wave: the long row that begins in it (there is at most one: it goes on behind the chunk's end), its pieces added in order.  A row of
// more than 16 pieces is shared out over the block's waves (runs of pieces in order, a chain each; the waves' sums meet in order); of those, eight chunks hold
// the beginning of one at most.
template <typename TW>
__global__ __launch_bounds__(512) void embed_long_kernel(const float *__restrict__ part, const uint32_t *__restrict__ row_start,
                                                         const uint32_t *__restrict__ edge, long V, int D, float scale, uint32_t chunk, long chunks,
                                                         TW *__restrict__ dw) {
    __shared__ float sums[8][64];
    __shared__ int heavy;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) heavy = -1;
    __syncthreads();
    // piece 0: the tail of chunk b; piece k: the head of chunk b + k
    auto add = [&](long b, long k0, long k1, int c) {
        float acc = 0.0f;
#pragma unroll 8
        for (long k = k0; k < k1; ++k) acc += part[(2 * (b + k) + (k == 0)) * (long)D + c];
        return acc;
    };
    auto pieces_of = [&](long b, long &v) -> long {
        const uint64_t p0 = (uint64_t)b * chunk;
        if (b >= chunks || p0 + chunk >= row_start[V]) return 0;         // nothing goes on behind the last chunk
        v = edge[2 * b + 1];
        const uint32_t s = row_start[v], e = row_start[v + 1];
        return e - s > chunk && s >= p0 ? (long)((e - 1) / chunk) - b + 1 : 0;
    };
    const long mine = (long)blockIdx.x * 8 + wave;
    long v = 0;
    const long pieces = pieces_of(mine, v);
    if (pieces > 16) {
        if (lane == 0) heavy = wave;
    } else if (pieces > 0) {
        for (int c = blockIdx.y * 64 + lane; c < D; c += 64 * gridDim.y) dw[v * D + c] = from_f<TW>(add(mine, 0, pieces, c) * scale);
    }
    __syncthreads();
    if (heavy < 0) return;
    const long b = (long)blockIdx.x * 8 + heavy, all = pieces_of(b, v), per = (all + 7) / 8, k0 = wave * per, k1 = min(all, k0 + per);
    for (int c0 = blockIdx.y * 64; c0 < D; c0 += 64 * gridDim.y) {
        const int c = c0 + lane;
        sums[wave][lane] = c < D ? add(b, k0, k1, c) : 0.0f;
        __syncthreads();
        if (wave == 0 && c < D) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) t += sums[w][lane];
            dw[v * D + c] = from_f<TW>(t * scale);
        }
        __syncthreads();
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------

int log2_up(long x) { int b = 0; while ((1L << b) < x) ++b; return b; }
int pow2_lanes(int D, int vec) { int l = 1; while (l < 256 && l * vec < D) l <<= 1; return l; }

struct Plan {
    int shift, buckets, bucket_bits, slices;
    int chunk_bits;
    long chunks;
    size_t o_list, o_starts, o_rows, o_order, o_edge, o_part, bytes;
};

Plan make_plan(long N, long V, int D) {
    Plan p;
    const int bits = log2_up(V);
    // a table of up to 256 rows: one row a bucket.  Above, 256 buckets (one block of sixteen waves a CU; with 1024 buckets the second launch took 14 us
    // instead of 7) while a bucket's counters fit a block's LDS, then 1024 of them.
    p.shift = bits <= 8 ? 0 : bits <= 17 ? bits - 8 : bits - 10;
    p.buckets = (int)((V + (1L << p.shift) - 1) >> p.shift);
    p.bucket_bits = log2_up(p.buckets);
    p.slices = (int)((N + TILE - 1) / TILE);
    // 64 tokens: eight trips to memory for a row or a piece of one, and one fp32 row of partial sums written for 64 read
    p.chunk_bits = std::max(6, log2_up((N + 4095) / 4096));
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
void launch_fwd(const void *idx_, const void *w, long N, long V, int D, float scale, void *y_, hipStream_t s) {
    const bool a16 = (((uintptr_t)w | (uintptr_t)y_) & 15) == 0;
    // 16 bytes of the wider side a thread: two 16-byte loads of one thread (eight fp32) lie 32 bytes apart over the wave and cost twice the lines
    const int vec = a16 && D % 8 == 0 && sizeof(TW) == 2 && sizeof(TY) == 2 ? 8 : a16 && D % 4 == 0 ? 4 : 1;
    // by columns where a table that one L2 does not hold is read more than once over and an eighth of a row is a 64-byte piece at least
    const size_t table = (size_t)V * D * sizeof(TW);
    const int split = N > 2 * V && table > (4u << 20) && table <= (32u << 20) && D % (8 * vec) == 0 && D * sizeof(TY) >= 512 ? 8 : 1;
    const uint32_t per_row = (uint32_t)(D / vec / split);
    const uint64_t reciprocal = per_row == 1 ? 0 : ~0ull / per_row + 1;
    const long most = per_row > 0x40000000u ? 1 : 0x40000000L / per_row;      // rows a launch: places count in 32 bits
    for (long n0 = 0; n0 < N; n0 += most) {
        const long n = std::min(most, N - n0);
        const uint32_t total = (uint32_t)(n * per_row);
        const unsigned blocks = (total + 1023) / 1024 * split;
        const TI *idx = (const TI *)idx_ + n0;
        TY *y = (TY *)y_ + n0 * D;
#define XQ_EMB(VEC) \
    hipLaunchKernelGGL((embed_fwd_kernel<TW, TY, TI, VEC>), dim3(blocks), dim3(256), 0, s, idx, (const TW *)w, V, D, split, per_row, total, reciprocal, scale, y)
        if (vec == 8) XQ_EMB(8);
        else if (vec == 4) XQ_EMB(4);
        else XQ_EMB(1);
#undef XQ_EMB
    }
}

template <typename TG, typename TW>
void launch_sums(const void *g, long V, int D, float scale, const Plan &p, const uint32_t *order, const uint32_t *rows, const uint32_t *edge, float *part, void *dw,
                 hipStream_t s) {
    const bool a16 = (((uintptr_t)g | (uintptr_t)dw) & 15) == 0;
#define XQ_SUM(VEC)                                                                                                                          \
    {                                                                                                                                        \
        const int lanes = pow2_lanes(D, VEC), groups = 256 / lanes;                                                                          \
        const long rb = (V + groups - 1) / groups, pb = (2 * p.chunks + groups - 1) / groups;                                                \
        hipLaunchKernelGGL((embed_sum_kernel<TG, TW, VEC>), dim3((unsigned)(rb + pb)), dim3(256), 0, s, (const TG *)g, order, rows, edge, V, D, \
                           lanes, scale, 1u << p.chunk_bits, p.chunks, pb, (TW *)dw, part);                                                  \
    }
    if (a16 && D % 8 == 0 && sizeof(TG) == 2) XQ_SUM(8)
    else if (a16 && D % 4 == 0 && sizeof(TG) == 4) XQ_SUM(4)
    else XQ_SUM(1)
#undef XQ_SUM
    hipLaunchKernelGGL((embed_long_kernel<TW>), dim3((unsigned)((p.chunks + 7) / 8), (unsigned)std::min(8, (D + 63) / 64)), dim3(512), 0, s, part, rows, edge,
                       V, D, scale, 1u << p.chunk_bits, p.chunks, (TW *)dw);
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
    const int pitch = std::max(p.buckets, 1 << p.shift);
#define XQ_BIN(TI)                                                                                                                                  \
    hipLaunchKernelGGL((embed_bin_kernel<TI>), dim3(p.slices), dim3(BIN_THREADS), (size_t)(BIN_THREADS / 64 + 1) * pitch * 4, s, (const TI *)idx, (long)N, (long)V, \
                       (long)skip, p.shift, p.buckets, p.bucket_bits, pitch, list, starts)
    if (idx_i64) XQ_BIN(int64_t);
    else XQ_BIN(int32_t);
#undef XQ_BIN
#define XQ_SORT(THREADS)                                                                                                                              \
    hipLaunchKernelGGL((embed_sort_kernel<THREADS>), dim3(p.buckets), dim3(THREADS), (size_t)((THREADS / 64 + 1) << p.shift) * 4, s, list, starts, (long)V, \
                       p.shift, p.buckets, p.slices, rows, order, p.chunk_bits, edge)
    if (p.shift <= 9) XQ_SORT(1024);
    else XQ_SORT(512);           // 1024 rows a bucket: sixteen waves' counters would not fit the 64 KB of a launch
#undef XQ_SORT
    if (g_bf16 && dw_bf16) launch_sums<bf16, bf16>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else if (g_bf16) launch_sums<bf16, float>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else if (dw_bf16) launch_sums<float, bf16>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    else launch_sums<float, float>(g, V, D, scale, p, order, rows, edge, part, dw, s);
    return xq_check_launch(fn);
}
