// xq_xattn.hip — attention of one sequence to another one: queries (B, Nq, H, D), keys and values (B, Nk, Hk, D) of another length and with their own
// strides, H = G Hk (query head h reads kv head h / G), the valid keys of a sample given by a length and / or a mask; forward and backward, bf16 MFMA with fp32
// softmax statistics and sums (gfx950).
//
//   S = scale q k^T;  P = exp(S - lse) on valid keys, 0 elsewhere;  O = P v;  a sample without a valid key: O = 0, gradients 0, lse = -inf.
//   dv = P^T dO;  delta = sum_d dO O;  dS = P (dO v^T - delta);  dq = scale dS k;  dk = scale dS^T q  (dk, dv over the G heads that share them).
//
// The rows of one kv head are its G Nq (query, head) pairs, query-major: shared heads fill a tile's rows like more queries do, and their sum in dk / dv is the
// contraction over rows itself.  D is any multiple of 8 up to 128, computed in the next multiple of 32 (DT) with zeros behind it.
//
// Layouts (v_mfma_f32_32x32x16_bf16: A[i][k] lane = i, 8 consecutive k per lane half; B[k][j] lane = j; D[i][j] column = lane & 31, row = (r & 3) +
// 8 (r >> 2) + 4 (lane >> 5)): the forward and the dq kernel hold one row per lane (S^T = K Q^T, P stays in registers and is the B operand of O^T = V^T P^T;
// V^T comes from the row-major LDS tile through ds_read_b64_tr_b16), the dk / dv kernel one key per lane.
// Masked keys are zero rows in LDS and -inf in S: what lies in memory there (infinities, NaN) reaches nothing.
// Roundings to bf16: P and dS before their products (they are operands of the bf16 matrix instructions; fp16 would not hold the range of the other operand, two
// bf16 parts would double the products), the results once; everything else is fp32.  Against 64 bits the results are 0.0021 .. 0.0029 off in norm (rounding them
// alone: 0.0017, the operand's rounding as much again in squares, and for dq / dk what delta takes from the rounded O).
#include "xq_common.hpp"
#include "xq_internal.hpp"
#include "../../include/xq_ops.h"
#include <algorithm>
#include <math.h>
#include <type_traits>

using namespace xq;

namespace {

typedef short bf16x8 __attribute__((ext_vector_type(8)));
typedef short bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bfv2 __attribute__((ext_vector_type(2)));
typedef float fv2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct View {                      // a (B, N, heads, D) bf16 tensor: element strides, the last one is 1
    short *p;
    long sb, sn, sh;
};

struct Args {
    View q, k, v, dq, dk, dv;
    const short *out_in, *dout;    // (B, Nq, H, D) contiguous
    short *out;
    float *lse, *delta;            // (B, Hk, G Nq)
    float *part, *stat;            // split over keys / rows: fp32 slabs [split][...], running (maximum, sum) [split][B Hk][R][2]
    const void *lens;              // valid keys of a sample, or null
    const unsigned char *mask;     // (B, Nk), or null
    int lens_i64, B, Nq, Nk, H, Hk, G, D, R;
    unsigned long long g_reciprocal;   // of G (0: one)
    float scale;
    int nper, groups, swizzle, splits;
};

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    fv2 v = {a, b};
    bfv2 r = __builtin_convertvector(v, bfv2);   // v_cvt_pk_bf16_f32 (RNE)
    return __builtin_bit_cast(unsigned, r);
}
__device__ __forceinline__ bf16x8 pack8(const float *s) {
    uint4 u = make_uint4(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]), pack_bf16(s[4], s[5]), pack_bf16(s[6], s[7]));
    return __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ float bf_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// LDS by byte address (the swizzle below is a XOR on it)
template <typename T> using lds_ptr = T __attribute__((address_space(3))) *;
__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr<const char>)p; }
__device__ __forceinline__ bf16x8 lds_16(uint32_t at) { return *(lds_ptr<const bf16x8>)(uintptr_t)at; }
__device__ __forceinline__ bf16x4 lds_tr(uint32_t at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<bf16x4>)(uintptr_t)at); }

// A row-major bf16 tile in LDS, rows of 64, 128 or 256 bytes (96 columns lie in 256).  Chunk c (16 bytes) of row R is kept at chunk c ^ twist(R), so that both
// ways of reading meet all 64 banks: 16 rows at one chunk (the operands over the head dimension) and 4 rows x 4 chunks (the transpose reads).  A pitch of
// DT + 8 instead serves the first way only: half of the LDS cycles were conflicts (dk / dv at 128 columns 1140 us, then 1108).
template <int DT>
struct Tile {
    static constexpr int PITCH = DT > 64 ? 128 : DT, ROW = 2 * PITCH;
    static __device__ __forceinline__ uint32_t twist(uint32_t r) {
        if (DT > 64) return (r & 3) << 2 | (r >> 2 & 3);
        if (DT > 32) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
        return r >> 2 & 3;
    }
    static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t chunk) { return row * ROW + ((chunk ^ twist(row)) << 4); }
    // chunk 2 k + hh of row li (+ 16 n: the twist goes by R mod 16): base ^ 32 k
    static __device__ __forceinline__ uint32_t row_base(int li, int hh) { return place(li, hh); }
    // A fragment of the transposed tile: contraction rows row0 + {4 hh .. + 3, 8 + 4 hh ..} (row0 a multiple of 16), output rows = columns 32 q + (lane & 31).
    // ds_read_b64_tr_b16: in each 16 lanes, lane i receives element i & 3 of the 8 bytes that lanes 4 j + (i >> 2) point at
    static __device__ __forceinline__ uint32_t tr_base(int lane) {
        const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), chunk = 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
        return place(row, chunk) + 8 * (lane & 1);
    }
    static __device__ __forceinline__ bf16x8 tr_frag(uint32_t base, int row0, int q) {
        const bf16x4 lo = lds_tr((base ^ 64 * q) + row0 * ROW), hi = lds_tr((base ^ 64 * q ^ 32) + (row0 + 8) * ROW);      // twist(R + 8) = twist(R) ^ 2
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // the same for 16x16x32: 32 contraction rows from row0 (a multiple of 32; in an order of their own, the same for both operands), columns 16 q + (lane & 15)
    static __device__ __forceinline__ uint32_t tr16_base(int lane) {
        return place(8 * (lane >> 4 & 1) + 4 * (lane >> 5) + ((lane & 15) >> 2), (lane & 3) >> 1) + 8 * (lane & 1);
    }
    static __device__ __forceinline__ bf16x8 tr16_frag(uint32_t base, int row0, int q) {
        const bf16x4 lo = lds_tr((base ^ 32 * q) + row0 * ROW), hi = lds_tr((base ^ 32 * q) + (row0 + 16) * ROW);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// The largest of three, NaN if one is (v_maximum3_f32; fmaxf would make every operand canonical first).  Not inline asm: the wait that a matrix instruction's
// result needs before it is read is the compiler's, and it does not see into asm.
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

// Order for the scheduler: N matrix instructions with PER LDS reads each, the reads AHEAD of them (left to itself it puts every read right before its use, and
// the wave waits for LDS once a product: dk / dv at 4 x 4096 x 4352 x 16 x 128 1110 us instead of 1087, dq at 8 x 2048 x 2048 x 12 x 64 197 instead of 192)
template <int N, int PER, int AHEAD>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, PER * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// the larger of a lane's value and its partner's in the other half of the wave (through LDS the tile waits for it: 525 us instead of 510)
__device__ __forceinline__ float max_of_halves(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max3(__uint_as_float(both[0]), __uint_as_float(both[1]), x);
}

#define XA_MFMA(A, B, C) __builtin_amdgcn_mfma_f32_32x32x16_bf16((A), (B), (C), 0, 0, 0)
#define XA_MFMA16(A, B, C) __builtin_amdgcn_mfma_f32_16x16x32_bf16((A), (B), (C), 0, 0, 0)

__device__ __forceinline__ uint32_t quotient(uint32_t a, uint64_t reciprocal) { return reciprocal ? (uint32_t)__umul64hi((uint64_t)a, reciprocal) : a; }

// (b, kv head) and the tile of a block.  Where the (batch, kv head) pairs divide over the eight XCDs, the blocks of one pair share an XCD (round-robin: block id
// mod 8), whose L2 then holds its keys and values (or rows) once; otherwise they run on in order, so that no XCD idles.
__device__ __forceinline__ bool map_block(const Args &a, int &g, int &i) {
    const int L = blockIdx.x;
    if (a.swizzle) {
        const int slot = L >> 3, gl = slot / a.nper;
        i = slot - gl * a.nper;
        g = gl * 8 + (L & 7);
    } else {
        g = L / a.nper;
        i = L - g * a.nper;
    }
    return g < a.groups;
}

__device__ __forceinline__ int keys_of(const Args &a, int b) {
    if (!a.lens) return a.Nk;
    const long n = a.lens_i64 ? (long)((const int64_t *)a.lens)[b] : (long)((const int32_t *)a.lens)[b];
    return (int)(n < 0 ? 0 : n > a.Nk ? a.Nk : n);
}

// The valid ones of 64 keys, one bit each (the same in every lane).  A mask's bytes are fetched a tile ahead of the tile's own loads, which wait for them.
struct KeyBits {
    const unsigned char *mask;
    int len, on;
    __device__ __forceinline__ void fetch(int kv0) {
        if (!mask) return;
        const int key = kv0 + (int)(threadIdx.x & 63);
        on = 0;
        if (key < len) on = mask[key];
    }
    __device__ __forceinline__ uint64_t take(int kv0) const {
        const int left = len - kv0;
        const uint64_t bits = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
        return mask ? bits & __ballot(on != 0) : bits;
    }
};

__device__ __forceinline__ uint4 zero_unless(uint4 v, bool ok) {
    if (!ok) v = make_uint4(0u, 0u, 0u, 0u);
    return v;
}

// the sum over aligned groups of N = 4, 8 or 16 lanes, in each of them (lane permutations of the vector unit: through LDS each step would wait for it)
template <int N>
__device__ __forceinline__ float sum_of_lanes(float x) {
    auto moved = [](float y, auto control) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y), decltype(control)::value, 0xf, 0xf, true)); };
    x += moved(x, std::integral_constant<int, 0xB1>());                     // lanes 1 0 3 2 of four
    x += moved(x, std::integral_constant<int, 0x4E>());                     // lanes 2 3 0 1
    if (N >= 8) x += moved(x, std::integral_constant<int, 0x141>());        // lanes 7 .. 0 of eight
    if (N >= 16) x += moved(x, std::integral_constant<int, 0x140>());       // lanes 15 .. 0 of sixteen
    return x;
}

// 16 bytes at a byte offset of up to 2^31 behind a wave-uniform base; FAR reads zeros (a buffer's bounds check), so that what is masked or behind the head
// dimension costs an offset and no select on the data, and is never touched
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t FAR = 0x80000000u;
__device__ __forceinline__ uint4 load16(const short *base, uint32_t off) {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7fffffff, 0x00020000);
    return __builtin_bit_cast(uint4, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0));
}

// element offset of row r of kv head hk in a query-sided view
__device__ __forceinline__ long row_offset(const Args &a, const View &t, int b, int hk, int r) {
    const uint32_t tok = quotient((uint32_t)r, a.g_reciprocal), g = (uint32_t)r - tok * a.G;
    return b * t.sb + (long)tok * t.sn + (long)(hk * a.G + (int)g) * t.sh;
}

// ROWS rows into registers (CH 16-byte chunks a thread), then into a row-major LDS tile; a row whose bit is clear arrives as zeros
template <int DT, int ROWS, int THREADS>
struct Stage {
    static constexpr int PER_ROW = DT / 8, CH = (ROWS * PER_ROW + THREADS - 1) / THREADS;
    static constexpr bool EVEN = ROWS * PER_ROW % THREADS == 0;
    uint32_t off[CH];
    uint4 r[CH];
    static __device__ __forceinline__ int row(int c) { return (int)(threadIdx.x + THREADS * c) / PER_ROW; }
    static __device__ __forceinline__ int col(int c) { return (int)(threadIdx.x + THREADS * c) % PER_ROW * 8; }
    __device__ __forceinline__ void places(long sn, int D) {
#pragma unroll
        for (int c = 0; c < CH; ++c) off[c] = col(c) < D && (EVEN || row(c) < ROWS) ? (uint32_t)(row(c) * (int)sn + col(c)) * 2 : FAR;
    }
    __device__ __forceinline__ void load(const short *base, uint64_t bits) {
        if (~bits) {
#pragma unroll
            for (int c = 0; c < CH; ++c) r[c] = load16(base, (bits >> (row(c) & 63)) & 1 ? off[c] : FAR);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c) r[c] = load16(base, off[c]);
        }
    }
    // `left` rows, then the row at element offset `first` again
    __device__ __forceinline__ void load_repeating(const short *base, int left, uint32_t first) {
#pragma unroll
        for (int c = 0; c < CH; ++c) r[c] = load16(base, row(c) < left || off[c] == FAR ? off[c] : (first + col(c)) * 2);
    }
    __device__ __forceinline__ void store(uint32_t tile) const {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (EVEN || row(c) < ROWS) *(lds_ptr<u32x4>)(uintptr_t)(tile + Tile<DT>::place(row(c), col(c) / 8)) = __builtin_bit_cast(u32x4, r[c]);
    }
};

// one lane's 8-element chunks of a row: the B operand over the head dimension
template <int DT>
__device__ __forceinline__ void load_row(const short *row, int D, int hh, bf16x8 (&f)[DT / 16]) {
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
        const int col = 16 * s + 8 * hh;
        const uint4 x = *reinterpret_cast<const uint4 *>(row + (col < D ? col : 0));
        f[s] = __builtin_bit_cast(bf16x8, zero_unless(x, col < D));
    }
}

// a lane's column of an (output row, lane) accumulator block, rounded: 16 bytes a lane, the lane halves exchanging register quads.  Every lane takes part.
template <int DT>
__device__ __forceinline__ void store_row(short *row, int D, int hh, const f32x16 (&acc)[DT / 32], float factor, bool ok) {
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            const uint2 x = make_uint2(pack_bf16(acc[t][4 * q] * factor, acc[t][4 * q + 1] * factor), pack_bf16(acc[t][4 * q + 2] * factor, acc[t][4 * q + 3] * factor));
            const uint2 y = make_uint2(pack_bf16(acc[t][4 * q + 4] * factor, acc[t][4 * q + 5] * factor),
                                       pack_bf16(acc[t][4 * q + 6] * factor, acc[t][4 * q + 7] * factor));
            const auto e = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false);
            const auto f = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
            const int col = 32 * t + 8 * q + 8 * hh;
            if (ok && col < D) *reinterpret_cast<uint4 *>(row + col) = make_uint4(e[0], f[0], e[1], f[1]);
        }
}

// the same into an fp32 slab
template <int DT>
__device__ __forceinline__ void store_part(float *row, int D, int hh, const f32x16 (&acc)[DT / 32], bool ok) {
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = 32 * t + 8 * q + 4 * hh;
            if (ok && col < D) *reinterpret_cast<float4 *>(row + col) = make_float4(acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]);
        }
}

// lse in log2 units; that of a row without a finite score stands for P = 0 (exp2(-inf - 0)), not for NaN
__device__ __forceinline__ float log2_of(float lse) { return lse == -INFINITY ? 0.0f : lse * LOG2E; }

// share `part` of `parts` of n tiles
__device__ __forceinline__ void share(int n, int part, int parts, int &from, int &to) {
    from = (int)((long)n * part / parts);
    to = (int)((long)n * (part + 1) / parts);
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// forward: 128 rows of one (sample, kv head) a block, 32 a wave; 64-key tiles of K and V in two LDS buffers.  4 x 4096 x <= 4352 keys x 16 heads of 128: 515 us,
// 890 TFLOP/s, the matrix pipe busy 48 % of the cycles and the vector units 46 %; 128 x 256 x 257 x 12 heads of 64: 59 us, 3.4 TB/s, the vector units 60 %; one token
// of 16 samples over 4056 .. 8111 keys, 32 heads over 8 of 128: 82 us, 4.9 TB/s (the keys split over four blocks)
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int DT, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xattn_fwd_kernel(Args a) {
    typedef Tile<DT> T;
    constexpr int KS = DT / 16, OT = DT / 32, BYTES = 64 * T::ROW;
    __shared__ __attribute__((aligned(256))) char tiles[4 * BYTES];         // K 0, K 1, V 0, V 1
    const uint32_t Ks = lds_address(tiles), Vs = Ks + 2 * BYTES;
    int g, i;
    if (!map_block(a, g, i)) return;
    const int split = SPLIT ? i % a.splits : 0, rb = SPLIT ? i / a.splits : i;
    const int b = g / a.Hk, hk = g - b * a.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, hh = lane >> 5;
    const uint32_t row_at = T::row_base(li, hh), tr_at = T::tr_base(lane);
    const int len = keys_of(a, b);
    const short *kb = a.k.p + b * a.k.sb + hk * a.k.sh, *vb = a.v.p + b * a.v.sb + hk * a.v.sh;
    const float c = a.scale * LOG2E;

    const int r = rb * 128 + wave * 32 + li, rc = r < a.R ? r : a.R - 1;
    const bool wave_live = rb * 128 + wave * 32 < a.R;
    bf16x8 qf[KS];
    load_row<DT>(a.q.p + row_offset(a, a.q, b, hk, rc), a.D, hh, qf);

    f32x16 o[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] = 0.0f;
    // m is the reference exponent (log2 units), moved only when a tile's maximum passes it by more than 2^8: P <= 2^8 loses nothing in bf16 / fp32, and the
    // rescale becomes a rare branch.  l: the lane's share of the row's sum, in fp32 before P is rounded (a product of ones with P^T instead of the additions is
    // an eighth more matrix work at 128 columns: 552 us instead of 537)
    float m = -INFINITY, l = 0.0f;
    const f32x16 zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};

    int t0, t1;
    share((len + 63) / 64, split, SPLIT ? a.splits : 1, t0, t1);
    Stage<DT, 64, 256> sk, sv;
    sk.places(a.k.sn, a.D);
    sv.places(a.v.sn, a.D);
    KeyBits keys = {a.mask ? a.mask + (long)b * a.Nk : nullptr, len, 0};
    uint64_t bits = 0, next = 0;
    if (t0 < t1) {
        keys.fetch(t0 * 64);
        bits = keys.take(t0 * 64);
        sk.load(kb + t0 * 64L * a.k.sn, bits);
        sv.load(vb + t0 * 64L * a.v.sn, bits);
        keys.fetch(t0 * 64 + 64);
        sk.store(Ks);
        sv.store(Vs);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        if (t + 1 < t1) {
            next = keys.take(t * 64 + 64);
            sk.load(kb + (t + 1) * 64L * a.k.sn, next);
            sv.load(vb + (t + 1) * 64L * a.v.sn, next);
            keys.fetch(t * 64 + 128);
        }
        if (wave_live && bits) {
            const uint32_t K = Ks + cur * BYTES + row_at, V = Vs + cur * BYTES + tr_at;
            const bool wide = (bits >> 32) != 0;           // the second 32 keys of the tile hold one at least
            f32x16 s[2];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[h] = zero16;                             // (the second half also where none of its keys is valid: the choice would copy both halves at every tile: 545 us instead of 525)
#pragma unroll
                for (int k = 0; k < KS; ++k) s[h] = XA_MFMA(lds_16((K ^ 32 * k) + 32 * h * T::ROW), qf[k], s[h]);
            }
            __builtin_amdgcn_s_setprio(0);
            if (~bits) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w = (uint32_t)(bits >> (32 * h)) >> (4 * hh);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (!((w >> ((j & 3) + 8 * (j >> 2))) & 1u)) s[h][j] = -INFINITY;
                }
            }
            float mx = max3(s[0][0], s[0][1], s[0][2]), my = max3(s[1][0], s[1][1], s[1][2]);
#pragma unroll
            for (int j = 3; j < 15; j += 2) {
                mx = max3(mx, s[0][j], s[0][j + 1]);
                my = max3(my, s[1][j], s[1][j + 1]);
            }
            mx = max3(mx, s[0][15], max3(my, s[1][15], my));
            mx = max_of_halves(mx);
            const float cand = mx * c;
            if (__any(cand > m + 8.0f)) {
                const float mn = fmaxf(m, cand);
                const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);      // (a row without a key so far: m = mn = -inf)
                m = mn;
                l *= alpha;
#pragma unroll
                for (int q = 0; q < OT; ++q)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[q][j] *= alpha;
            }
            const float mref = m == -INFINITY ? 0.0f : m;      // (every score so far -inf: P is 0, not NaN)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && !wide) continue;
                float p[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[h][j], c, -mref));
#pragma unroll
                for (int j = 0; j < 16; ++j) l += p[j];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bf16x8 pk = pack8(p + 8 * k);
#pragma unroll
                    for (int q = 0; q < OT; ++q) o[q] = XA_MFMA(T::tr_frag(V, 32 * h + 16 * k, q), pk, o[q]);
                }
            }
        }
        if (t + 1 < t1) {
            sk.store(Ks + (cur ^ 1) * BYTES);
            sv.store(Vs + (cur ^ 1) * BYTES);
            bits = next;
        }
        __syncthreads();
    }
    l += __shfl_xor(l, 32);          // the lane halves hold other keys of the row
    const bool ok = r < a.R;
    if (SPLIT) {
        const long slot = ((long)split * a.groups + g) * a.R + (ok ? r : 0);
        store_part<DT>(a.part + slot * a.D, a.D, hh, o, ok);
        if (ok && hh == 0) *reinterpret_cast<float2 *>(a.stat + 2 * slot) = make_float2(m, l);
    } else {
        const uint32_t tok = quotient((uint32_t)rc, a.g_reciprocal), gg = (uint32_t)rc - tok * a.G;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        store_row<DT>(a.out + (((long)b * a.Nq + tok) * a.H + hk * a.G + gg) * a.D, a.D, hh, o, inv, ok);
        if (a.lse && ok && hh == 0) a.lse[(long)g * a.R + r] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// forward of at most 32 rows a kv head over at most 1024 keys (serving: one token, its heads, one image's or text's states): the four waves share out the keys,
// each with its own 32-key tiles and no meeting with the others until their results are joined.  K and V go through LDS tiles of the wave's own (loads of whole
// rows), fetched a tile ahead.  Bound by latency: one token over 257 keys, 12 heads of 64, takes 6.0 us (in the tiles of the many-row kernel, where one
// wave of four has rows, 8.8).  Over more keys the many-row kernel with its keys split over blocks reads as fast (16 samples over 4056 .. 8111 keys: 82 us, here
// 84) and a block's share is no longer one wave's chain.
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256, 2) void xattn_few_rows_kernel(Args a) {
    typedef Tile<DT> T;
    constexpr int KS = DT / 16, OT = DT / 32, PER_ROW = DT / 8, CH = 32 * PER_ROW / 64, BYTES = 32 * T::ROW, PITCH = DT + 4;
    constexpr int JOIN = 4 * 32 * PITCH * 4;
    __shared__ __attribute__((aligned(256))) char mem[JOIN > 8 * BYTES ? JOIN : 8 * BYTES];       // the waves' K and V tiles, then their results
    __shared__ float2 stat[4][32];
    const int g = blockIdx.x;
    const int b = g / a.Hk, hk = g - b * a.Hk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31,
              hh = lane >> 5;          // (the wave's number is the same in its lanes: the buffers' bases lie in scalar registers: 6.0 us instead of 6.9)
    const uint32_t Kw = lds_address(mem) + 2 * wave * BYTES, Vw = Kw + BYTES, row_at = Kw + T::row_base(li, hh), tr_at = Vw + T::tr_base(lane);
    const int len = keys_of(a, b);
    const short *kb = a.k.p + b * a.k.sb + hk * a.k.sh, *vb = a.v.p + b * a.v.sb + hk * a.v.sh;
    const float c = a.scale * LOG2E;
    bf16x8 qf[KS];
    load_row<DT>(a.q.p + row_offset(a, a.q, b, hk, li < a.R ? li : a.R - 1), a.D, hh, qf);

    uint32_t k_at[CH], v_at[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int id = lane + 64 * i, row = id / PER_ROW, col = id % PER_ROW * 8;
        k_at[i] = col < a.D ? (uint32_t)(row * (int)a.k.sn + col) * 2 : FAR;
        v_at[i] = col < a.D ? (uint32_t)(row * (int)a.v.sn + col) * 2 : FAR;
    }
    KeyBits keys = {a.mask ? a.mask + (long)b * a.Nk : nullptr, len, 0};
    uint4 kr[CH], vr[CH];
    auto load = [&](int t, uint32_t bits) {
        const short *K = kb + t * 32L * a.k.sn, *V = vb + t * 32L * a.v.sn;
        if (~bits) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const bool on = (bits >> ((lane + 64 * i) / PER_ROW)) & 1;
                kr[i] = load16(K, on ? k_at[i] : FAR);
                vr[i] = load16(V, on ? v_at[i] : FAR);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i) kr[i] = load16(K, k_at[i]);
#pragma unroll
            for (int i = 0; i < CH; ++i) vr[i] = load16(V, v_at[i]);
        }
    };

    f32x16 o[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const f32x16 zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int t0 = wave, t1 = (len + 31) / 32;
    uint32_t bits = 0, next = 0;
    if (t0 < t1) {
        keys.fetch(t0 * 32);
        bits = (uint32_t)keys.take(t0 * 32);
        load(t0, bits);
        keys.fetch(t0 * 32 + 128);
    }
    for (int t = t0; t < t1; t += 4) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = lane + 64 * i;
            const uint32_t at = T::place(id / PER_ROW, id % PER_ROW);
            *(lds_ptr<u32x4>)(uintptr_t)(Kw + at) = __builtin_bit_cast(u32x4, kr[i]);
            *(lds_ptr<u32x4>)(uintptr_t)(Vw + at) = __builtin_bit_cast(u32x4, vr[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // the lanes read what other lanes of the wave have written (in order for the hardware, not for the compiler)
        if (t + 4 < t1) {
            next = (uint32_t)keys.take(t * 32 + 128);
            load(t + 4, next);
            keys.fetch(t * 32 + 256);
        }
        f32x16 s = zero16;
#pragma unroll
        for (int k = 0; k < KS; ++k) s = XA_MFMA(lds_16(row_at ^ 32 * k), qf[k], s);
        if (~bits) {
            const uint32_t w = bits >> (4 * hh);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (!((w >> ((j & 3) + 8 * (j >> 2))) & 1u)) s[j] = -INFINITY;
        }
        float mx = max3(s[0], s[1], s[2]);
#pragma unroll
        for (int j = 3; j < 15; j += 2) mx = max3(mx, s[j], s[j + 1]);
        mx = max3(mx, s[15], s[15]);
        mx = max_of_halves(mx);
        const float cand = mx * c;
        if (__any(cand > m + 8.0f)) {
            const float mn = fmaxf(m, cand);
            const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int q = 0; q < OT; ++q)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[q][j] *= alpha;
        }
        const float mref = m == -INFINITY ? 0.0f : m;
        float p[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c, -mref));
#pragma unroll
        for (int j = 0; j < 16; ++j) l += p[j];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const bf16x8 pk = pack8(p + 8 * k);
#pragma unroll
            for (int q = 0; q < OT; ++q) o[q] = XA_MFMA(T::tr_frag(tr_at, 16 * k, q), pk, o[q]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        bits = next;
    }
    l += __shfl_xor(l, 32);
    __syncthreads();
    float *sum = reinterpret_cast<float *>(mem);
    if (li < a.R) {
        float *row = sum + (wave * 32 + li) * PITCH;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4 *>(row + 32 * t + 8 * q + 4 * hh) = make_float4(o[t][4 * q], o[t][4 * q + 1], o[t][4 * q + 2], o[t][4 * q + 3]);
        if (hh == 0) stat[wave][li] = make_float2(m, l);
    }
    __syncthreads();
    const int per_row = a.D / 4;
    for (int id = threadIdx.x; id < a.R * per_row; id += 256) {
        const int r = id / per_row, col = (id - r * per_row) * 4;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, stat[w][r].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 ml = stat[w][r];
            const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            const float4 y = *reinterpret_cast<const float4 *>(sum + (w * 32 + r) * PITCH + col);
            L = fmaf(ml.y, f, L);
            x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const uint32_t tok = quotient((uint32_t)r, a.g_reciprocal), gg = (uint32_t)r - tok * a.G;
        *reinterpret_cast<uint2 *>(a.out + (((long)b * a.Nq + tok) * a.H + hk * a.G + gg) * a.D + col) =
            make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        if (a.lse && col == 0) a.lse[(long)g * a.R + r] = L == 0.0f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * LN2;
    }
}

// the slabs of a split over keys: O = sum_s w_s O_s / sum_s w_s l_s, w_s = 2^(m_s - max m); four columns a thread
__global__ __launch_bounds__(256) void xattn_join_kernel(Args a, int per_row, unsigned long long row_reciprocal, long total) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const uint32_t row = quotient((uint32_t)id, row_reciprocal);          // g R + r (the host keeps total below 2^32)
    const int col = ((uint32_t)id - row * per_row) * 4;
    const long rows = (long)a.groups * a.R;
    float M = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.stat[2 * (s * rows + row)]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.stat + 2 * (s * rows + row));
        const float4 x = *reinterpret_cast<const float4 *>(a.part + (s * rows + row) * a.D + col);
        const float w = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
        l = fmaf(ml.y, w, l);
        o.x = fmaf(x.x, w, o.x); o.y = fmaf(x.y, w, o.y); o.z = fmaf(x.z, w, o.z); o.w = fmaf(x.w, w, o.w);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int g = row / a.R, r = row - (long)g * a.R, b = g / a.Hk, hk = g - b * a.Hk;
    const uint32_t tok = quotient((uint32_t)r, a.g_reciprocal), gg = (uint32_t)r - tok * a.G;
    *reinterpret_cast<uint2 *>(a.out + (((long)b * a.Nq + tok) * a.H + hk * a.G + gg) * a.D + col) =
        make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    if (a.lse && col == 0) a.lse[row] = l == 0.0f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// dq: one row per lane as the forward; delta in the prologue, written for the dk / dv kernel behind it.  4 x 4096 x <= 4352 keys x 16 heads of 128: 720 us,
// 950 TFLOP/s, the matrix pipe busy half of the cycles
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int DT, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xattn_dq_kernel(Args a) {
    typedef Tile<DT> T;
    constexpr int KS = DT / 16, OT = DT / 32, BYTES = 64 * T::ROW;
    __shared__ __attribute__((aligned(256))) char tiles[4 * BYTES];         // K 0, K 1, V 0, V 1
    const uint32_t Ks = lds_address(tiles), Vs = Ks + 2 * BYTES;
    int g, i;
    if (!map_block(a, g, i)) return;
    const int split = SPLIT ? i % a.splits : 0, rb = SPLIT ? i / a.splits : i;
    const int b = g / a.Hk, hk = g - b * a.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, hh = lane >> 5;
    const uint32_t row_at = T::row_base(li, hh), tr_at = T::tr_base(lane);
    const int len = keys_of(a, b);
    const short *kb = a.k.p + b * a.k.sb + hk * a.k.sh, *vb = a.v.p + b * a.v.sb + hk * a.v.sh;
    const float c = a.scale * LOG2E;

    const int r = rb * 128 + wave * 32 + li, rc = r < a.R ? r : a.R - 1;
    const bool wave_live = rb * 128 + wave * 32 < a.R, ok = r < a.R;
    bf16x8 qf[KS], df[KS];
    load_row<DT>(a.q.p + row_offset(a, a.q, b, hk, rc), a.D, hh, qf);
    const uint32_t tok = quotient((uint32_t)rc, a.g_reciprocal), gg = (uint32_t)rc - tok * a.G;
    const long orow = (((long)b * a.Nq + tok) * a.H + hk * a.G + gg) * a.D;
    load_row<DT>(a.dout + orow, a.D, hh, df);
    float delta = 0.0f;
    {
        bf16x8 of[KS];
        load_row<DT>(a.out_in + orow, a.D, hh, of);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const uint4 x = __builtin_bit_cast(uint4, of[k]), y = __builtin_bit_cast(uint4, df[k]);
            delta = fmaf(bf_lo(x.x), bf_lo(y.x), delta); delta = fmaf(bf_hi(x.x), bf_hi(y.x), delta);
            delta = fmaf(bf_lo(x.y), bf_lo(y.y), delta); delta = fmaf(bf_hi(x.y), bf_hi(y.y), delta);
            delta = fmaf(bf_lo(x.z), bf_lo(y.z), delta); delta = fmaf(bf_hi(x.z), bf_hi(y.z), delta);
            delta = fmaf(bf_lo(x.w), bf_lo(y.w), delta); delta = fmaf(bf_hi(x.w), bf_hi(y.w), delta);
        }
        delta += __shfl_xor(delta, 32);
        if (hh == 0 && ok && split == 0) a.delta[(long)g * a.R + r] = delta;
    }
    const float lse2 = log2_of(a.lse[(long)g * a.R + rc]);

    f32x16 acc[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[t][j] = 0.0f;

    int t0, t1;
    share((len + 63) / 64, split, SPLIT ? a.splits : 1, t0, t1);
    Stage<DT, 64, 256> sk, sv;
    sk.places(a.k.sn, a.D);
    sv.places(a.v.sn, a.D);
    KeyBits keys = {a.mask ? a.mask + (long)b * a.Nk : nullptr, len, 0};
    uint64_t bits = 0, next = 0;
    if (t0 < t1) {
        keys.fetch(t0 * 64);
        bits = keys.take(t0 * 64);
        sk.load(kb + t0 * 64L * a.k.sn, bits);
        sv.load(vb + t0 * 64L * a.v.sn, bits);
        keys.fetch(t0 * 64 + 64);
        sk.store(Ks);
        sv.store(Vs);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        if (t + 1 < t1) {
            next = keys.take(t * 64 + 64);
            sk.load(kb + (t + 1) * 64L * a.k.sn, next);
            sv.load(vb + (t + 1) * 64L * a.v.sn, next);
            keys.fetch(t * 64 + 128);
        }
        if (wave_live && bits) {
            const uint32_t K = Ks + cur * BYTES + row_at, V = Vs + cur * BYTES + row_at, KT = Ks + cur * BYTES + tr_at;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && !(bits >> 32)) continue;         // no valid key among the second 32
                f32x16 s, p;
#pragma unroll
                for (int j = 0; j < 16; ++j) { s[j] = 0.0f; p[j] = 0.0f; }
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    s = XA_MFMA(lds_16((K ^ 32 * k) + 32 * h * T::ROW), qf[k], s);
                    p = XA_MFMA(lds_16((V ^ 32 * k) + 32 * h * T::ROW), df[k], p);
                }
                if (DT <= 96) reads_ahead<2 * KS, 1, 4>();         // (at 128 columns that many registers are not there: 725 us instead of 711)
                const uint32_t w = (uint32_t)(bits >> (32 * h)) >> (4 * hh);
                float d[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) d[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c, -lse2)) * (p[j] - delta);      // scale: once, in the end
                if (~bits) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (!((w >> ((j & 3) + 8 * (j >> 2))) & 1u)) d[j] = 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bf16x8 dk = pack8(d + 8 * k);
#pragma unroll
                    for (int q = 0; q < OT; ++q) acc[q] = XA_MFMA(T::tr_frag(KT, 32 * h + 16 * k, q), dk, acc[q]);
                }
                if (DT <= 96) reads_ahead<2 * OT, 2, 2>();
            }
        }
        if (t + 1 < t1) {
            sk.store(Ks + (cur ^ 1) * BYTES);
            sv.store(Vs + (cur ^ 1) * BYTES);
            bits = next;
        }
        __syncthreads();
    }
    if (SPLIT) {
        const long slot = ((long)split * a.groups + g) * a.R + (ok ? r : 0);
        store_part<DT>(a.part + slot * a.D, a.D, hh, acc, ok);
    } else {
        store_row<DT>(a.dq.p + row_offset(a, a.dq, b, hk, rc), a.D, hh, acc, a.scale, ok);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// REPEATED ROWS: in the last tile of rows of the two kernels below, those behind the last hold q of the tile's first row, dO = 0, lse = inf and delta = 0: P and dS are 0
// there.  Not q = 0: that times a key that holds an infinity is NaN, where every real row may have P = 0 (a score of -inf) and the key zero gradients; with a real
// row's q a score is NaN or inf only where it is in that row too.
// dk, dv: one key per lane, 32 W keys of one (sample, kv head) a block; tiles of QT rows of q and dO (and lse, delta) in two LDS buffers.
// 4 x 4096 x <= 4352 keys x 16 heads of 128: 1075 us, 850 TFLOP/s, the matrix pipe busy 43 % of the cycles: the waves (two a SIMD, their registers full) wait for LDS
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int DT, int W, bool SPLIT>
__global__ __launch_bounds__(64 * W, DT > 64 ? 2 : 3) void xattn_dkdv_kernel(Args a) {
    typedef Tile<DT> T;
    // 64 rows a tile where eight waves fill the CU by themselves: half of the meetings (1140 us instead of 1169)
    constexpr int QT = W == 8 ? 64 : 32, KS = DT / 16, OT = DT / 32, BYTES = QT * T::ROW;
    // a wave's own 32 rows of V: only at 96 columns do its fragments stay in registers beside the accumulators (elsewhere that would cost a wave a SIMD)
    constexpr bool V_IN_LDS = DT != 96;
    // at 128 columns the products begin at -lse / scale and -delta instead of zero (two operations a score less: 1135 -> 1082 us at 4 x 4096 x 4352 x 16); at 64 the
    // wait for the two before the first product costs more than that (121 -> 140 us at 128 x 256 x 257 x 12 heads)
    constexpr bool BEGIN = DT > 96;
    __shared__ __attribute__((aligned(256))) char tiles[4 * BYTES + (V_IN_LDS ? 32 * W * T::ROW : 0)];      // q 0, q 1, dO 0, dO 1, v
    __shared__ __attribute__((aligned(16))) float Ls[2][QT];
    __shared__ __attribute__((aligned(16))) float Ds[2][QT];
    const uint32_t Qs = lds_address(tiles), Os = Qs + 2 * BYTES, Vs = Qs + 4 * BYTES;
    int g, i;
    if (!map_block(a, g, i)) return;
    const int split = SPLIT ? i % a.splits : 0, kbk = SPLIT ? i / a.splits : i;
    const int b = g / a.Hk, hk = g - b * a.Hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const uint32_t row_at = T::row_base(li, hh), tr_at = T::tr_base(lane);
    const int len = keys_of(a, b);
    const float c = a.scale * LOG2E;
    const float lse_factor = BEGIN ? -1.0f / c : 1.0f;
    const float *lse = a.lse + (long)g * a.R, *dlt = a.delta + (long)g * a.R;

    const int n = (kbk * W + wave) * 32 + li, nc = n < a.Nk ? n : a.Nk - 1;
    bool valid = n < len;
    if (a.mask && valid) valid = a.mask[(long)b * a.Nk + n] != 0;
    const bool wave_live = __any(valid);      // a wave without a valid key only helps to stage
    bf16x8 kf[KS], vf[KS];
    load_row<DT>(a.k.p + b * a.k.sb + hk * a.k.sh + (long)nc * a.k.sn, a.D, hh, kf);
    load_row<DT>(a.v.p + b * a.v.sb + hk * a.v.sh + (long)nc * a.v.sn, a.D, hh, vf);
    if (V_IN_LDS) {
#pragma unroll
        for (int k = 0; k < KS; ++k) *(lds_ptr<bf16x8>)(uintptr_t)(Vs + wave * 32 * T::ROW + (row_at ^ 32 * k)) = vf[k];
    }

    f32x16 dk[OT], dv[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) { dk[t][j] = 0.0f; dv[t][j] = 0.0f; }

    // row r0 + i of a tile: token (r0 + i) / G.  Where G divides QT its offset from the tile's first token is the same in every tile
    Stage<DT, QT, 64 * W> sq, so;
    const long on = (long)a.H * a.D, oh = a.D;
    float rl = 0.0f;
    int rows = 0;
    auto places = [&](int g0) {
#pragma unroll
        for (int ch = 0; ch < sq.CH; ++ch) {
            const uint32_t rr = g0 + sq.row(ch), tok = quotient(rr, a.g_reciprocal), gg = rr - tok * a.G;
            const bool ok = sq.col(ch) < a.D && (sq.EVEN || sq.row(ch) < QT);
            sq.off[ch] = ok ? (tok * (uint32_t)a.q.sn + gg * (uint32_t)a.q.sh + sq.col(ch)) * 2 : FAR;
            so.off[ch] = ok ? (tok * (uint32_t)on + gg * (uint32_t)oh + sq.col(ch)) * 2 : FAR;
        }
    };
    const bool same_places = QT % a.G == 0;
    places(0);
    auto load = [&](int r0) {
        const int tok0 = (int)quotient((uint32_t)r0, a.g_reciprocal), left = a.R - r0;
        if (!same_places) places(r0 - tok0 * a.G);
        const uint64_t bits = left >= QT ? ~0ull : (1ull << left) - 1;
        const short *q0 = a.q.p + b * a.q.sb + tok0 * a.q.sn + (long)hk * a.G * a.q.sh;
        if (left >= QT) sq.load(q0, ~0ull);
        else sq.load_repeating(q0, left, (uint32_t)(r0 - tok0 * a.G) * (uint32_t)a.q.sh);
        so.load(a.dout + ((long)b * a.Nq + tok0) * on + (long)hk * a.G * oh, bits);
        if (tid < 2 * QT) {
            const int r = min(r0 + tid % QT, a.R - 1);
            rl = tid < QT ? lse[r] : dlt[r];              // (what is made of it waits for it: in store)
        }
        rows = left;
    };
    auto store = [&](int buf) {
        sq.store(Qs + buf * BYTES);
        so.store(Os + buf * BYTES);
        if (tid < QT) Ls[buf][tid] = tid < rows ? log2_of(rl) * lse_factor : BEGIN ? -INFINITY : INFINITY;
        else if (tid < 2 * QT) Ds[buf][tid - QT] = tid - QT >= rows ? 0.0f : BEGIN ? -rl : rl;
    };

    int t0, t1;
    share(kbk * 32 * W < len ? (a.R + QT - 1) / QT : 0, split, SPLIT ? a.splits : 1, t0, t1);
    if (t0 < t1) {
        load(t0 * QT);
        store(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        if (t + 1 < t1) load(t * QT + QT);
        if (wave_live) {
#pragma unroll 1
        for (int h = 0; h < QT / 32; ++h) {
            if (h && t * QT + 32 * h >= a.R) break;
            const uint32_t Qh = Qs + cur * BYTES + 32 * h * T::ROW, Oh = Qh + 2 * BYTES, Q = Qh + row_at, O = Oh + row_at, Vw = Vs + wave * 32 * T::ROW + row_at;
            // register j <-> row (j & 3) + 8 (j >> 2) + 4 hh of the tile; rows behind the last: REPEATED ROWS above
            f32x16 s, p;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&Ls[cur][32 * h + 8 * q + 4 * hh]);
                const f32x4 d4 = *reinterpret_cast<const f32x4 *>(&Ds[cur][32 * h + 8 * q + 4 * hh]);
#pragma unroll
                for (int j = 0; j < 4; ++j) { s[4 * q + j] = BEGIN ? l4[j] : 0.0f; p[4 * q + j] = BEGIN ? d4[j] : 0.0f; }
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                s = XA_MFMA(lds_16(Q ^ 32 * k), kf[k], s);
                p = XA_MFMA(lds_16(O ^ 32 * k), V_IN_LDS ? lds_16(Vw ^ 32 * k) : vf[k], p);
            }
            reads_ahead<2 * KS, V_IN_LDS ? 2 : 1, 2>();
            float e[16], d[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&Ls[cur][32 * h + 8 * q + 4 * hh]);
                const f32x4 d4 = *reinterpret_cast<const f32x4 *>(&Ds[cur][32 * h + 8 * q + 4 * hh]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    e[4 * q + j] = __builtin_amdgcn_exp2f(BEGIN ? s[4 * q + j] * c : fmaf(s[4 * q + j], c, -l4[j]));
                    d[4 * q + j] = e[4 * q + j] * (BEGIN ? p[4 * q + j] : p[4 * q + j] - d4[j]);
                }
            }
            const uint32_t ot = Oh + tr_at, qt = Qh + tr_at;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bf16x8 pb = pack8(e + 8 * k), db = pack8(d + 8 * k);
#pragma unroll
                for (int q = 0; q < OT; ++q) {
                    dv[q] = XA_MFMA(T::tr_frag(ot, 16 * k, q), pb, dv[q]);
                    dk[q] = XA_MFMA(T::tr_frag(qt, 16 * k, q), db, dk[q]);
                }
            }
            reads_ahead<4 * OT, 2, 2>();
        }
        }
        if (t + 1 < t1) store(cur ^ 1);
        __syncthreads();
    }
    // a masked key's column holds what its bytes gave: zero goes out for it
    if (!valid) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) { dk[t][j] = 0.0f; dv[t][j] = 0.0f; }
    }
    const bool ok = n < a.Nk;
    if (SPLIT) {
        const long slots = (long)a.groups * a.Nk, slot = (long)g * a.Nk + nc;
        float *pk = a.part + (2 * split * slots + slot) * a.D, *pv = a.part + ((2 * split + 1) * slots + slot) * a.D;
        store_part<DT>(pk, a.D, hh, dk, ok);
        store_part<DT>(pv, a.D, hh, dv, ok);
    } else {
        store_row<DT>(a.dk.p + b * a.dk.sb + hk * a.dk.sh + (long)nc * a.dk.sn, a.D, hh, dk, a.scale, ok);
        store_row<DT>(a.dv.p + b * a.dv.sb + hk * a.dv.sh + (long)nc * a.dv.sn, a.D, hh, dv, 1.0f, ok);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// the whole backward of a (sample, kv head) whose keys fit one block (up to 32 W of them): one key per lane as in the dk / dv kernel; dS also goes to LDS
// (key-major), and the waves share out dq = dS k of the tile before.  q, dO and out are read once, P and dP computed once: five products instead of seven.
// 128 x 256 rows x 257 keys x 12 heads of 64 (nine waves): 158 us, 2.5 TB/s of its 400 MB and 410 TFLOP/s.  Bound by latency: the vector units and LDS are busy 33 % of
// the cycles each, the matrix pipe 22 %, and the waves wait half of theirs (a CU holds one such block: nothing runs beside its first loads and last stores,
// 50 us of it).
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int DT, int W, bool SPLIT>
__global__ __launch_bounds__(64 * W, DT > 64 ? 2 : 3) void xattn_bwd_kernel(Args a) {
    typedef Tile<DT> T;
    typedef Tile<32> TS;
    constexpr int QT = 32, KS = DT / 16, OT = DT / 32, BYTES = QT * T::ROW, SBYTES = 32 * W * TS::ROW;
    constexpr int SB = DT > 64 ? 1 : 2;                     // buffers of dS: with one, a second meeting a tile, but two blocks a CU
    // at 128 columns the next tile is fetched when the scores are done with: beside them there are no registers for it (8 x 1024 x 128 keys x 32 heads over 8: 124 us
    // instead of 107; q in one step with the others 109)
    constexpr bool LATE = DT > 96;
    constexpr bool V_IN_LDS = W == 9;                       // (with four waves a block fewer blocks would fit a CU)
    // dq: NA x NB tiles of 16 columns x 16 rows a wave
    constexpr int NA = W == 4 ? (DT == 96 ? 3 : DT == 128 ? 2 : 1) : 1, NB = W == 4 && (DT == 64 || DT == 128) ? 2 : 1, FIRST = W == 4 ? 0 : 1;
    // staging: 16 bytes of dO and out, and of q, a thread; where there are threads enough, other threads take q
    constexpr int PR = DT > 64 ? 16 : DT / 8, CHUNKS = QT * PR;
    constexpr bool ROLES = 64 * W >= 2 * CHUNKS;
    constexpr int CH = ROLES ? 1 : CHUNKS / (64 * W);
    static_assert(ROLES || CHUNKS % (64 * W) == 0, "whole rounds");
    __shared__ __attribute__((aligned(256))) char tiles[4 * BYTES + (V_IN_LDS ? 2 : 1) * 32 * W * T::ROW + SB * SBYTES];      // q 0, q 1, dO 0, dO 1, k, dS, v
    __shared__ __attribute__((aligned(16))) float Ls[2][QT];
    __shared__ __attribute__((aligned(16))) float Ds[2][QT];
    const uint32_t Qs = lds_address(tiles), Os = Qs + 2 * BYTES, Kb = Qs + 4 * BYTES, Sb = Kb + 32 * W * T::ROW, Vb = Sb + SB * SBYTES;
    int g, split;
    if (!map_block(a, g, split)) return;
    const int b = g / a.Hk, hk = g - b * a.Hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, hh = lane >> 5;
    const uint32_t row_at = T::row_base(li, hh), tr_at = T::tr_base(lane);
    const int len = keys_of(a, b);
    const float c = a.scale * LOG2E;
    const float lse_factor = -1.0f / c;
    const float *lse = a.lse + (long)g * a.R;
    const unsigned char *mask = a.mask ? a.mask + (long)b * a.Nk : nullptr;
    const short *kb = a.k.p + b * a.k.sb + hk * a.k.sh;

    const int n = wave * 32 + li, nc = n < a.Nk ? n : a.Nk - 1;
    bool valid = n < len;
    if (mask && valid) valid = mask[n] != 0;
    const bool wave_live = __any(valid), all_valid = __all(valid);
    // (the prologue's loads are all in flight before the first is waited for)
    bf16x8 vf[KS];
    const short *vb = a.v.p + b * a.v.sb + hk * a.v.sh;
    if (!V_IN_LDS) load_row<DT>(vb + (long)nc * a.v.sn, a.D, hh, vf);
    uint4 kr[DT / 16], vr[DT / 16];
#pragma unroll
    for (int j = 0; j < DT / 16; ++j) {
        const int id = tid + 64 * W * j, row = id / (DT / 8), chunk = id % (DT / 8);
        bool there = row < len && 8 * chunk < a.D;
        if (mask && there) there = mask[row] != 0;
        kr[j] = vr[j] = make_uint4(0u, 0u, 0u, 0u);
        if (there) kr[j] = *reinterpret_cast<const uint4 *>(kb + (long)row * a.k.sn + 8 * chunk);
        if (V_IN_LDS && there) vr[j] = *reinterpret_cast<const uint4 *>(vb + (long)row * a.v.sn + 8 * chunk);
    }
    if (!wave_live) {
        for (int j = 0; j < SB; ++j)
            for (int i = lane; i < 32 * TS::ROW / 16; i += 64)
                *(lds_ptr<u32x4>)(uintptr_t)(Sb + j * SBYTES + wave * 32 * TS::ROW + 16 * i) = __builtin_bit_cast(u32x4, make_uint4(0u, 0u, 0u, 0u));
    }

    f32x16 dk[OT], dv[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) { dk[t][j] = 0.0f; dv[t][j] = 0.0f; }

    const long on = (long)a.H * a.D, oh = a.D;
    const int role = ROLES ? wave / (CHUNKS / 64) : 0;
    uint32_t off_q[CH], off_o[CH];
    uint4 rq[CH], rd[CH], ro[CH];
    float rl = 0.0f;
    int rows = 0;
    auto row_of = [&](int ch) { return (ROLES ? tid % CHUNKS : tid + 64 * W * ch) / PR; };
    auto chunk_of = [&](int ch) { return (ROLES ? tid % CHUNKS : tid + 64 * W * ch) % PR; };
    // row r0 + i of a tile: token (r0 + i) / G.  Where G divides QT its offset from the tile's first token is the same in every tile
    auto places = [&](int g0) {
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
            const uint32_t rr = g0 + row_of(ch), tok = quotient(rr, a.g_reciprocal), gg = rr - tok * a.G;
            const int col = 8 * chunk_of(ch);
            off_q[ch] = col < a.D ? (tok * (uint32_t)a.q.sn + gg * (uint32_t)a.q.sh + col) * 2 : FAR;
            off_o[ch] = col < a.D ? (tok * (uint32_t)on + gg * (uint32_t)oh + col) * 2 : FAR;
        }
    };
    const bool same_places = QT % a.G == 0;
    places(0);
    auto load_q = [&](int r0) {
        const int tok0 = (int)quotient((uint32_t)r0, a.g_reciprocal), left = a.R - r0;
        if (!ROLES || role == 1) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch)
                rq[ch] = load16(a.q.p + b * a.q.sb + tok0 * a.q.sn + (long)hk * a.G * a.q.sh,
                                row_of(ch) < left || off_q[ch] == FAR ? off_q[ch] : ((uint32_t)(r0 - tok0 * a.G) * (uint32_t)a.q.sh + 8 * chunk_of(ch)) * 2);
        }
    };
    auto load = [&](int r0) {
        const int tok0 = (int)quotient((uint32_t)r0, a.g_reciprocal), left = a.R - r0;
        if (!same_places) places(r0 - tok0 * a.G);
        const long o = ((long)b * a.Nq + tok0) * on + (long)hk * a.G * oh;
        if (role == 0) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                const uint32_t at = row_of(ch) < left ? off_o[ch] : FAR;
                rd[ch] = load16(a.dout + o, at);
                ro[ch] = load16(a.out_in + o, at);
            }
        }
        if (!LATE) load_q(r0);
        if (tid < QT) rl = lse[tid < left ? r0 + tid : r0];            // (what is made of it waits for it: in store)
        rows = left;
    };
    auto store = [&](int buf) {
        if (role == 0) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                const uint4 x = rd[ch], y = ro[ch];
                float s = bf_lo(x.x) * bf_lo(y.x);
                s = fmaf(bf_hi(x.x), bf_hi(y.x), s);
                s = fmaf(bf_lo(x.y), bf_lo(y.y), s); s = fmaf(bf_hi(x.y), bf_hi(y.y), s);
                s = fmaf(bf_lo(x.z), bf_lo(y.z), s); s = fmaf(bf_hi(x.z), bf_hi(y.z), s);
                s = fmaf(bf_lo(x.w), bf_lo(y.w), s); s = fmaf(bf_hi(x.w), bf_hi(y.w), s);
                s = sum_of_lanes<PR>(s);
                if (chunk_of(ch) == 0) Ds[buf][row_of(ch)] = -s;
                *(lds_ptr<u32x4>)(uintptr_t)(Os + buf * BYTES + T::place(row_of(ch), chunk_of(ch))) = __builtin_bit_cast(u32x4, x);
            }
        }
        if (!ROLES || role == 1) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch)
                *(lds_ptr<u32x4>)(uintptr_t)(Qs + buf * BYTES + T::place(row_of(ch), chunk_of(ch))) = __builtin_bit_cast(u32x4, rq[ch]);
        }
        if (tid < QT) Ls[buf][tid] = tid < rows ? log2_of(rl) * lse_factor : -INFINITY;
    };

    const int unit = wave - FIRST;
    const int ct = NB == 2 ? NA * unit : NA * (unit >> 1), half = NB == 2 ? 0 : unit & 1;       // the wave's first columns and rows of dq
    const uint32_t kt16 = Kb + T::tr16_base(lane), st16 = TS::tr16_base(lane);
    auto dq_tile = [&](int t, uint32_t S) {
        if (ct * 16 >= DT || unit < 0) return;
        f32x4 acc[NA][NB];
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < W; ++k) {
            bf16x8 ka[NA], sb[NB];
#pragma unroll
            for (int i = 0; i < NA; ++i) ka[i] = T::tr16_frag(kt16, 32 * k, ct + i);
#pragma unroll
            for (int j = 0; j < NB; ++j) sb[j] = TS::tr16_frag(S + st16, 32 * k, half + j);
#pragma unroll
            for (int i = 0; i < NA; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = XA_MFMA16(ka[i], sb[j], acc[i][j]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int r = t * QT + 16 * (half + j) + (lane & 15);
            if (r >= a.R) continue;
            short *row = a.dq.p + row_offset(a, a.dq, b, hk, r);
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int col = 16 * (ct + i) + 4 * (lane >> 4);
                const f32x4 x = acc[i][j];
                if (col < a.D) *reinterpret_cast<uint2 *>(row + col) = make_uint2(pack_bf16(x[0] * a.scale, x[1] * a.scale), pack_bf16(x[2] * a.scale, x[3] * a.scale));
            }
        }
    };

    int t0, t1;
    share((a.R + QT - 1) / QT, split, SPLIT ? a.splits : 1, t0, t1);
    if (t0 < t1) load(t0 * QT);
    if (LATE && t0 < t1) load_q(t0 * QT);
    const uint32_t Kw = Kb + wave * 32 * T::ROW + row_at, Vw = Vb + wave * 32 * T::ROW + row_at;
    // every key's row, zeros for one that is not valid: what dq adds of its k is 0 x 0
#pragma unroll
    for (int j = 0; j < DT / 16; ++j) {
        const int id = tid + 64 * W * j;
        const uint32_t at = T::place(id / (DT / 8), id % (DT / 8));
        *(lds_ptr<u32x4>)(uintptr_t)(Kb + at) = __builtin_bit_cast(u32x4, kr[j]);
        if (V_IN_LDS) *(lds_ptr<u32x4>)(uintptr_t)(Vb + at) = __builtin_bit_cast(u32x4, vr[j]);
    }
    if (t0 < t1) store(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        if (t + 1 < t1 && !LATE) load(t * QT + QT);
        if (SB == 2 && t > t0) dq_tile(t - 1, Sb + (cur ^ 1) * SBYTES);
        if (wave_live) {
            const uint32_t Qh = Qs + cur * BYTES, Oh = Os + cur * BYTES, Q = Qh + row_at, O = Oh + row_at;
            // the products begin at -lse / scale and -delta.  Register j <-> row (j & 3) + 8 (j >> 2) + 4 hh of the tile; rows behind the last: REPEATED ROWS above
            f32x16 s, p;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&Ls[cur][8 * q + 4 * hh]);
                const f32x4 d4 = *reinterpret_cast<const f32x4 *>(&Ds[cur][8 * q + 4 * hh]);
#pragma unroll
                for (int j = 0; j < 4; ++j) { s[4 * q + j] = l4[j]; p[4 * q + j] = d4[j]; }
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                s = XA_MFMA(lds_16(Q ^ 32 * k), lds_16(Kw ^ 32 * k), s);
                p = XA_MFMA(lds_16(O ^ 32 * k), V_IN_LDS ? lds_16(Vw ^ 32 * k) : vf[k], p);
            }
            reads_ahead<2 * KS, 2, 2>();
            float e[16], d[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                e[j] = __builtin_amdgcn_exp2f(s[j] * c);
                d[j] = e[j] * p[j];
            }
            if (LATE && t + 1 < t1) { load(t * QT + QT); load_q(t * QT + QT); }
            const uint32_t ot = Oh + tr_at, qt = Qh + tr_at;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bf16x8 pb = pack8(e + 8 * k);
                uint4 db = __builtin_bit_cast(uint4, pack8(d + 8 * k));
                if (!all_valid) db = zero_unless(db, valid);          // (P of a key that is not valid may be infinite)
                // rows 16 k + 4 hh .. + 3 and 16 k + 8 + 4 hh .. + 3 of the lane's key
                const uint32_t at = Sb + (SB == 2 ? cur : 0) * SBYTES + 8 * hh;
                *(lds_ptr<u32x2>)(uintptr_t)(at + TS::place(n, 2 * k)) = u32x2{db.x, db.y};
                *(lds_ptr<u32x2>)(uintptr_t)(at + TS::place(n, 2 * k + 1)) = u32x2{db.z, db.w};
#pragma unroll
                for (int q = 0; q < OT; ++q) {
                    dv[q] = XA_MFMA(T::tr_frag(ot, 16 * k, q), pb, dv[q]);
                    dk[q] = XA_MFMA(T::tr_frag(qt, 16 * k, q), __builtin_bit_cast(bf16x8, db), dk[q]);
                }
            }
            reads_ahead<4 * OT, 2, 2>();
        }
        if (LATE && !wave_live && t + 1 < t1) { load(t * QT + QT); load_q(t * QT + QT); }
        if (SB == 1) {
            __syncthreads();
            dq_tile(t, Sb);
        }
        if (t + 1 < t1) store(cur ^ 1);
        __syncthreads();
    }
    if (SB == 2 && t0 < t1) dq_tile(t1 - 1, Sb + ((t1 - 1 - t0) & 1) * SBYTES);
    // a masked key's column holds what its bytes gave: zero goes out for it
    if (!valid) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) { dk[t][j] = 0.0f; dv[t][j] = 0.0f; }
    }
    const bool ok = n < a.Nk;
    if (SPLIT) {
        const long slots = (long)a.groups * a.Nk, slot = (long)g * a.Nk + nc;
        float *pk = a.part + (2 * split * slots + slot) * a.D, *pv = a.part + ((2 * split + 1) * slots + slot) * a.D;
        store_part<DT>(pk, a.D, hh, dk, ok);
        store_part<DT>(pv, a.D, hh, dv, ok);
    } else {
        store_row<DT>(a.dk.p + b * a.dk.sb + hk * a.dk.sh + (long)nc * a.dk.sn, a.D, hh, dk, a.scale, ok);
        store_row<DT>(a.dv.p + b * a.dv.sb + hk * a.dv.sh + (long)nc * a.dv.sn, a.D, hh, dv, 1.0f, ok);
    }
}

// slabs of a split gradient, added in order: KIND 0 dq rows (g R + r), 1 dk and dv keys (2 x (g Nk + n)); four columns a thread
template <int KIND>
__global__ __launch_bounds__(256) void xattn_sum_kernel(Args a, int per_row, unsigned long long row_reciprocal, long total) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const uint32_t row = quotient((uint32_t)id, row_reciprocal);
    const int col = ((uint32_t)id - row * per_row) * 4;
    const long rows = KIND == 0 ? (long)a.groups * a.R : 2L * a.groups * a.Nk;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float4 y = *reinterpret_cast<const float4 *>(a.part + (s * rows + row) * a.D + col);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    short *dst;
    float f = a.scale;
    if (KIND == 0) {
        const int g = row / a.R, b = g / a.Hk;
        dst = a.dq.p + row_offset(a, a.dq, b, g - b * a.Hk, row - (long)g * a.R);
    } else {
        const long key = row < (uint32_t)(a.groups * (long)a.Nk) ? row : row - (long)a.groups * a.Nk;
        const View &t = key == row ? a.dk : a.dv;
        if (key != row) f = 1.0f;
        const int g = (int)(key / a.Nk), b = g / a.Hk;
        dst = t.p + b * t.sb + (g - b * a.Hk) * t.sh + (key - (long)g * a.Nk) * t.sn;
    }
    *reinterpret_cast<uint2 *>(dst + col) = make_uint2(pack_bf16(x.x * f, x.y * f), pack_bf16(x.z * f, x.w * f));
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------

unsigned long long reciprocal_of(long d) { return d <= 1 ? 0 : ~0ull / (unsigned long long)d + 1; }

// blocks of `tile` rows (or keys) for each (sample, kv head)
long tiles_of(long n, int tile) { return (n + tile - 1) / tile; }

// shares of the contracted axis (`steps` tiles long) so that about two blocks run on every CU; a share has at least `least` tiles.  No blocks (an empty batch, no
// queries or no keys): one share
int splits_for(long blocks, long steps, int least) {
    const long want = 2L * num_cus();
    if (blocks < 1 || blocks >= want || steps < 2 * least) return 1;
    return (int)std::max<long>(1, std::min(steps / least, (want + blocks - 1) / blocks));
}

struct Sizes {
    long groups, R;
    int fwd_splits, dq_splits, kv_splits, kv_waves;
    int one_waves;                 // waves of the one-block backward (0: the two kernels)
    bool few_rows;
    size_t fwd_part, fwd_bytes, delta_bytes, bwd_bytes;
};

Sizes sizes_of(int B, int Nq, int Nk, int H, int Hk, int D) {
    Sizes z;
    z.groups = (long)B * Hk;
    z.R = (long)Nq * (H / Hk);
    z.kv_waves = D > 96 ? 8 : 4;
    const long rb = z.groups * tiles_of(z.R, 128), kb = z.groups * tiles_of(Nk, 32 * z.kv_waves);
    z.few_rows = z.R <= 32 && Nk <= 1024;
    z.fwd_splits = z.few_rows ? 1 : splits_for(rb, tiles_of(Nk, 64), 4);
    z.dq_splits = splits_for(rb, tiles_of(Nk, 64), 4);
    z.kv_splits = splits_for(kb, tiles_of(z.R, 32), 8);
    const size_t rows = (size_t)z.groups * z.R;
    z.fwd_part = align_up(z.fwd_splits > 1 ? rows * z.fwd_splits * D * 4 : 0, 256);
    z.fwd_bytes = z.fwd_splits > 1 ? z.fwd_part + rows * z.fwd_splits * 8 : 0;
    z.delta_bytes = align_up(rows * 4, 256);
    // one block for all keys of a (sample, kv head): nine waves fit a CU's LDS and registers up to 64 columns.  Against the two kernels: 128 x 256 rows x 257
    // keys x 12 heads of 64 158 us instead of 203, 128 keys 69 instead of 101, 16 x 500 x 200 x 8 35 instead of 45, 24 x 286 x 93 x 16 heads of 96 over 4 42
    // instead of 60; 64 x 256 x 77 x 16 heads of 128 108 instead of 142, 32 x 256 x 77 x 8 heads of 128 39 instead of 45
    z.one_waves = Nk < 1 || Nq < 1 ? 0 : Nk <= 128 ? 4 : D <= 64 && Nk <= 288 ? 9 : 0;
    if (z.one_waves) {
        // shares of the rows no more than the blocks that two a CU hold (a few over that wait for a second round: at 24 x 286 x 93 58 us instead of 46), of eight tiles at least
        z.kv_splits = (int)std::max<long>(1, std::min(tiles_of(z.R, 32) / 8, 2L * num_cus() / std::max<long>(1, z.groups)));
        z.delta_bytes = 0;
        z.dq_splits = 1;
    }
    const size_t dq = z.dq_splits > 1 ? rows * z.dq_splits * D * 4 : 0, kv = z.kv_splits > 1 ? 2 * (size_t)z.groups * Nk * z.kv_splits * D * 4 : 0;
    z.bwd_bytes = z.delta_bytes + std::max(dq, kv);
    return z;
}

int check_sizes(const char *fn, int B, int Nq, int Nk, int H, int Hk, int D, float scale) {
    if (B < 0 || Nq < 0 || Nk < 0 || H < 1 || Hk < 1) return xq_set_error(XQ_EINVAL, "%s: bad sizes (H=%ld, Hk=%ld)", fn, (long)H, (long)Hk);
    if (H % Hk) return xq_set_error(XQ_EINVAL, "%s: %ld query heads do not share %ld kv heads evenly", fn, (long)H, (long)Hk);
    if (D < 8 || D > 128 || D % 8) return xq_set_error(XQ_EINVAL, "%s: head dim %ld is not a multiple of 8 up to 128", fn, (long)D);
    // (the backward begins its products at lse / scale: that has to stay far from fp32's end)
    if (!(scale >= 0x1p-64f) || !(scale <= 0x1p64f)) return xq_set_error(XQ_EINVAL, "%s: scale has to lie in 2^-64 .. 2^64", fn);
    if ((long)B * Hk * (tiles_of((long)Nq * (H / Hk), 128) + 8) > (1L << 22) || (long)B * Hk * (tiles_of(Nk, 128) + 8) > (1L << 22) ||
        (long)Nq * (H / Hk) > 0x7fffff00L || (long)B * H * Nq > 0x7fffffffL || (long)B * Hk * Nk > 0x3fffffffL)
        return xq_set_error(XQ_EINVAL, "%s: too many rows (%ld) or keys (%ld) for one call", fn, (long)B * H * Nq, (long)B * Hk * Nk);
    return XQ_OK;
}

// reach: heads that a tile of rows passes over (G for a query-sided view, 1 for a key-sided one)
int check_view(const char *fn, const char *what, const void *p, const int64_t *s, int reach) {
    if (s[0] < 0 || s[1] < 0 || s[2] < 0 || s[1] >= (1L << 24) || s[2] >= (1L << 24) || 64 * s[1] + reach * s[2] > (1L << 30)) {
        snprintf(g_err, sizeof(g_err), "%s: token or head stride of %s out of range (64 tokens within 2^30 elements)", fn, what);
        return XQ_EINVAL;
    }
    if (((uintptr_t)p & 15) || s[0] % 8 || s[1] % 8 || s[2] % 8) {
        snprintf(g_err, sizeof(g_err), "%s: %s has to be 16-byte aligned in every row (pointer and strides in multiples of 8 elements)", fn, what);
        return XQ_EINVAL;
    }
    return XQ_OK;
}

View view_of(const void *p, const int64_t *s) { return View{(short *)p, (long)s[0], (long)s[1], (long)s[2]}; }

void plan_blocks(Args &a, long tiles, int splits, unsigned &blocks) {
    a.splits = splits;
    a.nper = (int)(tiles * splits);
    a.swizzle = a.groups % 8 == 0 || a.groups >= 64;
    blocks = (unsigned)((a.swizzle ? (a.groups + 7) / 8 * 8 : a.groups) * (long)a.nper);
}

#define XA_BY_WIDTH(D, CALL)          \
    do {                              \
        if ((D) <= 32) CALL(32);      \
        else if ((D) <= 64) CALL(64); \
        else if ((D) <= 96) CALL(96); \
        else CALL(128);               \
    } while (0)

}  // namespace

extern "C" size_t xq_xattn_forward_workspace_bytes(int B, int Nq, int Nk, int H, int Hk, int D) {
    if (check_sizes("xq_xattn_forward_workspace_bytes", B, Nq, Nk, H, Hk, D, 1.0f)) return 0;
    return sizes_of(B, Nq, Nk, H, Hk, D).fwd_bytes;
}

extern "C" size_t xq_xattn_backward_workspace_bytes(int B, int Nq, int Nk, int H, int Hk, int D) {
    if (check_sizes("xq_xattn_backward_workspace_bytes", B, Nq, Nk, H, Hk, D, 1.0f)) return 0;
    return sizes_of(B, Nq, Nk, H, Hk, D).bwd_bytes;
}

extern "C" int xq_xattn_forward(const void *q, const void *k, const void *v, int B, int Nq, int Nk, int H, int Hk, int D, const int64_t *strides,
                                const void *kv_lens, int lens_i64, const void *key_mask, float scale, void *out, float *lse, void *workspace,
                                size_t workspace_bytes, xq_stream_t stream) {
    const char *fn = "xq_xattn_forward";
    if (int rc = check_sizes(fn, B, Nq, Nk, H, Hk, D, scale)) return rc;
    if (B == 0 || Nq == 0) return XQ_OK;
    if (!q || !out || !strides || (Nk > 0 && (!k || !v))) return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    if (int rc = check_view(fn, "q", q, strides, H / Hk)) return rc;
    if (int rc = check_view(fn, "k", k, strides + 3, 1)) return rc;
    if (int rc = check_view(fn, "v", v, strides + 6, 1)) return rc;
    if ((uintptr_t)out & 15) return xq_set_error(XQ_EINVAL, "%s: out has to be 16-byte aligned", fn);
    const Sizes z = sizes_of(B, Nq, Nk, H, Hk, D);
    if (z.fwd_bytes && (!workspace || workspace_bytes < z.fwd_bytes))
        return xq_set_error(XQ_ENOSPACE, "%s: workspace too small (need %ld bytes, got %ld)", fn, (long)z.fwd_bytes, (long)workspace_bytes);
    hipStream_t s = (hipStream_t)stream;
    Args a = {};
    a.q = view_of(q, strides); a.k = view_of(k, strides + 3); a.v = view_of(v, strides + 6);
    a.out = (short *)out; a.lse = lse;
    a.lens = kv_lens; a.lens_i64 = lens_i64; a.mask = (const unsigned char *)key_mask;
    a.B = B; a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hk = Hk; a.G = H / Hk; a.D = D; a.R = (int)z.R;
    a.g_reciprocal = reciprocal_of(a.G);
    a.scale = scale; a.groups = (int)z.groups;
    a.part = (float *)workspace; a.stat = (float *)((char *)workspace + z.fwd_part);
    unsigned blocks;
    plan_blocks(a, tiles_of(z.R, 128), z.fwd_splits, blocks);
    if (z.few_rows) {
#define XA_CALL(DT) hipLaunchKernelGGL((xattn_few_rows_kernel<DT>), dim3((unsigned)z.groups), dim3(256), 0, s, a)
        XA_BY_WIDTH(D, XA_CALL);
#undef XA_CALL
    } else {
#define XA_CALL(DT)                                                                                                              \
        do {                                                                                                                     \
            if (z.fwd_splits > 1) hipLaunchKernelGGL((xattn_fwd_kernel<DT, true>), dim3(blocks), dim3(256), 0, s, a);            \
            else hipLaunchKernelGGL((xattn_fwd_kernel<DT, false>), dim3(blocks), dim3(256), 0, s, a);                            \
        } while (0)
        XA_BY_WIDTH(D, XA_CALL);
#undef XA_CALL
    }
    if (z.fwd_splits > 1) {
        const long total = z.groups * z.R * (D / 4);
        hipLaunchKernelGGL(xattn_join_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a, D / 4, reciprocal_of(D / 4), total);
    }
    return xq_check_launch(fn);
}

extern "C" int xq_xattn_backward(const void *q, const void *k, const void *v, const void *out, const void *dout, const float *lse, int B, int Nq, int Nk, int H,
                                 int Hk, int D, const int64_t *strides, const void *kv_lens, int lens_i64, const void *key_mask, float scale, void *dq, void *dk,
                                 void *dv, const int64_t *grad_strides, void *workspace, size_t workspace_bytes, xq_stream_t stream) {
    const char *fn = "xq_xattn_backward";
    if (int rc = check_sizes(fn, B, Nq, Nk, H, Hk, D, scale)) return rc;
    if (B == 0 || (Nq == 0 && Nk == 0)) return XQ_OK;
    if (!strides || !grad_strides || (Nq > 0 && (!q || !out || !dout || !lse || !dq)) || (Nk > 0 && (!k || !v || !dk || !dv)))
        return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    const void *in[3] = {q, k, v}, *gr[3] = {dq, dk, dv};
    const char *names[6] = {"q", "k", "v", "dq", "dk", "dv"};
    for (int i = 0; i < 3; ++i) {
        if (int rc = check_view(fn, names[i], in[i], strides + 3 * i, i ? 1 : H / Hk)) return rc;
        if (int rc = check_view(fn, names[3 + i], gr[i], grad_strides + 3 * i, i ? 1 : H / Hk)) return rc;
        const int64_t extent[3] = {B, i ? Nk : Nq, i ? Hk : H};
        for (int j = 0; j < 3; ++j)
            if (extent[j] > 1 && grad_strides[3 * i + j] == 0) {
                snprintf(g_err, sizeof(g_err), "%s: %s has a stride of 0 (several rows in one place)", fn, names[3 + i]);
                return XQ_EINVAL;
            }
    }
    if (((uintptr_t)out | (uintptr_t)dout) & 15) return xq_set_error(XQ_EINVAL, "%s: out and dout have to be 16-byte aligned", fn);
    // (out and dout are read like q: a tile's rows at 32-bit byte offsets)
    if ((Nq > 1 ? 64 * (long)H * D : 0) + (long)(H / Hk) * D > (1L << 30))
        return xq_set_error(XQ_EINVAL, "%s: rows of out and dout are too wide (64 tokens within 2^30 elements: %ld heads of %ld)", fn, (long)H, (long)D);
    const Sizes z = sizes_of(B, Nq, Nk, H, Hk, D);
    if (z.bwd_bytes && (!workspace || workspace_bytes < z.bwd_bytes))
        return xq_set_error(XQ_ENOSPACE, "%s: workspace too small (need %ld bytes, got %ld)", fn, (long)z.bwd_bytes, (long)workspace_bytes);
    hipStream_t s = (hipStream_t)stream;
    Args a = {};
    a.q = view_of(q, strides); a.k = view_of(k, strides + 3); a.v = view_of(v, strides + 6);
    a.dq = view_of(dq, grad_strides); a.dk = view_of(dk, grad_strides + 3); a.dv = view_of(dv, grad_strides + 6);
    a.out_in = (const short *)out; a.dout = (const short *)dout; a.lse = (float *)lse;
    a.lens = kv_lens; a.lens_i64 = lens_i64; a.mask = (const unsigned char *)key_mask;
    a.B = B; a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hk = Hk; a.G = H / Hk; a.D = D; a.R = (int)z.R;
    a.g_reciprocal = reciprocal_of(a.G);
    a.scale = scale; a.groups = (int)z.groups;
    a.delta = (float *)workspace; a.part = (float *)((char *)workspace + z.delta_bytes);
    unsigned blocks;
    if (z.one_waves) {
        plan_blocks(a, 1, z.kv_splits, blocks);
#define XA_GO(DT, W)                                                                                                                  \
    do {                                                                                                                              \
        if (z.kv_splits > 1) hipLaunchKernelGGL((xattn_bwd_kernel<DT, W, true>), dim3(blocks), dim3(64 * W), 0, s, a);                \
        else hipLaunchKernelGGL((xattn_bwd_kernel<DT, W, false>), dim3(blocks), dim3(64 * W), 0, s, a);                               \
    } while (0)
        if (z.one_waves == 9) {
            if (D <= 32) XA_GO(32, 9);
            else XA_GO(64, 9);
        } else {
#define XA_CALL(DT) XA_GO(DT, 4)
            XA_BY_WIDTH(D, XA_CALL);
#undef XA_CALL
        }
#undef XA_GO
    }
    if (Nq > 0 && !z.one_waves) {
        plan_blocks(a, tiles_of(z.R, 128), z.dq_splits, blocks);
        if (z.dq_splits > 1) {
#define XA_CALL(DT) hipLaunchKernelGGL((xattn_dq_kernel<DT, true>), dim3(blocks), dim3(256), 0, s, a)
            XA_BY_WIDTH(D, XA_CALL);
#undef XA_CALL
            const long total = z.groups * z.R * (D / 4);
            hipLaunchKernelGGL((xattn_sum_kernel<0>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a, D / 4, reciprocal_of(D / 4), total);
        } else {
#define XA_CALL(DT) hipLaunchKernelGGL((xattn_dq_kernel<DT, false>), dim3(blocks), dim3(256), 0, s, a)
            XA_BY_WIDTH(D, XA_CALL);
#undef XA_CALL
        }
    }
    if (Nk > 0 && !z.one_waves) {
        plan_blocks(a, tiles_of(Nk, 32 * z.kv_waves), z.kv_splits, blocks);
#define XA_GO(DT, W)                                                                                                                  \
    do {                                                                                                                              \
        if (z.kv_splits > 1) hipLaunchKernelGGL((xattn_dkdv_kernel<DT, W, true>), dim3(blocks), dim3(64 * W), 0, s, a);               \
        else hipLaunchKernelGGL((xattn_dkdv_kernel<DT, W, false>), dim3(blocks), dim3(64 * W), 0, s, a);                              \
    } while (0)
        if (D <= 32) XA_GO(32, 4);
        else if (D <= 64) XA_GO(64, 4);
        else if (D <= 96) XA_GO(96, 4);
        else XA_GO(128, 8);
#undef XA_GO
    }
    if (Nk > 0 && z.kv_splits > 1) {
        const long total = 2 * z.groups * (long)Nk * (D / 4);
        hipLaunchKernelGGL((xattn_sum_kernel<1>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a, D / 4, reciprocal_of(D / 4), total);
    }
    return xq_check_launch(fn);
}
