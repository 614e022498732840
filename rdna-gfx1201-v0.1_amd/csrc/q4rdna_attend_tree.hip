// Attention of drafted tokens over the 8-bit paged cache and over each other
// (q4rdna_kv_attend_tree): attend_tree_kernel.
//
// A wave takes 32 rows (query token, query head of one kv head), a lane each,
// and walks blocks of 64 cached tokens as attend_many_kernel does: S^T = K q^T,
// a softmax in the lane, O^T += V^T p^T, by 32x32x16 fp16 matrix instructions
// (q4rdna_rows_device.h).  There are few rows and no time to share: the codes go
// from memory into the wave's registers and become fp16 there, since
//  * the 16 bytes that a lane loads of K are 16 numbers of one token, two
//    operands' worth when q has its numbers in the same order;
//  * the 16 bytes that it loads of V are 16 tokens of one number, the tokens
//    whose scores the lane holds after the first product.
// A workgroup has one tile of 32 rows, and its four waves every fourth block of
// it: no wave waits for another before the end, when their parts meet in LDS.
// (Tiles of 128 rows, a wave per 32, read each block once rather than once a
// tile, but left three waves idle where rows are few or odd, and parts four times
// as large to join: an eighth slower for 32 sequences of 100 .. 8000 tokens, 1 .. 24
// drafts, 8 kv heads of 4 by 128.  The second read is the L2's.)
//
// The open block and the drafted tokens are cut into halves of 32, one for a wave
// at most (as whole blocks 4 drafts after 33 tokens take 1.5 us more).  The workgroup
// lays the drafts' rows into LDS in fp16, scaled by a power of two for each token,
// fp32 ones in two parts: four tokens a thread, or one where they are few (1.2 us
// less for these).  A row's mask is 64 bits.
//
// What is rounded: fp32 q, k and v to two fp16 parts, weights of all types to two
// (2^-22 of each); fp16 and bf16 rows and the cache's codes are exact in one.  (One
// part of the weights and K's codes with a bias, 8% faster for the 32 sequences in
// bf16, put fp16 results further off than their own rounding, and scores off by
// 2^-14 of a block's scale times sum |q|.)
//
// A tile's blocks are split over workgroups, dealt on the device by the
// sequences' lengths, and joined in a fixed order by a second kernel.
//
// What bounds it, for the 32 sequences above (118 MB of codes, 150 MB read, 2.6
// TB/s) in bf16: nothing alone.  A block of 64 tokens takes a wave some 500 vector
// instructions (16384 codes into fp16, 2048 weights) and 48 matrix ones; with the
// workgroups' start, drafts and joining, 44% of all vector instructions, the vector
// unit is busy 47% of the time and the matrix unit 20%.  A SIMD has 1.4 waves on
// average of the two that fit, since parts end unevenly, and these wait 28% of their
// time for data and as long for their turn.  For one sequence it is the chain of
// dependent loads and the first fetch of the code.
// Eight kv heads of 4 by 128: fp32, 4 drafts after 33 tokens 9.6 us; 16 drafts
// after 4001 15.4 us and 3.9 us the joining; the 32 sequences in bf16 56.8 us and
// 4.8 us, in fp32 66.9 and 5.4 (with one workgroup a CU a fifth more; two leave
// registers for all but eight, and cost a few tokens' call 1%).
#include <type_traits>

#include "q4rdna_rows_device.h"

namespace q4rdna {
namespace {

constexpr int kWaves = 4, kTreeThreads = 64 * kWaves;
constexpr int kBlock = static_cast<int>(kKvBlock);

template <int D>
struct TreeTile {
    _Float16 k[kKvBlock * (D + 8)];  // rows of 272 (144) bytes: 16 lanes' 16-byte reads of 16 rows cover all banks once
    _Float16 v[D * kKvBlock];        // V^T, see v_place
};
// Place of a row of V^T's numbers `at` and on (of 64, in the order of the lanes'
// scores): its 16-byte pieces are turned by the row, so that 16 rows side by side
// (the products') and 16 rows of every eighth (the staging's) lie in all banks.
__device__ __forceinline__ int v_place(int row, int at) { return row * kBlock + (((at >> 3) ^ ((row >> 3) + row)) & 7) * 8 + (at & 7); }
template <int D, int SPLIT>
struct TreeStage {
    TreeTile<D> part[SPLIT];
    float scales[2 * kKvBlock];  // K's, V's
};
// Parts of one row joined: its maximum m, the accumulators' exponent e (a whole
// number) and its sum l, in units of 2^(m - 7).
struct Joined {
    float m, l, e;
};
template <int D>
struct TreeJoin {
    float o[kWaves][32][D + 4];
    float m[kWaves][32], l[kWaves][32], e[kWaves][32];
    Joined joined[32];
};

// K or V of a block as it lies in memory, 16 bytes of a lane each: of K
// [32 tokens][32 numbers], of V [32 numbers][tokens with bit 3 clear, set].
template <int D>
struct TreeRaw {
    i32x4 x[D / 16];
};
// (Buffer loads: their base is in scalar registers, so that all of them share
// one vector register of offsets and need no vector instruction.)
struct Tile {
    __amdgpu_buffer_rsrc_t at;
};
__device__ __forceinline__ Tile tile_at(const int8_t *p, uint32_t bytes) {
    return Tile{__builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p), 0, static_cast<int>(bytes), 0x00020000)};
}
// 16 (8) bytes of a lane, `at` + c on, c a constant.
__device__ __forceinline__ i32x4 load_piece(const Tile &tile, uint32_t at, uint32_t c) {
    return __builtin_amdgcn_raw_buffer_load_b128(tile.at, at, c, 0);
}
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ i32x2 load_half_piece(const Tile &tile, uint32_t at, uint32_t c) {
    return __builtin_amdgcn_raw_buffer_load_b64(tile.at, at, c, 0);
}
template <int D>
__device__ __forceinline__ void load_k(TreeRaw<D> &r, const Tile &tile) {
    const uint32_t lane = threadIdx.x & 63, at = (lane & 31) / 16 * (D / 64 * 1024) + (lane >> 5) * 256 + (lane & 15) * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) r.x[t * (D / 32) + x] = load_piece(tile, at, t * (D / 64 * 2048) + x / 2 * 1024 + x % 2 * 512);
}
template <int D>
__device__ __forceinline__ void load_v(TreeRaw<D> &r, const Tile &tile) {
    const uint32_t lane = threadIdx.x & 63, at = (lane & 31) / 16 * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int y = 0; y < 2; ++y) r.x[d * 2 + y] = load_piece(tile, at, kBlock * D + d * 2048 + y * 512);
}
// Of the open block's half `which`: K's planes of high and low bytes one behind the
// other, and of V's eight tokens of each of the two in one piece.
template <int D>
__device__ __forceinline__ void load_open_k(TreeRaw<D> &r, const Tile &planes, uint32_t which) {
    const uint32_t lane = threadIdx.x & 63, at = (lane & 31) / 16 * (D / 64 * 1024) + (lane >> 5) * 256 + (lane & 15) * 16 + which * (D / 64 * 2048);
#pragma unroll
    for (int low = 0; low < 2; ++low)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) r.x[low * (D / 32) + x] = load_piece(planes, at, low * (kBlock * D) + x / 2 * 1024 + x % 2 * 512);
}
template <int D>
__device__ __forceinline__ void load_open_v(TreeRaw<D> &r, const Tile &planes, uint32_t which) {
    const uint32_t lane = threadIdx.x & 63, at = (lane & 31) / 16 * 1024 + (lane >> 5) * 256 + (lane & 15) * 16 + 8 * which;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const i32x2 high = load_half_piece(planes, at, 2 * kBlock * D + d * 2048 + y * 512);
            const i32x2 low = load_half_piece(planes, at, 3 * kBlock * D + d * 2048 + y * 512);
            r.x[d * 2 + y] = i32x4{high[0], high[1], low[0], low[1]};
        }
}
// Half of 16 codes as fp16, times 2^-8 where they are low bytes.
template <bool LOW>
__device__ __forceinline__ h16x8 half_piece(i32x4 piece, int half) {
    h16x2 x[4];
    codes_to_half(static_cast<uint32_t>(piece[2 * half]), x[0], x[1]);
    codes_to_half(static_cast<uint32_t>(piece[2 * half + 1]), x[2], x[3]);
    if (LOW) {
        const h16x2 f = {static_cast<_Float16>(0x1p-8f), static_cast<_Float16>(0x1p-8f)};
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] *= f;
    }
    h16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e / 2][e % 2];
    return r;
}

// s[t] += the products of K's fragments (32 tokens t, 16 numbers f) with the rows.
template <int N, int D, int SPLIT, typename K>
__device__ __forceinline__ void add_scores(const ManyState<D, SPLIT> &st, f32x16 (&s)[N], K fragment) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int f = 0; f < D / 16; ++f) {
            const h16x8 k = fragment(t, f);
#pragma unroll
            for (int x = 0; x < SPLIT; ++x) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, st.q[f][x], s[t], 0, 0, 0);
        }
    }
}
// o += the products of V's fragments (32 numbers d; tokens 16 a + 8 y + 4 half + b,
// a = 2 t, 2 t + 1) with the weights, which are held in two fp16 parts whatever the
// type of the queries: 22 bits of each.  (In 11 bits an fp16 row was further off
// by its weights than by its own rounding.)
template <int N, int D, int SPLIT, typename V>
__device__ __forceinline__ void add_rows(ManyState<D, SPLIT> &st, const f32x16 (&s)[N], V fragment) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            float minus = -1.0f;
            asm("" : "+s"(minus));  // (a product, so that one instruction takes a half as it is)
            h16x8 p[2];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const int at = 4 * (2 * (e / 4) + y) + e % 4;
                const f32x2 w = {s[t][at], s[t][at + 1]};
                h16x2 high = __builtin_convertvector(w, h16x2);
                asm("" : "+v"(high));  // or each would be converted once more by itself
                const f32x2 rest = {fmaf(static_cast<float>(high[0]), minus, w[0]), fmaf(static_cast<float>(high[1]), minus, w[1])};
                const h16x2 low = __builtin_convertvector(rest, h16x2);
                p[0][e] = high[0];
                p[0][e + 1] = high[1];
                p[1][e] = low[0];
                p[1][e + 1] = low[1];
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const h16x8 v = fragment(d, y, t);
#pragma unroll
                for (int x = 0; x < 2; ++x) st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[x], st.o[d], 0, 0, 0);
            }
        }
    }
}
template <int N>
__device__ __forceinline__ void clear(f32x16 (&s)[N]) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
}
// All ones where bit i is set.  (As an instruction of its own: the compiler would
// make a compare of it, and 32 of them would each hold a pair of scalar registers.)
__device__ __forceinline__ uint32_t bit_ones(uint32_t bits, int i) { return static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), i, 1)); }
// `instead` where a bit is clear.
template <int N>
__device__ __forceinline__ void hide(f32x16 (&s)[N], uint32_t seen, float instead) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t m = bit_ones(seen, 16 * t + i);
            s[t][i] = __uint_as_float((__float_as_uint(s[t][i]) & m) | (__float_as_uint(instead) & ~m));
        }
}
// The largest and the sum of the lane's numbers, four chains of them side by side.
template <int N>
__device__ __forceinline__ float largest(const f32x16 (&s)[N]) {
    float top[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) top[x] = s[x * N / 4][4 * N * x % 16];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int i = 1; i < 4 * N; ++i) top[x] = fmaxf(top[x], s[x * N / 4][4 * N * x % 16 + i]);
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
template <int N>
__device__ __forceinline__ float total(const f32x16 (&s)[N]) {
    float sum[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) sum[x] = s[x * N / 4][4 * N * x % 16];
#pragma unroll
    for (int i = 1; i < 4 * N; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[x] += s[x * N / 4][4 * N * x % 16 + i];
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
// s * unit - m, the product rounded first: a score that is the reference becomes
// zero, however large both are.
template <int N>
__device__ __forceinline__ void subtract(f32x16 (&s)[N], float unit, float m) {
#pragma clang fp contract(off)
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = s[t][i] * unit - m;
}
// Scores to weights: s = 2^(s * unit + shift), zero where hidden; their sum.
template <int N>
__device__ __forceinline__ float exponentials(f32x16 (&s)[N], float unit, float shift, uint32_t seen, bool masked) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], unit, shift));
    if (masked) hide(s, seen, 0.0f);
    return total(s);
}

// From scores of this size on (base 2) fp32 has steps that a weight would show.
constexpr float kFar = 0x1p16f;
// refer() for a weight times V of 2^(base + rel), which is not added up: the steps
// of a large score are larger than rel.
template <int D, int SPLIT>
__device__ __forceinline__ void refer(ManyState<D, SPLIT> &st, float now, float base, float rel) {
    const bool grown = now > st.m + kLazy, more = (base - st.m) + rel > st.e + kLazy;
    if (__builtin_amdgcn_ballot_w64(grown || more) == 0) return;
    if (!(grown || more)) return;
    const float m = grown ? now : st.m, most = fmaxf((st.m - m) + st.e, (base - m) + rel);
    const float e = most == kNegInf ? kNegInf : ceilf(most);
    st.l *= __builtin_amdgcn_exp2f(st.m - m);  // 0 from -inf
    const float f = st.e == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((st.m - m) + (st.e - e));  // (o is zero there)
#pragma unroll
    for (int d = 0; d < D / 32; ++d) st.o[d] *= f;
    st.m = m;
    st.e = e;
}

// The softmax of a full block: integer products to weights in the accumulators'
// units, V's scale among them.
template <int D, int SPLIT>
__device__ __forceinline__ void soften_block(ManyState<D, SPLIT> &st, f32x16 (&s)[2], float k_scale, float v_scale, uint32_t seen,
                                             bool masked) {
    if (masked) hide(s, seen, kNegInf);
    const float unit = st.q_scale * k_scale, top = max_xor32(largest(s));
    const bool none = top == kNegInf;
    const float now = none ? kNegInf : top * unit;
    // The block's scale of V, 2^(v_exp + v_log), goes into the exponent, and comes out of the sum.
    const bool finite = v_scale < __builtin_inff();
    const float v_exp = static_cast<float>(__builtin_amdgcn_frexp_expf(v_scale));
    const float v_log = finite ? __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v_scale)) : __builtin_nanf("");
    refer(st, now, now, v_exp + v_log);
    const float ratio = none ? 0.0f : finite ? fmaxf(v_log + (v_exp - st.e), kLeast) : __builtin_nanf("");
    const float m = st.m == kNegInf ? 0.0f : st.m;
    float times = unit, shift = kWeight - m + ratio;
    if (__builtin_expect(!none && __builtin_fabsf(now) > kFar, 0)) {
        subtract(s, unit, m);
        times = 1.0f;
        shift = kWeight + ratio;
    }
    const float sum = exponentials(s, times, shift, seen, masked);
    st.l += sum * __builtin_amdgcn_exp2f(-ratio);
}
// The same of 32 tokens with a scale each, K's and 64 further on V's, the lane's
// own four at a time; `unit_log` is 8 for 16-bit codes, whose tiles are in units
// of 256 times the scales.
template <int D, int SPLIT>
__device__ __forceinline__ void soften_tokens(ManyState<D, SPLIT> &st, f32x16 (&s)[1], int unit_log, uint32_t seen, const float *scales) {
    // A token's scale and the row's by their exponents together: either alone may
    // take the products out of fp32's range where the score is within it.
    const float unit = 2.0f * __builtin_amdgcn_frexp_mantf(st.q_scale);
    const int q_exp = st.q_scale == 0.0f ? -400 : __builtin_amdgcn_frexp_expf(st.q_scale) - 1 + unit_log;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const f32x4 kt = *reinterpret_cast<const f32x4 *>(scales + 8 * x);
#pragma unroll
        for (int b = 0; b < 4; ++b)
            s[0][4 * x + b] = __builtin_amdgcn_ldexpf(s[0][4 * x + b] * __builtin_amdgcn_frexp_mantf(kt[b]), __builtin_amdgcn_frexp_expf(kt[b]) + q_exp);
    }
    hide(s, seen, kNegInf);
    const float top = max_xor32(largest(s));
    const float now = top == kNegInf ? kNegInf : top * unit;
    // Weights of 2^8 at most times the scales, under 2^122, in fp32; the largest
    // of them is what the row refers to.
    const float m = now > st.m + kLazy ? now : st.m;
    subtract(s, unit, m == kNegInf ? 0.0f : m);
    const float sum = exponentials(s, 1.0f, 0.0f, seen, true);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const f32x4 vt = *reinterpret_cast<const f32x4 *>(scales + kBlock + 8 * x);
#pragma unroll
        for (int b = 0; b < 4; ++b) s[0][4 * x + b] *= vt[b] + (vt[b] - vt[b]);  // an infinite scale is made NaN
    }
    hide(s, seen, 0.0f);
    refer(st, now, m, __builtin_amdgcn_logf(max_xor32(fmaxf(largest(s), 0.0f))) + static_cast<float>(unit_log));
    st.l += __builtin_amdgcn_ldexpf(sum, static_cast<int>(kWeight));
    // From units of 2^(m + unit_log) to the accumulators'.
    const int up = st.e == kNegInf ? 0 : unit_log + static_cast<int>(kWeight) - static_cast<int>(st.e);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = __builtin_amdgcn_ldexpf(s[0][i], up);
}

// Numbers as they lie in memory, N side by side at any alignment: they become
// floats where they are used, since a conversion waits for them.
template <typename T, int N>
struct Numbers {
    typedef T TN __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    TN v;
};
template <typename T, int N>
__device__ __forceinline__ void load_numbers(Numbers<T, N> &x, const T *p) {
    typedef __attribute__((address_space(1))) const typename Numbers<T, N>::TN *gptr;
    x.v = *(gptr)(uintptr_t)p;
}
template <typename T>
using Eight = Numbers<T, 8>;

// Rows of q, the numbers of a fragment f in the order in which K's pieces have
// them: 64 (f / 4) + 32 (f / 2 % 2) + 16 half + 8 (f % 2) and on.
__device__ __forceinline__ int fragment_number(int f, int half) { return f / 4 * 64 + f / 2 % 2 * 32 + 16 * half + f % 2 * 8; }
template <int D, typename T>
__device__ __forceinline__ void load_query(Eight<T> (&x)[D / 16], const T *row) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int f = 0; f < D / 16; ++f) load_numbers(x[f], row + fragment_number(f, half));
}
template <int D, int SPLIT, typename T>
__device__ __forceinline__ void set_query(ManyState<D, SPLIT> &st, const Eight<T> (&raw)[D / 16], float scale) {
    float x[D / 16][8];
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[f][e] = static_cast<float>(raw[f].v[e]);
    uint32_t top = 0;
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[f][e]) & 0x7fffffffu);
    top = __float_as_uint(max_xor32(__uint_as_float(min(top, 0x7f800000u))));  // NaN as infinity
    const bool finite = top < 0x7f800000u;
    // The largest number of the row to 2^13 .. 2^14: small ones stay normal in fp16.
    const int up = finite && top != 0 ? 14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = finite ? __builtin_amdgcn_ldexpf(x[f][e], up) : 0.0f;
            st.q[f][0][e] = static_cast<_Float16>(v);
            if (SPLIT == 2) st.q[f][SPLIT - 1][e] = static_cast<_Float16>(v - static_cast<float>(st.q[f][0][e]));
        }
    st.q_scale = finite ? __builtin_amdgcn_ldexpf(scale * kLog2e, -up) : __builtin_nanf("");
    st.m = kNegInf;
    st.l = 0.0f;
    st.e = kNegInf;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[d][i] = 0.0f;
}

// The drafted tokens' K and V into LDS: a thread takes eight numbers of B tokens,
// D / 8 threads side by side a row: of four (of 64 numbers two), or, where there
// are few, of one.
template <int D, typename T, int B>
struct DraftRows {
    static constexpr int kOctets = D / 8;
    static constexpr int kTokens = B * kTreeThreads / kOctets;
    Eight<T> raw[2][B];
    __device__ __forceinline__ static int octet() { return threadIdx.x % kOctets; }
    __device__ __forceinline__ static int token() { return threadIdx.x / kOctets * B; }  // the first
};
template <int D, typename T, int B>
__device__ __forceinline__ void load_drafts(DraftRows<D, T, B> &r, const TreeArgs &a, int first, int count, uint32_t head) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const q4rdna_kv_rows &rows = which == 0 ? a.d.k : a.d.v;
#pragma unroll
        for (int b = 0; b < B; ++b) {
            // (Tokens behind the last one are that one, and seen by nobody.)
            load_numbers(r.raw[which][b], static_cast<const T *>(rows.data) + static_cast<int64_t>(first + min(r.token() + b, count - 1)) * rows.token_stride +
                                              head * rows.head_stride + 8 * r.octet());
        }
    }
}
template <int D, int SPLIT, typename T, int B>
__device__ __forceinline__ void stage_drafts(TreeStage<D, SPLIT> &stage, const DraftRows<D, T, B> &r) {
    const int octet = r.octet(), token = r.token();
    float x[2][B][8];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[which][b][e] = static_cast<float>(r.raw[which][b].v[e]);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[which][b][e]) & 0x7fffffffu);
            top = lanes_max<DraftRows<D, T, B>::kOctets>(top);
            const bool finite = top < 0x7f800000u;
            // The largest to 2^13 .. 2^14, but for numbers under 2^-96: the scale stays a normal number.
            const int up = finite && top != 0 ? min(14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)), 110) : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[which][b][e] = finite ? __builtin_amdgcn_ldexpf(x[which][b][e], up) : 0.0f;
            if (octet == 0) stage.scales[which * kBlock + token + b] = finite ? __builtin_amdgcn_ldexpf(1.0f, -up) : __builtin_nanf("");
        }
    typedef _Float16 Tokens __attribute__((ext_vector_type(B)));
    typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int part = 0; part < SPLIT; ++part) {
        TreeTile<D> &tile = stage.part[part];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            h16x8 k;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[e] = static_cast<_Float16>(x[0][b][e]);
                x[0][b][e] -= static_cast<float>(k[e]);
            }
            *reinterpret_cast<h16x8 *>(tile.k + (token + b) * (D + 8) + 8 * octet) = k;
        }
        // Row d of V: the tokens in the order of the lanes' scores.
        const int quad = token / 4, at = (quad & 1) * 32 + (quad >> 1 & 1) * 16 + (quad >> 2) * 4 + token % 4;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            Tokens v;
#pragma unroll
            for (int b = 0; b < B; ++b) {
                v[b] = static_cast<_Float16>(x[1][b][e]);
                x[1][b][e] -= static_cast<float>(v[b]);
            }
            *reinterpret_cast<Tokens *>(tile.v + v_place(8 * octet + e, at)) = v;
        }
        // The other tokens of the first 32 are zeros (of weight zero; K's are hidden).
        if constexpr (DraftRows<D, T, B>::kTokens == 16) {
#pragma unroll
            for (int i = threadIdx.x; i < 4 * D; i += kTreeThreads)
                *reinterpret_cast<h16x4 *>(tile.v + v_place(i / 4, i % 4 * 16 + 4)) = h16x4{};
        }
    }
}

// One sequence of a step: as seq_of, but its tokens are not in the cache.
__device__ __forceinline__ Seq draft_seq(const TreeArgs &a, uint32_t i) {
    Seq s;
    // (Loads without branches: what is not there is read from past.)
    const bool starts = a.batch.cu_tokens != nullptr, slots = a.batch.slots != nullptr;
    const int32_t *from = starts ? a.batch.cu_tokens : a.batch.past;
    const int first = from[i], last = from[starts ? i + 1 : i], slot = (slots ? a.batch.slots : a.batch.past)[i];
    s.past = a.batch.past[i];
    s.first = starts ? first : static_cast<int>(i);
    const int end = starts ? last : static_cast<int>(i) + 1;
    s.slot = slots ? slot : static_cast<int>(i);
    s.ok = s.first >= 0 && end >= s.first && static_cast<uint32_t>(end) <= a.batch.tokens;
    s.count = s.ok ? end - s.first : 0;
    const int64_t room = static_cast<int64_t>(a.batch.table_width) * kBlock;
    s.ok = s.ok && static_cast<uint32_t>(s.count) <= a.batch.max_tokens && s.past >= 0 && s.past <= room &&
           static_cast<uint32_t>(s.slot) < a.cache.slot_count;
    s.length = s.past;
    return s;
}
// The cached blocks that any row sees: no row stands before past - 1.
__device__ __forceinline__ int first_block(const TreeArgs &a, int past) {
    return a.d.window != 0 && static_cast<uint32_t>(past) > a.d.window ? (past - static_cast<int>(a.d.window)) / kBlock : 0;
}

// What a sequence's workgroups take: each tile of 32 rows of each head is cut into
// parts of about `chunk` of its units: full blocks of the cache, 32 tokens of the
// open one, 32 drafts.
struct TreeWork {
    Seq s;
    uint32_t jobs, units;
};
__device__ __forceinline__ TreeWork tree_work(const TreeArgs &a, uint32_t i) {
    TreeWork w;
    w.jobs = w.units = 0;
    w.s = draft_seq(a, min(i, a.batch.sequences - 1));
    if (i >= a.batch.sequences || !w.s.ok || w.s.count == 0) return w;
    w.jobs = (w.s.count * a.group + kTreeRows - 1) / kTreeRows * a.cache.kv_heads;
    w.units = w.s.past / kBlock - first_block(a, w.s.past) + (w.s.past % kBlock + 31) / 32 + (w.s.count + 31) / 32;
    return w;
}
// (A part has a unit for every wave.)
__device__ __forceinline__ uint32_t tree_parts(const TreeArgs &a, const TreeWork &w, uint32_t chunk) {
    chunk = max(chunk, static_cast<uint32_t>(kWaves));
    return min((w.units + chunk - 1) / chunk, a.splits);
}

struct TreeItem {
    int seq;  // -1: nothing
    Seq s;
    uint32_t head, tile;
    int split, splits;
    uint32_t first;  // workgroup of part 0; part i is kv_heads * i further on
};
// The item of workgroup x: the device knows the lengths, the host does not, so
// every wave adds up the sequences' parts, 64 at a time.
__device__ __forceinline__ TreeItem find_tree_item(const TreeArgs &a) {
    const uint32_t x = blockIdx.x;
    TreeItem it;
    it.seq = -1;
    const int lane = threadIdx.x & 63;
    const uint32_t heads = a.cache.kv_heads;
    if (a.splits == 1) {  // as many workgroups as there may be tiles
        it.seq = static_cast<int>(blockIdx.z);
        it.s = draft_seq(a, blockIdx.z);
        it.tile = x;
        it.head = blockIdx.y;
        it.split = 0;
        it.splits = 1;
        it.first = x;
        return it;
    }
    TreeWork w;
    uint32_t all = 0, jobs = 0;  // jobs * units, fewer than 2^32 by the host's bound
    for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
        w = tree_work(a, i + lane);
        all += __builtin_amdgcn_readlane(wave_scan(w.jobs * w.units), 63);
        jobs += __builtin_amdgcn_readlane(wave_scan(w.jobs), 63);
    }
    // A part for a CU, or fewer and larger ones, so that all of them run at once.
    // Where there are as many tiles as CUs and eight units a wave, two for a CU,
    // which share it well, and as large as it takes for the long ones to run at
    // once: a second round costs a whole part's time, while short ones fill the
    // gaps.  (The host has launched workgroups for as many.)  (48 sequences of 100 .. 4000 tokens 58.7 and 48.9 us, 24 of up to 12000 by
    // 64 33.3 and 29.3; but one of 60000 39.1 and 44.8.)
    uint32_t chunk = (max(all, 1u) - 1) / a.cus + 1;
    const bool two = jobs >= a.cus && chunk >= 8 * kWaves;
    if (two) chunk = (all - 1) / (2 * a.cus) + 1;
    if (a.batch.sequences <= 64 && (two || jobs < a.cus))
        for (int i = 0; i < 12; ++i) {
            const float parts = ceilf(static_cast<float>(w.units) * __builtin_amdgcn_rcpf(static_cast<float>(max(chunk, static_cast<uint32_t>(kWaves)))));
            const uint32_t n = !two || 2 * w.units > chunk ? w.jobs * static_cast<uint32_t>(parts) : 0;
            if (static_cast<uint32_t>(__builtin_amdgcn_readlane(wave_scan(n), 63)) <= (two ? 2 * a.cus : a.cus)) break;
            chunk += chunk / 8 + 1;
        }
    // Long parts first: those of more than half a chunk, then the others.
    uint32_t base = 0;
    for (int small = 0; small < 2; ++small)
        for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
            if (a.batch.sequences > 64) w = tree_work(a, i + lane);
            const uint32_t parts = tree_parts(a, w, chunk), mine = (two && 2 * w.units <= chunk) == (small != 0) ? w.jobs * parts : 0;
            const uint32_t end = base + wave_scan(mine);
            const uint64_t later = __builtin_amdgcn_ballot_w64(end > x);
            if (later != 0) {
                const int owner = __builtin_ctzll(later);
                const uint32_t its = __builtin_amdgcn_readlane(parts, owner);
                const uint32_t local = x - __builtin_amdgcn_readlane(end - mine, owner);  // (tile, part, head)
                it.seq = static_cast<int>(i) + owner;
                it.s.first = __builtin_amdgcn_readlane(w.s.first, owner);
                it.s.count = __builtin_amdgcn_readlane(w.s.count, owner);
                it.s.past = __builtin_amdgcn_readlane(w.s.past, owner);
                it.s.slot = __builtin_amdgcn_readlane(w.s.slot, owner);
                it.s.length = it.s.past;
                it.s.ok = true;
                it.head = local % heads;
                it.split = static_cast<int>(local / heads % its);
                it.tile = local / heads / its;
                it.splits = static_cast<int>(its);
                it.first = x - it.split * heads;
                return it;
            }
            base = __builtin_amdgcn_readlane(end, 63);
        }
    return it;
}

// A part's e where the row's maximum is `ref`, and its factor in the row's unit e.
// (A part without e is zero, or NaN.)
__device__ __forceinline__ float shifted_unit(float ref, float m, float e) { return e == kNegInf ? kNegInf : ceilf((m - ref) + e); }
__device__ __forceinline__ float part_factor(float ref, float row_e, float m, float e) {
    return e == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((m - ref) + (e - row_e));
}

// row / group.  (A row is below 64 * 2^15 and the group up to 2^15: div_split may
// be one too many.)
__device__ __forceinline__ int token_of(const TreeArgs &a, int row) {
    const uint32_t t = div_split(row, a.group, a.group_magic);
    return static_cast<int>(t * a.group > static_cast<uint32_t>(row) ? t - 1 : t);
}

// Four numbers of a row.
template <typename T>
__device__ __forceinline__ void write_row(const TreeArgs &a, const Seq &s, uint32_t head, int row, int d, const Joined &w, f32x4 o) {
    const int token = token_of(a, row), n = s.first + token;
    const uint32_t to_head = head * a.group + (row - token * a.group);
    const float inv = w.l == 0.0f ? 0.0f : 1.0f / w.l;
    const int places = static_cast<int>(fminf(fmaxf(w.e, -400.0f), 400.0f));
    typedef __attribute__((address_space(1))) typename Numbers<T, 4>::TN *gptr;
    typename Numbers<T, 4>::TN v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(__builtin_amdgcn_ldexpf(o[e] * inv, places));
    *(gptr)(uintptr_t)(static_cast<T *>(a.d.out.data) + static_cast<int64_t>(n) * a.d.out.token_stride + to_head * a.d.out.head_stride + d) = v;
    if (d == 0 && a.d.lse != nullptr)
        a.d.lse[static_cast<size_t>(n) * a.d.q_heads + to_head] = (w.m + log2f(w.l) - kWeight) * (1.0f / kLog2e);
}

// The parts' results of workgroup x: [row][D], and behind all of these [m, l, e][row].
template <int D>
__device__ __forceinline__ float *part_rows(const TreeArgs &a, uint32_t x) { return a.partials + static_cast<size_t>(x) * kTreeRows * D; }
template <int D>
__device__ __forceinline__ float *part_stats(const TreeArgs &a, uint32_t x) {
    return a.partials + static_cast<size_t>(a.workgroups) * kTreeRows * D + static_cast<size_t>(x) * kTreeRows * 3;
}

template <int D, int SPLIT, typename T, bool WINDOW, int PER_CU>
__global__ __launch_bounds__(kTreeThreads, PER_CU) void attend_tree_kernel(const TreeArgs a) {
    __shared__ __align__(16) union Shared {
        TreeStage<D, SPLIT> stage;
        TreeJoin<D> join;
    } shared;
    __shared__ __align__(16) float open_scales[kWaves][2 * kBlock];
    const int tid = threadIdx.x, lane = tid & 63, column = lane & 31, half = lane >> 5, wave = wave_id();
    const TreeItem it = find_tree_item(a);
    // (What is rare is told apart: its code goes behind the rest, which is fetched in order.)
    if (__builtin_expect(wave == kWaves - 1 && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1, 0))
        for (uint32_t i = lane; i < a.batch.sequences; i += 64)  // bad entries, once
            if (!draft_seq(a, i).ok) count_fault(a.cache);
    if (it.seq < 0 || !it.s.ok) return;
    const uint32_t head = it.head;
    const Seq &s = it.s;
    const int group = static_cast<int>(a.group), rows = s.count * group;
    const int first_row = static_cast<int>(it.tile * kTreeRows);
    if (first_row >= rows) return;
    const int live_rows = min(static_cast<int>(kTreeRows), rows - first_row);
    // Units: full blocks from block0 on, the halves of the open one, those of the
    // drafts.  These four go to different waves.
    const int block0 = first_block(a, s.past), full_blocks = s.past / kBlock;
    const int opens = full_blocks, drafts = opens + (s.past % kBlock + 31) / 32, units = drafts + (s.count + 31) / 32 - block0;
    const int splits = min(it.splits, units), split = it.split;
    if (split >= splits) return;
    if (a.splits > 1 && split == 0 && tid == 0)
        a.jobs[(static_cast<size_t>(it.seq) * a.tiles + it.tile) * a.cache.kv_heads + head] = TreeJob{it.first, static_cast<uint32_t>(splits)};
    // (Products of 64 parts and 2^24 columns.)
    const int from = block0 + static_cast<int>(static_cast<uint32_t>(split * units) / static_cast<uint32_t>(splits));
    const int to = block0 + static_cast<int>(static_cast<uint32_t>((split + 1) * units) / static_cast<uint32_t>(splits));
    const bool has_drafts = drafts < to;

    // Everything that depends on the item alone is under way first.  The wave's
    // full blocks: from + wave + 4 n.  Lane x keeps the page of the x-th of
    // the next 64, -1 for a bad one.
    const int32_t *table = a.batch.table + static_cast<size_t>(it.seq) * a.batch.table_width;
    const int start = from + wave, full_to = min(to, full_blocks);
    const int full = full_to > start ? (full_to - start + kWaves - 1) / kWaves : 0;
    int unit = max(opens, from);  // the wave's own of those of 32 tokens
    unit += (from + wave - unit) & (kWaves - 1);
    const bool open_mine = unit < min(to, drafts), drafts_mine = unit >= drafts && unit < to;
    const int which = open_mine ? unit - opens : unit - drafts;  // half
    int pages = 0;
    if (full > 0) pages = table[min(start + kWaves * lane, full_to - 1)];
    const Tile planes = tile_at(a.cache.open + open_tile(a.cache, s.slot, full_blocks, head), 4 * kBlock * D);
    f32x2 open_scale = {0.0f, 0.0f};
    if (open_mine) {
        const float *scales = a.cache.open_scales + open_scale_row(a.cache, s.slot, full_blocks, head);
        open_scale = f32x2{scales[lane], scales[kBlock + lane]};
    }
    Eight<T> query[D / 16];
    const int row = first_row + column, token = row < rows ? token_of(a, row) : 0;
    load_query<D, T>(query, static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(s.first + token) * a.d.q.token_stride +
                                (head * a.group + (row < rows ? row - token * group : 0)) * a.d.q.head_stride);
    uint64_t seen = a.d.seen[s.first + token];  // of the drafts, by the lane's row
    DraftRows<D, T, D / 32> draft_rows;  // all 64 by all threads
    DraftRows<D, T, 1> few_rows;
    const bool few = s.count <= DraftRows<D, T, 1>::kTokens;
    if (has_drafts) {
        if (few) load_drafts(few_rows, a, s.first, s.count, head);
        else load_drafts(draft_rows, a, s.first, s.count, head);
    }
    tile_end();
    constexpr size_t kPlane = kKvBlock * D;
    const int8_t *head_pages = a.cache.pages + head * (2 * kPlane);
    const float *head_scales = a.cache.scales + 2 * head;
    const uint32_t page_bytes = a.cache.kv_heads * static_cast<uint32_t>(2 * kPlane), page_count = a.cache.page_count;
    TreeRaw<D> ka, vb;  // K and V of a full block, or K's high and low bytes, V's of the open one's half
    f32x2 scale_next = {0.0f, 0.0f};
    Tile tile = planes;
    const auto check_pages = [&](int n) {
        if (__builtin_expect(static_cast<uint32_t>(pages) >= page_count, 0)) {
            if (n + lane < full) count_fault(a.cache);
            pages = -1;
        }
    };
    const auto next = [&](int n) {
        if (__builtin_expect(n % 64 == 0 && n != 0, 0)) {
            pages = table[min(start + kWaves * (n + lane), full_to - 1)];
            check_pages(n);
        }
        const int page = __builtin_amdgcn_readlane(pages, n % 64), safe = max(page, 0);
        tile = tile_at(head_pages + static_cast<size_t>(static_cast<uint32_t>(safe)) * page_bytes, 2 * kBlock * D);
        scale_next = *(gptr_f32x2)(uintptr_t)(head_scales + static_cast<size_t>(static_cast<uint32_t>(safe)) * (2 * a.cache.kv_heads));
        return page >= 0;
    };
    bool good_next = true;
    if (full > 0) {
        check_pages(0);
        good_next = next(0);
        load_k(ka, tile);
        load_v(vb, tile);
    } else if (open_mine) {
        load_open_k(ka, planes, which);
        load_open_v(vb, planes, which);
    }
    tile_end();
    ManyState<D, SPLIT> st;
    set_query<D, SPLIT, T>(st, query, a.d.scale);
    const uint64_t there = s.count >= 64 ? ~0ull : (1ull << s.count) - 1;
    seen &= there;
    st.position = s.past - 1 + __builtin_popcountll(seen);
    if (open_mine) {
        open_scales[wave][lane] = open_scale[0];
        open_scales[wave][kBlock + lane] = open_scale[1];
    }
    if (has_drafts) {  // the same for the whole workgroup
        if (few) stage_drafts(shared.stage, few_rows);
        else stage_drafts(shared.stage, draft_rows);
        __syncthreads();
    }

    // Of the half of the drafts that is the wave's, in the order of its scores.
    uint32_t drafts_seen = 0;
    if (drafts_mine) {
        // Drafted tokens that lie too far above: by 64 at most, all of a row's that sees
        // 64 over one that sees none.
        if (WINDOW && __builtin_expect(a.d.window <= kTreeMax, 0)) {
            const int depth = st.position - (s.past - 1);
            const int depths = __builtin_popcountll(a.d.seen[s.first + min(lane, s.count - 1)] & there);
            for (int j = 0; j < s.count; ++j)
                if (__builtin_amdgcn_readlane(depths, j) + static_cast<int>(a.d.window) <= depth) seen &= ~(1ull << j);
        }
        const uint32_t of = static_cast<uint32_t>(seen >> (32 * which));
#pragma unroll
        for (int x = 0; x < 4; ++x) drafts_seen |= (of >> (8 * x + 4 * half) & 15u) << (4 * x);
    }
    // Of the lane's 32 tokens of a block, in the order of its scores: those cached and within the window.
    const auto seen_from = [&](int first) {
        const int ahead = s.past - 1 - first - 4 * half;
        uint32_t bits = first_tokens(ahead);
        if (WINDOW) {
            const int64_t behind = static_cast<int64_t>(st.position) - first - 4 * half - a.d.window;
            bits &= ~first_tokens(static_cast<int>(max(behind, static_cast<int64_t>(-1))));
        }
        return bits;
    };
    // A full block; `masked` ones are the first of a window's.
    const auto block = [&](int n, auto masked) {
        f32x16 sc[2];
        const float nan = __builtin_nanf("");
        const float k_scale = good_next ? scale_next[0] : nan, v_scale = good_next ? scale_next[1] : nan;
        clear(sc);
        add_scores(st, sc, [&](int t, int f) { return half_piece<false>(ka.x[t * (D / 32) + f / 2], f % 2); });
        tile_end();
        if (n + 1 < full) {
            good_next = next(n + 1);
            load_k(ka, tile);
        } else if (open_mine) {
            load_open_k(ka, planes, which);
        }
        tile_end();
        soften_block(st, sc, k_scale, v_scale, masked ? seen_from((start + kWaves * n) * kBlock) : 0xffffffffu, masked);
        tile_end();
        add_rows(st, sc, [&](int d, int y, int pair) { return half_piece<false>(vb.x[d * 2 + y], pair); });
        tile_end();
        if (n + 1 < full) load_v(vb, tile);
        else if (open_mine) load_open_v(vb, planes, which);
        tile_end();
    };
    int n = 0;
    if (WINDOW)  // no row stands behind past + 63
        for (; n < full && static_cast<int64_t>(s.past) + 63 - (start + kWaves * n) * kBlock >= static_cast<int64_t>(a.d.window); ++n)
            block(n, std::true_type());
    for (; n < full; ++n) block(n, std::false_type());
    // Half of the open block or of the drafts.
    if (open_mine || drafts_mine) {
        f32x16 sc[1];
        clear(sc);
        uint32_t bits = drafts_seen;
        const float *scales;
        if (open_mine) {
            add_scores(st, sc, [&](int, int f) { return half_piece<false>(ka.x[f / 2], f % 2); });
            add_scores(st, sc, [&](int, int f) { return half_piece<true>(ka.x[D / 32 + f / 2], f % 2); });
            bits = seen_from(full_blocks * kBlock) >> (16 * which);
            scales = open_scales[wave];
        } else {
#pragma unroll
            for (int part = 0; part < SPLIT; ++part)
                add_scores(st, sc, [&](int, int f) {
                    return *reinterpret_cast<const h16x8 *>(shared.stage.part[part].k + (32 * which + column) * (D + 8) + fragment_number(f, half));
                });
            scales = shared.stage.scales;
        }
        soften_tokens(st, sc, open_mine ? 8 : 0, bits, scales + 32 * which + 4 * half);
        if (open_mine) {
            add_rows(st, sc, [&](int d, int y, int) { return half_piece<false>(vb.x[d * 2 + y], 0); });
            add_rows(st, sc, [&](int d, int y, int) { return half_piece<true>(vb.x[d * 2 + y], 1); });
        } else {
#pragma unroll
            for (int part = 0; part < SPLIT; ++part)
                add_rows(st, sc, [&](int d, int y, int) {
                    return *reinterpret_cast<const h16x8 *>(shared.stage.part[part].v + v_place(32 * d + column, 32 * half + 16 * y + 8 * which));
                });
        }
    }

    const float l = add_xor32(st.l);
    float *stats = part_stats<D>(a, blockIdx.x);
    const auto write = [&](int r, int d, const Joined &joined, f32x4 o) {
        if (splits == 1) {
            write_row<T>(a, s, head, first_row + r, d, joined, o);
            return;
        }
        *reinterpret_cast<f32x4 *>(part_rows<D>(a, blockIdx.x) + static_cast<size_t>(r) * D + d) = o;
        if (d == 0) {
            stats[r] = joined.m;
            stats[kTreeRows + r] = joined.l;
            stats[2 * kTreeRows + r] = joined.e;
        }
    };
    // The waves' rows meet in LDS, their statistics first: each wave brings its rows
    // to the row's own unit.
    __syncthreads();
    TreeJoin<D> &j = shared.join;
    if (half == 0) {
        j.m[wave][column] = st.m;
        j.l[wave][column] = l;
        j.e[wave][column] = st.e;
    }
    __syncthreads();
    Joined own = {kNegInf, 0.0f, kNegInf};
    for (int i = 0; i < kWaves; ++i) own.m = fmaxf(own.m, j.m[i][column]);
    const float ref = own.m == kNegInf ? 0.0f : own.m;
    for (int i = 0; i < kWaves; ++i) {
        own.e = fmaxf(own.e, shifted_unit(ref, j.m[i][column], j.e[i][column]));
        own.l += j.l[i][column] * __builtin_amdgcn_exp2f(j.m[i][column] - ref);
    }
    if (wave == 0 && half == 0) j.joined[column] = own;
    const float factor = part_factor(ref, own.e, st.m, st.e);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4 *>(&j.o[wave][column][32 * d + 8 * x + 4 * half]) =
                f32x4{st.o[d][4 * x], st.o[d][4 * x + 1], st.o[d][4 * x + 2], st.o[d][4 * x + 3]} * factor;
    __syncthreads();
#pragma unroll
    for (int x = tid; x < 32 * (D / 4); x += kTreeThreads) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        if (r >= live_rows) break;
        f32x4 o[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) o[i] = *reinterpret_cast<const f32x4 *>(&j.o[i][r][d]);
        write(r, d, j.joined[r], (o[0] + o[1]) + (o[2] + o[3]));
    }
}

// Joins the parts of split tiles, in their order: a workgroup takes 1024 / D
// rows, D / 4 threads a row, a launch of its own, since the last workgroup of a tile
// to arrive would read them alone.
template <int D, typename T>
__global__ __launch_bounds__(256) void join_tree_kernel(const TreeArgs a) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes, kParts = static_cast<int>(kTreeSplits), kEach = kParts / kLanes;
    __shared__ float factor[kRows][kParts];
    const int tid = threadIdx.x, lane = tid % kLanes, d = 4 * lane;
    constexpr uint32_t per = kTreeRows / kRows;
    const uint32_t heads = a.cache.kv_heads, head = blockIdx.y, tile = blockIdx.x / per, i = blockIdx.z;
    const TreeJob parts = a.jobs[(static_cast<size_t>(i) * a.tiles + tile) * heads + head];  // (of another call's where the sequence has no such tile)
    const Seq s = draft_seq(a, i);
    const int first_row = static_cast<int>(tile * kTreeRows), r = static_cast<int>(blockIdx.x % per) * kRows + tid / kLanes;
    const int rows = s.ok ? s.count * static_cast<int>(a.group) : 0, here = min(rows - first_row, static_cast<int>(kTreeRows));
    if (static_cast<int>(blockIdx.x % per) * kRows >= here) return;
    const int splits = static_cast<int>(parts.splits);
    if (splits <= 1) return;
    const bool live = r < here;
    const int at = live ? r : 0;
    const auto load = [&](int p) {
        return *(gptr_f32x4)(uintptr_t)(part_rows<D>(a, parts.first + static_cast<uint32_t>(min(p, splits - 1)) * heads) + static_cast<size_t>(at) * D + d);
    };
    // The first parts' rows are under way while the row's lanes, a part each or
    // more, turn its statistics into the parts' factors.
    constexpr int kBatch = 8;
    f32x4 v[kBatch];
#pragma unroll
    for (int p = 0; p < kBatch; ++p) v[p] = load(p);
    float m[kEach], l[kEach], e[kEach];
    Joined w = {kNegInf, 0.0f, kNegInf};
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
        const int p = lane + x * kLanes;
        m[x] = e[x] = kNegInf;
        l[x] = 0.0f;
        if (p < splits) {
            const float *stat = part_stats<D>(a, parts.first + static_cast<uint32_t>(p) * heads) + at;
            m[x] = stat[0];
            l[x] = stat[kTreeRows];
            e[x] = stat[2 * kTreeRows];
        }
        w.m = fmaxf(w.m, m[x]);
    }
    const auto most = [&](float x) {
        x = fmaxf(x, dpp<kDppXor1>(x));
        x = fmaxf(x, dpp<kDppXor2>(x));
        x = fmaxf(x, dpp<kDppMirror8>(x));
        x = fmaxf(x, dpp<kDppMirror16>(x));
        return kLanes == 32 ? max_xor16(x) : x;
    };
    w.m = most(w.m);
    const float ref = w.m == kNegInf ? 0.0f : w.m;
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
        w.e = fmaxf(w.e, shifted_unit(ref, m[x], e[x]));
        w.l += l[x] * __builtin_amdgcn_exp2f(m[x] - ref);
    }
    w.e = most(w.e);
    w.l = lanes_sum<16>(w.l);
    if (kLanes == 32) w.l = add_xor16(w.l);
#pragma unroll
    for (int x = 0; x < kEach; ++x) factor[tid / kLanes][lane + x * kLanes] = part_factor(ref, w.e, m[x], e[x]);
    __syncthreads();
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < splits; p0 += kBatch) {
#pragma unroll
        for (int p = 0; p < kBatch; ++p)
            if (p0 + p < splits) o += v[p] * factor[tid / kLanes][p0 + p];
        if (p0 + kBatch < splits) {
#pragma unroll
            for (int p = 0; p < kBatch; ++p) v[p] = load(p0 + kBatch + p);
        }
    }
    if (live) write_row<T>(a, s, head, first_row + r, d, w, o);
}

}  // namespace

template <int D, int SPLIT, typename T>
static void launch_tree_as(const TreeArgs &a, hipStream_t stream) {
    const dim3 tiles(a.tiles, a.cache.kv_heads, a.batch.sequences);
    auto go = [&](auto kernel) { kernel<<<a.splits == 1 ? tiles : dim3(a.workgroups), kTreeThreads, 0, stream>>>(a); };
    constexpr int kAlone = D == 128 && SPLIT == 2 ? 1 : 2;
    if (a.per_cu == 1) a.d.window == 0 ? go(attend_tree_kernel<D, SPLIT, T, false, kAlone>) : go(attend_tree_kernel<D, SPLIT, T, true, kAlone>);
    else a.d.window == 0 ? go(attend_tree_kernel<D, SPLIT, T, false, 2>) : go(attend_tree_kernel<D, SPLIT, T, true, 2>);
    if (a.splits == 1) return;
    join_tree_kernel<D, T><<<dim3(a.tiles * (kTreeRows * D / 1024), tiles.y, tiles.z), 256, 0, stream>>>(a);
}
template <int SPLIT, typename T>
static void launch_tree_as(const TreeArgs &a, hipStream_t stream) {
    a.cache.head_dim == 64 ? launch_tree_as<64, SPLIT, T>(a, stream) : launch_tree_as<128, SPLIT, T>(a, stream);
}
hipError_t launch_attend_tree(const TreeArgs &a, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_tree_as<2, float>(a, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_tree_as<1, _Float16>(a, stream);
    else launch_tree_as<1, __bf16>(a, stream);
    return hipGetLastError();
}

}  // namespace q4rdna
