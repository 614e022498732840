// The 8-bit paged key/value cache: appending a step's tokens (q4rdna_kv_append)
// and reading tokens back (q4rdna_kv_read).  The cache's format and its rounding
// rules are those of include/q4rdna.h.
//
// Both kernels move bytes and do little else.  A workgroup takes one block of
// one kv head, K and V: it needs all of a block's scales when the block fills,
// and LDS turns rows of numbers into the pages' order and writes whole 16-byte
// pieces.  7873 tokens of six prompts (bf16, 8 kv heads, 32 heads of q with norm
// and rotation, 177 MB) take 55 us, 3.2 TB/s of the 5.2 that a copy reaches: the
// vector unit is busy 36 % of the time, the rest is waiting for rows, with the
// four workgroups that the stage's 36 KB lets a CU have, those of q among them,
// which use none of it.  Reading them back (48 MB) takes 14 us, for the same
// reason: a workgroup's loads, then its stores.  One token takes 4.4 us and 64
// sequences' tokens 9.3 us, where some fill their blocks: a block that closes is
// a chain of loads (lengths, open planes, page) with LDS round trips between.
#include "q4rdna_layer_device.h"
#include "q4rdna_rotate_device.h"

namespace q4rdna {
namespace {

// A workgroup stages its block's 16-bit codes as [K, V][64 tokens][D + 8]
// shorts: the pad keeps rows 16-byte aligned and shifts them by four banks.
template <int D>
constexpr int kRow = D + 8;

// x * f rounded to the nearest integer, as the low bits of a float's: the sum
// with 1.5 * 2^23 has a last place of one.  For |x * f| < 2^22; a NaN gives 0
// in its low bits.
__device__ __forceinline__ uint32_t rounded(float x, float f) { return __float_as_uint(fmaf(x, f, 12582912.0f)); }
// The same with the product rounded first.  Where the exact product lies midway
// between two integers, which numbers of few bits often meet, a factor that is off
// by a last place would decide; rounded, it is midway again and goes to the even one.
__device__ __forceinline__ uint32_t rounded_twice(float x, float f) {
#pragma clang fp contract(off)
    const float y = x * f;
    return __float_as_uint(y + 12582912.0f);
}
// 32512 / largest, rounded once, for 1e-30 and more: a quarter of both, since the
// reciprocal of a number above 2^126 would be subnormal, which the instruction
// gives as zero; its refined reciprocal, the quotient and that one's remainder.
__device__ __forceinline__ float code_factor(float largest) {
#pragma clang fp contract(off)
    const float b = 0.25f * largest, a = 0.25f * kKvCode16;
    float y = __builtin_amdgcn_rcpf(b);
    y = fmaf(fmaf(-b, y, 1.0f), y, y);
    const float q = a * y;
    return fmaf(fmaf(-b, q, a), y, q);
}
// largest / 32512, rounded once: the product with the reciprocal and its remainder.
// (At fp32's very end it is rounded down, for the largest code times it to be finite.)
__device__ __forceinline__ float token_scale(float largest) {
    const float per = 1.0f / kKvCode16, q = largest * per;
    return fminf(fmaf(fmaf(-q, kKvCode16, largest), per, q), 0x1.0204060000000p+113f);
}
// The low halves of four of them.
__device__ __forceinline__ s16x4 pack_codes(const float (&x)[4], float f) {
    const uint32_t w[2] = {__builtin_amdgcn_perm(rounded(x[1], f), rounded(x[0], f), 0x05040100u),
                           __builtin_amdgcn_perm(rounded(x[3], f), rounded(x[2], f), 0x05040100u)};
    return __builtin_bit_cast(s16x4, w);
}

// The low bytes of four values, packed.
__device__ __forceinline__ uint32_t pack4(int x0, int x1, int x2, int x3) {
    const uint32_t lo = __builtin_amdgcn_perm(static_cast<uint32_t>(x1), static_cast<uint32_t>(x0), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(static_cast<uint32_t>(x3), static_cast<uint32_t>(x2), 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// Four words of four bytes, transposed.
__device__ __forceinline__ void transpose4(const uint32_t (&t)[4], uint32_t (&n)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400u), b = __builtin_amdgcn_perm(t[1], t[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(t[3], t[2], 0x05010400u), d = __builtin_amdgcn_perm(t[3], t[2], 0x07030602u);
    n[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    n[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    n[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    n[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// A 16-bit code as 256 * high + low, low a signed byte.
__device__ __forceinline__ int high_of(int v) { return (v + 128) >> 8; }
__device__ __forceinline__ short join16(i32x4 high, i32x4 low, int e) {
    const int h = static_cast<int8_t>(static_cast<uint32_t>(high[e / 4]) >> (8 * (e % 4)));
    const int l = static_cast<int8_t>(static_cast<uint32_t>(low[e / 4]) >> (8 * (e % 4)));
    return static_cast<short>(256 * h + l);
}

// 16-byte pieces of a block of one head, in memory order.  A K piece is 16
// numbers (from k_number) of one token, a V piece 16 tokens (v_token of 0..15)
// of one number.
template <int D>
__device__ __forceinline__ int k_token(int piece) { return piece / (64 * (D / 64)) * 16 + piece % 16; }
template <int D>
__device__ __forceinline__ int k_number(int piece) { return piece / 64 % (D / 64) * 64 + piece / 16 % 4 * 16; }
__device__ __forceinline__ int v_token(int piece, int e) { return e / 4 * 16 + piece / 16 % 4 * 4 + e % 4; }
__device__ __forceinline__ int v_number(int piece) { return piece / 64 * 16 + piece % 16; }
template <int D>
__device__ __forceinline__ int k_piece(int token, int number) {
    return ((token / 16 * (D / 64) + number / 64) * 4 + number / 16 % 4) * 16 + token % 16;
}
__device__ __forceinline__ int v_piece(int token, int number) {
    return (number / 16 * 4 + token / 4 % 4) * 16 + number % 16;
}
__device__ __forceinline__ int v_byte(int token) { return token / 16 * 4 + token % 4; }

template <int D>
struct AppendStage {
    short code[2][kKvBlock * kRow<D>];
    float scale[2][kKvBlock];
    float ratio[2][kKvBlock];
    float block_scale[2];
};

// One (sequence, block, kv head): the step's tokens in the block to 16-bit codes
// in LDS, then the open planes, and the page where the block is full.
template <int D, bool INTERLEAVED, typename T>
__device__ void append_block(const AppendArgs &a, const Seq &s, uint32_t i, uint32_t head, int block, AppendStage<D> &st) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes, kPieces = kKvBlock * D / 16;
    const uint32_t heads = a.cache.kv_heads;
    const int tid = threadIdx.x;
    const int start = block * static_cast<int>(kKvBlock);
    const int from = max(s.past - start, 0), to = min(s.length - start, static_cast<int>(kKvBlock));
    const int fresh = to - from;
    const bool full = to == static_cast<int>(kKvBlock);
    const bool keep = block >= s.length / static_cast<int>(kKvBlock) - 1;

    // Rows: the block's K rows, then its V rows, a group of D / 8 lanes each,
    // kEach of them in flight: an fp32 block's in one turn (four and eight:
    // 128 tokens 10.5 and 9.7 us, 1024 14.7 and 12.9, one 4.0 and 4.1; bf16
    // 128 10.4 and 10.1, 4096 24.1 and 24.5, one 3.8 and 4.0).
    constexpr int kEach = sizeof(T) == 4 ? 8 : 4;
    const int lane = tid % kLanes;
    Weights weights;
    load_weights(weights, a.d.k_norm, place_of<INTERLEAVED>(lane, a.d.rotary));
    for (int row0 = tid / kLanes; row0 < 2 * fresh; row0 += kEach * kRows) {
        Row r[kEach];
        Turn turn[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int row = row0 + x * kRows;
            if (row < 2 * fresh) {
                const bool is_v = row >= fresh;
                const int t = from + (is_v ? row - fresh : row);
                const size_t n = static_cast<size_t>(s.first) + (start + t - s.past);
                const void *data = is_v ? a.d.v.data : a.d.k.data;
                const int64_t token_stride = is_v ? a.d.v.token_stride : a.d.k.token_stride;
                const int64_t head_stride = is_v ? a.d.v.head_stride : a.d.k.head_stride;
                const Place at = place_of<INTERLEAVED>(lane, is_v ? 0 : a.d.rotary);
                load_row(r[x], static_cast<const T *>(data) + n * token_stride + head * head_stride, at,
                         a.wide != 0);
                load_turn(turn[x], at, a.d.cos, a.d.sin, a.d.rotary, start + t);
            }
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int row = row0 + x * kRows;
            if (row < 2 * fresh) {
                const bool is_v = row >= fresh;
                const int t = from + (is_v ? row - fresh : row);
                const Place at = place_of<INTERLEAVED>(lane, is_v ? 0 : a.d.rotary);
                if (!is_v && a.d.k_norm != nullptr) norm_row<D>(r[x], weights, a.d.eps);
                turn_row<INTERLEAVED>(r[x], at, turn[x]);
                // The largest magnitude by its bits: infinities and NaN come out on top.
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top = max(top, max(__float_as_uint(r[x].a[e]) & 0x7fffffffu, __float_as_uint(r[x].b[e]) & 0x7fffffffu));
                top = lanes_max<kLanes>(top);
                const float largest = __uint_as_float(top);
                const bool finite = top < 0x7f800000u, some = finite && largest >= kKvZero;
                const float inv = some ? code_factor(largest) : 0.0f;
                short *out = &st.code[is_v][t * kRow<D>];
                *reinterpret_cast<s16x4 *>(out + at.a_at) = pack_codes(r[x].a, inv);
                *reinterpret_cast<s16x4 *>(out + at.b_at) = pack_codes(r[x].b, inv);
                if (lane == 0) st.scale[is_v][t] = some ? token_scale(largest) : finite ? 0.0f : __builtin_nanf("");
            }
        }
    }

    int8_t *planes = a.cache.open + open_tile(a.cache, s.slot, block, head);
    float *scales = a.cache.open_scales + open_scale_row(a.cache, s.slot, block, head);
    constexpr size_t kPlane = kKvBlock * D;
    if (full && from > 0) {  // the tokens that were there, from the open block
        for (int piece = tid; piece < kPieces; piece += 256) {
            const int t = k_token<D>(piece);
            if (t < from) {
                const i32x4 h = load16(planes + 16 * piece), l = load16(planes + kPlane + 16 * piece);
                s16x8 *row = reinterpret_cast<s16x8 *>(&st.code[0][t * kRow<D> + k_number<D>(piece)]);
                s16x8 c[2];
#pragma unroll
                for (int e = 0; e < 16; ++e) c[e / 8][e % 8] = join16(h, l, e);
                row[0] = c[0];
                row[1] = c[1];
            }
            if (v_token(piece, 0) < from) {
                const i32x4 h = load16(planes + 2 * kPlane + 16 * piece), l = load16(planes + 3 * kPlane + 16 * piece);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (v_token(piece, e) < from)
                        st.code[1][v_token(piece, e) * kRow<D> + v_number(piece)] = join16(h, l, e);
            }
        }
        if (tid < 128 && tid % 64 < from) st.scale[tid / 64][tid % 64] = scales[tid];
    }
    __syncthreads();

    if (keep) {
        if (tid < 128 && tid % 64 >= from && tid % 64 < to) scales[tid] = st.scale[tid / 64][tid % 64];
        for (int x = tid; x < fresh * (D / 16); x += 256) {
            const int t = from + x / (D / 16), number = x % (D / 16) * 16;
            const s16x8 *row = reinterpret_cast<const s16x8 *>(&st.code[0][t * kRow<D> + number]);
            const s16x8 c[2] = {row[0], row[1]};
            i32x4 h, l;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const s16x8 v = c[w / 2];
                const int e = 4 * (w % 2);
                h[w] = static_cast<int>(pack4(high_of(v[e]), high_of(v[e + 1]), high_of(v[e + 2]), high_of(v[e + 3])));
                l[w] = static_cast<int>(pack4(v[e], v[e + 1], v[e + 2], v[e + 3]));
            }
            const int at = 16 * k_piece<D>(t, number);
            store16(planes + at, h);
            store16(planes + kPlane + at, l);
        }
        int8_t *v_planes = planes + 2 * kPlane;
        if (fresh < 16) {  // few tokens: their bytes
            for (int x = tid; x < fresh * D; x += 256) {
                const int t = from + x / D, number = x % D;
                const int v = st.code[1][t * kRow<D> + number];
                const int at = 16 * v_piece(t, number) + v_byte(t);
                v_planes[at] = static_cast<int8_t>(high_of(v));
                v_planes[kPlane + at] = static_cast<int8_t>(v);
            }
        } else {
            // Whole pieces, 16 tokens of each of four numbers.  Tokens before
            // `from` keep their bytes; what lies behind `to` is never read.
            for (int x = tid; x < D; x += 256) {
                const int number = x % (D / 4) * 4, g = x / (D / 4), at = 16 * v_piece(4 * g, number);
                i32x4 h[4], l[4];
                if (from > 4 * g) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        h[n] = load16(v_planes + at + 16 * n);
                        l[n] = load16(v_planes + kPlane + at + 16 * n);
                    }
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t ht[4], lt[4], hn[4], ln[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const s16x4 c = *reinterpret_cast<const s16x4 *>(&st.code[1][(16 * w + 4 * g + b) * kRow<D> + number]);
                        ht[b] = pack4(high_of(c[0]), high_of(c[1]), high_of(c[2]), high_of(c[3]));
                        lt[b] = pack4(c[0], c[1], c[2], c[3]);
                    }
                    transpose4(ht, hn);
                    transpose4(lt, ln);
                    const int kept = min(max(from - (16 * w + 4 * g), 0), 4);  // tokens of the word that were there
                    const uint32_t mask = kept == 4 ? 0xffffffffu : (1u << (8 * kept)) - 1u;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint32_t oh = kept ? static_cast<uint32_t>(h[n][w]) : 0, ol = kept ? static_cast<uint32_t>(l[n][w]) : 0;
                        h[n][w] = static_cast<int>((hn[n] & ~mask) | (oh & mask));
                        l[n][w] = static_cast<int>((ln[n] & ~mask) | (ol & mask));
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    store16(v_planes + at + 16 * n, h[n]);
                    store16(v_planes + kPlane + at + 16 * n, l[n]);
                }
            }
        }
    }
    if (!full) return;

    // The page: the block's scale is 256 times the largest token scale.
    const int page = a.batch.table[static_cast<size_t>(i) * a.batch.table_width + block];
    if (static_cast<uint32_t>(page) >= a.cache.page_count) {
        if (tid == 0) count_fault(a.cache);
        return;
    }
    if (tid < 128) {
        const int which = tid / 64;
        const float mine = st.scale[which][tid % 64];
        uint32_t top = __float_as_uint(mine) & 0x7fffffffu;  // scales are not negative; NaN comes out on top
        top = lanes_max<16>(top);
        top = max(max(static_cast<uint32_t>(__builtin_amdgcn_readlane(top, 0)),
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(top, 16))),
                  max(static_cast<uint32_t>(__builtin_amdgcn_readlane(top, 32)),
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(top, 48))));
        const float whole = 256.0f * __uint_as_float(top);
        const bool some = top != 0 && top < 0x7f800000u;
        st.ratio[which][tid % 64] = some ? mine / whole : 0.0f;
        if (tid % 64 == 0)
            a.cache.scales[(static_cast<size_t>(page) * heads + head) * 2 + which] = whole;
    }
    __syncthreads();
    int8_t *tile = a.cache.pages + page_tile(a.cache, page, head);
    if (tid < 128) {
        // K: 16 numbers of a token are a piece.
        for (int piece = tid; piece < kPieces; piece += 128) {
            const int t = k_token<D>(piece);
            const s16x8 *row = reinterpret_cast<const s16x8 *>(&st.code[0][t * kRow<D> + k_number<D>(piece)]);
            const float r = st.ratio[0][t];
            i32x4 k;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const s16x8 c = row[w / 2];
                int x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = static_cast<int>(rounded_twice(c[4 * (w % 2) + e], r));
                k[w] = static_cast<int>(pack4(x[0], x[1], x[2], x[3]));
            }
            store16(tile + 16 * piece, k);
        }
    } else {
        // V: 16 tokens of each of four numbers, transposed four by four.
        for (int x = tid - 128; x < D; x += 128) {
            const int number = x % (D / 4) * 4, g = x / (D / 4);
            i32x4 v[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t by_token[4], by_number[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int t = 16 * w + 4 * g + b;
                    const s16x4 c = *reinterpret_cast<const s16x4 *>(&st.code[1][t * kRow<D> + number]);
                    const float r = st.ratio[1][t];
                    by_token[b] = pack4(static_cast<int>(rounded_twice(c[0], r)), static_cast<int>(rounded_twice(c[1], r)),
                                        static_cast<int>(rounded_twice(c[2], r)), static_cast<int>(rounded_twice(c[3], r)));
                }
                transpose4(by_token, by_number);
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n][w] = static_cast<int>(by_number[n]);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) store16(tile + kPlane + 16 * (v_piece(4 * g, number) + n), v[n]);
        }
    }
}

// The blocks of one place and kv head.
template <int D, bool INTERLEAVED, typename T>
__device__ void append_place(const AppendArgs &a, uint32_t unit, AppendStage<D> &st) {
    const uint32_t place = unit / a.cache.kv_heads, head = unit - place * a.cache.kv_heads;
    uint32_t first_place;
    const uint32_t i = place_seq(a.batch, place, &first_place);
    Seq s = seq_of(a.batch, a.cache, i);
    if (s.ok && a.d.rotary != 0 && static_cast<uint32_t>(s.length) > a.d.positions) s.ok = false;
    if (!s.ok) {
        if (threadIdx.x == 0 && head == 0 && place == first_place) count_fault(a.cache);
        return;
    }
    constexpr int kBlock = kKvBlock;
    const int first = s.past / kBlock;
    const int64_t block64 = static_cast<int64_t>(first) + (place - first_place);
    if (s.count == 0 || block64 * kBlock >= s.length) return;
    const int block = static_cast<int>(block64);
    // The first block may hold tokens in the open planes that a later block of
    // the same parity, one of the last two, writes in this step.  Then the
    // later block's workgroup fills both, the first one first.
    int owner = first;
    if (s.past % kBlock != 0) {
        const int last = s.length / kBlock;
        const int same = (last ^ first) & 1 ? last - 1 : last;
        if (same > first && same * kBlock < s.length) owner = same;
    }
    if (owner != first) {
        if (block == first) return;
        if (block == owner) {
            append_block<D, INTERLEAVED, T>(a, s, i, head, first, st);
            __syncthreads();
        }
    }
    append_block<D, INTERLEAVED, T>(a, s, i, head, block, st);
}

// a.q_rows rows (token, query head) of q, kEach per group of D / 8 lanes in
// flight.  The waves of a CU are many here, and more rows each cost registers
// (two, four and eight, fp32: 2048 tokens 18.1, 20.2 and 25.2 us).
template <int D, bool INTERLEAVED, typename T>
__device__ void turn_q(const AppendArgs &a, uint32_t unit) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes, kEach = 2;
    const int lane = threadIdx.x % kLanes;
    const Place at = place_of<INTERLEAVED>(lane, a.d.rotary);
    Weights weights;
    load_weights(weights, a.d.q_norm, at);
    const uint32_t heads = a.d.q_heads;
    // One division per workgroup, a multiplication per row.
    const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * heads, row_first = static_cast<uint64_t>(unit) * a.q_rows;
    const uint32_t n_first = mul_div(unit, a.q_rows, heads);
    const uint32_t head_first = static_cast<uint32_t>(row_first - static_cast<uint64_t>(n_first) * heads);
    const uint32_t row_count = static_cast<uint32_t>(min(rows - row_first, static_cast<uint64_t>(a.q_rows)));
    // The workgroup's tokens are mostly of one sequence: the first one's.
    const Seq s0 = seq_of(a.batch, a.cache, wave_token_seq(a.batch, n_first));
    for (uint32_t x0 = threadIdx.x / kLanes; x0 < row_count; x0 += kEach * kRows) {
        Row r[kEach];
        Turn turn[kEach];
        uint32_t n[kEach], head[kEach];
        bool live[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            live[x] = x0 + x * kRows < row_count;
            const uint32_t local = head_first + (live[x] ? x0 + x * kRows : 0), token = div_split(local, heads, a.heads_magic);
            n[x] = n_first + token;
            head[x] = local - token * heads;
            if (live[x])
                load_row(r[x], static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(n[x]) * a.d.q.token_stride +
                                   head[x] * a.d.q.head_stride, at, a.wide != 0);
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            if (!live[x]) continue;
            Seq s = s0;
            if (!s.ok || static_cast<int>(n[x]) < s.first || static_cast<int>(n[x]) >= s.first + s.count)
                s = seq_of(a.batch, a.cache, token_seq(a.batch, n[x]));
            // A refused sequence's rows are not written (it is counted with its blocks).
            live[x] = s.ok && static_cast<int>(n[x]) >= s.first && static_cast<int>(n[x]) < s.first + s.count &&
                      (a.d.rotary == 0 || static_cast<uint32_t>(s.length) <= a.d.positions);
            if (live[x]) load_turn(turn[x], at, a.d.cos, a.d.sin, a.d.rotary, s.past + static_cast<int>(n[x]) - s.first);
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            if (!live[x]) continue;
            if (a.d.q_norm != nullptr) norm_row<D>(r[x], weights, a.d.eps);
            turn_row<INTERLEAVED>(r[x], at, turn[x]);
            T *out = static_cast<T *>(a.d.q_out.data) + static_cast<int64_t>(n[x]) * a.d.q_out.token_stride +
                     head[x] * a.d.q_out.head_stride;
            store_floats<T, 4>(out + at.a_at, a.wide != 0, r[x].a);
            store_floats<T, 4>(out + at.b_at, a.wide != 0, r[x].b);
        }
    }
}

template <int D, bool INTERLEAVED, typename T>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
    __shared__ AppendStage<D> stage;
    // The blocks' workgroups, which wait a lot, spread evenly among q's, which
    // move the most bytes.
    const uint32_t before = mul_div(blockIdx.x, a.kv_units, gridDim.x);
    if (mul_div(blockIdx.x + 1, a.kv_units, gridDim.x) != before)
        append_place<D, INTERLEAVED, T>(a, before, stage);
    else
        turn_q<D, INTERLEAVED, T>(a, blockIdx.x - before);
}

// Byte e of a word as a signed number.
__device__ __forceinline__ int byte_of(uint32_t w, int e) { return static_cast<int8_t>(w >> (8 * e)); }

// One (sequence, block, kv head): its tokens past .. length - 1 as numbers.
// Half of the threads take K, a piece (16 numbers of a token) at a time, eight
// lanes a token's row; the others V, 16 tokens of four numbers, which are
// transposed four by four, so that lanes side by side write a row.
template <int D, typename T>
__global__ __launch_bounds__(256) void read_kernel(const ReadArgs a) {
    const uint32_t heads = a.cache.kv_heads;
    const uint32_t place = blockIdx.x / heads, head = blockIdx.x - place * heads;
    const int tid = threadIdx.x;
    uint32_t first_place;
    const uint32_t i = place_seq(a.batch, place, &first_place);
    const Seq s = seq_of(a.batch, a.cache, i);
    if (!s.ok) {
        if (tid == 0 && head == 0 && place == first_place) count_fault(a.cache);
        return;
    }
    const int64_t block64 = static_cast<int64_t>(s.past) / kKvBlock + (place - first_place);
    if (s.count == 0 || block64 * kKvBlock >= s.length) return;
    const int block = static_cast<int>(block64);
    const int start = block * static_cast<int>(kKvBlock);
    const int from = max(s.past - start, 0), to = min(s.length - start, static_cast<int>(kKvBlock));
    const bool full = start + static_cast<int>(kKvBlock) <= s.length;
    constexpr size_t kPlane = kKvBlock * D;
    const int8_t *tile;
    const float *scales;
    float bad = 0.0f;
    if (full) {
        int page = a.batch.table[static_cast<size_t>(i) * a.batch.table_width + block];
        if (static_cast<uint32_t>(page) >= a.cache.page_count) {
            if (tid == 0) count_fault(a.cache);
            page = 0;
            bad = __builtin_nanf("");
        }
        tile = a.cache.pages + page_tile(a.cache, page, head);
        scales = a.cache.scales + (static_cast<size_t>(page) * heads + head) * 2;
    } else {
        tile = a.cache.open + open_tile(a.cache, s.slot, block, head);
        scales = a.cache.open_scales + open_scale_row(a.cache, s.slot, block, head);
    }
    const int64_t row0 = static_cast<int64_t>(s.first) + (start - s.past);  // of the block's token 0
    if (tid < 128) {
        T *out = static_cast<T *>(a.k.data) + head * a.k.head_stride;
#pragma unroll
        for (int x = tid; x < kKvBlock * D / 16; x += 128) {
            const int t = x / (D / 16), number = x % (D / 16) * 16, piece = k_piece<D>(t, number);
            if (t < from || t >= to) continue;
            const i32x4 h = load16(tile + 16 * piece);
            i32x4 l = {0, 0, 0, 0};
            if (!full) l = load16(tile + kPlane + 16 * piece);
            const float scale = full ? scales[0] + bad : scales[t], high = full ? 1.0f : 256.0f;
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                v[e] = (byte_of(h[e / 4], e % 4) * high + byte_of(l[e / 4], e % 4)) * scale;
            store_floats<T, 16>(out + (row0 + t) * a.k.token_stride + number, a.wide != 0, v);
        }
    } else {
        T *out = static_cast<T *>(a.v.data) + head * a.v.head_stride;
        const int8_t *plane = tile + (full ? 1 : 2) * kPlane;
        for (int x = tid - 128; x < D; x += 128) {
            const int number = x % (D / 4) * 4, g = x / (D / 4), piece = v_piece(4 * g, number);
            if (4 * g >= to || 4 * g + 51 < from) continue;
            i32x4 h[4], l[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                h[n] = load16(plane + 16 * (piece + n));
                l[n] = i32x4{0, 0, 0, 0};
                if (!full) l[n] = load16(plane + kPlane + 16 * (piece + n));
            }
            const float high = full ? 1.0f : 256.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const f32x4 by_token = full ? f32x4{scales[1] + bad, scales[1] + bad, scales[1] + bad, scales[1] + bad}
                                            : *(gptr_f32x4)(uintptr_t)(scales + 64 + 16 * w + 4 * g);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int t = 16 * w + 4 * g + b;
                    if (t < from || t >= to) continue;
                    float v[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        v[n] = (byte_of(h[n][w], b) * high + byte_of(l[n][w], b)) * by_token[b];
                    store_floats<T, 4>(out + (row0 + t) * a.v.token_stride + number, a.wide != 0, v);
                }
            }
        }
    }
}

}  // namespace

template <bool INTERLEAVED, typename T>
static void launch_append_as(const AppendArgs &a, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<a.kv_units + a.q_units, 256, 0, stream>>>(a); };
    a.cache.head_dim == 64 ? go(append_kernel<64, INTERLEAVED, T>) : go(append_kernel<128, INTERLEAVED, T>);
}
template <typename T>
static void launch_append_as(const AppendArgs &a, hipStream_t stream) {
    a.d.interleaved != 0 ? launch_append_as<true, T>(a, stream) : launch_append_as<false, T>(a, stream);
}
hipError_t launch_append(const AppendArgs &a, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_append_as<float>(a, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_append_as<_Float16>(a, stream);
    else launch_append_as<__bf16>(a, stream);
    return hipGetLastError();
}

hipError_t launch_read(const ReadArgs &a, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<a.units, 256, 0, stream>>>(a); };
    if (a.cache.head_dim == 64)
        a.dtype == Q4RDNA_F32 ? go(read_kernel<64, float>) : a.dtype == Q4RDNA_F16 ? go(read_kernel<64, _Float16>) : go(read_kernel<64, __bf16>);
    else
        a.dtype == Q4RDNA_F32 ? go(read_kernel<128, float>) : a.dtype == Q4RDNA_F16 ? go(read_kernel<128, _Float16>) : go(read_kernel<128, __bf16>);
    return hipGetLastError();
}

}  // namespace q4rdna
