// The 8-bit paged key/value cache: appending a step's tokens (q4rdna_kv_append)
// and reading tokens back (q4rdna_kv_read).  The cache's format and its rounding
// rules are those of include/q4rdna.h.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

// A workgroup stages its block's 16-bit codes as [K, V][64 tokens][D + 8]
// shorts: the pad keeps rows 16-byte aligned and shifts them by four banks.
template <int D>
constexpr int kRow = D + 8;

// One row of a head in the lanes of a group of D / 8: eight numbers per lane in
// two runs of four, at a_at and b_at.
struct Row {
    float a[4], b[4];
};
struct Place {
    int a_at, b_at;
    bool turned;  // the lane's numbers are rotated
    int pair;     // the first of its four pairs
};

template <int D>
__device__ __forceinline__ Place place_of(int lane, uint32_t rotary, bool interleaved) {
    const int half = static_cast<int>(rotary) / 2;
    Place p;
    p.pair = 4 * lane;
    p.turned = p.pair < half;  // rotary is a multiple of 8: a lane's pairs lie on one side
    if (p.turned && !interleaved) {
        p.a_at = p.pair;
        p.b_at = p.pair + half;
    } else {
        p.a_at = 8 * lane;
        p.b_at = 8 * lane + 4;
    }
    return p;
}

template <typename T>
__device__ __forceinline__ void load_row(Row &r, const T *row, const Place &p, bool wide) {
    load_floats<T, 4>(row + p.a_at, wide, r.a);
    load_floats<T, 4>(row + p.b_at, wide, r.b);
}
// The lane's four cosines and sines at a position.
struct Turn {
    float c[4], s[4];
};
__device__ __forceinline__ void load_turn(Turn &t, const Place &p, const q4rdna_kv_append_desc &d, int position) {
    if (!p.turned) return;
    const size_t at = static_cast<size_t>(position) * (d.rotary / 2) + p.pair;
    load_floats<float, 4>(d.cos + at, true, t.c);
    load_floats<float, 4>(d.sin + at, true, t.s);
}

// The norm of a head's row and its rotation, each product and sum rounded by
// itself (no contraction), as elementary fp32 operations give them.
template <int D>
__device__ __forceinline__ void norm_row(Row &r, const Place &p, const float *weight, float eps) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += r.a[e] * r.a[e] + r.b[e] * r.b[e];
    sum = lanes_sum<D / 8>(sum);
    const float inv = 1.0f / sqrtf(sum * (1.0f / D) + eps);
    float wa[4], wb[4];
    load_floats<float, 4>(weight + p.a_at, true, wa);
    load_floats<float, 4>(weight + p.b_at, true, wb);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r.a[e] = r.a[e] * inv * wa[e];
        r.b[e] = r.b[e] * inv * wb[e];
    }
}
// (By value throughout: references that differ between the two orders of pairs
// would put the rows into scratch memory.)
__device__ __forceinline__ f32x2 turn_pair(float a, float b, float c, float s) {
#pragma clang fp contract(off)
    return f32x2{a * c - b * s, b * c + a * s};
}
__device__ __forceinline__ void turn_row(Row &r, const Place &p, const Turn &t, bool interleaved) {
    if (!p.turned) return;
    // Pair i is (first[i], second[i]).
    const float first[4] = {r.a[0], interleaved ? r.a[2] : r.a[1], interleaved ? r.b[0] : r.a[2], interleaved ? r.b[2] : r.a[3]};
    const float second[4] = {interleaved ? r.a[1] : r.b[0], interleaved ? r.a[3] : r.b[1], interleaved ? r.b[1] : r.b[2], r.b[3]};
    f32x2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = turn_pair(first[i], second[i], t.c[i], t.s[i]);
    r.a[0] = x[0][0];
    r.a[1] = interleaved ? x[0][1] : x[1][0];
    r.a[2] = interleaved ? x[1][0] : x[2][0];
    r.a[3] = interleaved ? x[1][1] : x[3][0];
    r.b[0] = interleaved ? x[2][0] : x[0][1];
    r.b[1] = interleaved ? x[2][1] : x[1][1];
    r.b[2] = interleaved ? x[3][0] : x[2][1];
    r.b[3] = x[3][1];
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

// Two planes of 16 codes from 16 shorts: low bytes as signed numbers, and what
// is left.
__device__ __forceinline__ void split16(const short (&v)[16], i32x4 &high, i32x4 &low) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t h = 0, l = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = v[4 * w + e];
            l |= (static_cast<uint32_t>(x) & 255u) << (8 * e);
            h |= (static_cast<uint32_t>((x + 128) >> 8) & 255u) << (8 * e);
        }
        high[w] = static_cast<int>(h);
        low[w] = static_cast<int>(l);
    }
}
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
template <int D, typename T>
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
    // kEach of them in flight.
    constexpr int kEach = 4;
    const int lane = tid % kLanes;
    const bool interleaved = a.d.interleaved != 0;
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
                const Place at = place_of<D>(lane, is_v ? 0 : a.d.rotary, interleaved);
                load_row(r[x], static_cast<const T *>(data) + n * token_stride + head * head_stride, at,
                         a.wide != 0);
                load_turn(turn[x], at, a.d, start + t);
            }
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int row = row0 + x * kRows;
            if (row < 2 * fresh) {
                const bool is_v = row >= fresh;
                const int t = from + (is_v ? row - fresh : row);
                const Place at = place_of<D>(lane, is_v ? 0 : a.d.rotary, interleaved);
                if (!is_v && a.d.k_norm != nullptr) norm_row<D>(r[x], at, a.d.k_norm, a.d.eps);
                turn_row(r[x], at, turn[x], interleaved);
                // The largest magnitude by its bits: infinities and NaN come out on top.
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top = max(top, max(__float_as_uint(r[x].a[e]) & 0x7fffffffu, __float_as_uint(r[x].b[e]) & 0x7fffffffu));
                top = lanes_max<kLanes>(top);
                const float largest = __uint_as_float(top);
                const bool finite = top < 0x7f800000u, some = finite && largest >= kKvZero;
                const float inv = some ? kKvCode16 / largest : 0.0f;
                s16x4 ca, cb;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ca[e] = some ? static_cast<short>(static_cast<int>(rintf(r[x].a[e] * inv))) : 0;
                    cb[e] = some ? static_cast<short>(static_cast<int>(rintf(r[x].b[e] * inv))) : 0;
                }
                short *out = &st.code[is_v][t * kRow<D>];
                *reinterpret_cast<s16x4 *>(out + at.a_at) = ca;
                *reinterpret_cast<s16x4 *>(out + at.b_at) = cb;
                if (lane == 0) st.scale[is_v][t] = some ? largest / kKvCode16 : finite ? 0.0f : __builtin_nanf("");
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
                short *row = &st.code[0][t * kRow<D> + k_number<D>(piece)];
#pragma unroll
                for (int e = 0; e < 16; ++e) row[e] = join16(h, l, e);
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
            short v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = st.code[0][t * kRow<D> + number + e];
            i32x4 h, l;
            split16(v, h, l);
            const int at = 16 * k_piece<D>(t, number);
            store16(planes + at, h);
            store16(planes + kPlane + at, l);
        }
        if (fresh < 16) {
            for (int x = tid; x < fresh * D; x += 256) {
                const int t = from + x / D, number = x % D;
                const int v = st.code[1][t * kRow<D> + number];
                const int at = 16 * v_piece(t, number) + v_byte(t);
                planes[2 * kPlane + at] = static_cast<int8_t>((v + 128) >> 8);
                planes[3 * kPlane + at] = static_cast<int8_t>(v);
            }
        } else {
            for (int piece = tid; piece < kPieces; piece += 256) {
                short v[16];
                const int number = v_number(piece);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = st.code[1][v_token(piece, e) * kRow<D> + number];
                i32x4 h, l;
                split16(v, h, l);
                if (v_token(piece, 0) >= from && v_token(piece, 15) < to) {
                    store16(planes + 2 * kPlane + 16 * piece, h);
                    store16(planes + 3 * kPlane + 16 * piece, l);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (v_token(piece, e) >= from && v_token(piece, e) < to) {
                            planes[2 * kPlane + 16 * piece + e] = static_cast<int8_t>((v[e] + 128) >> 8);
                            planes[3 * kPlane + 16 * piece + e] = static_cast<int8_t>(v[e]);
                        }
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
                for (int e = 0; e < 4; ++e) x[e] = static_cast<int>(rintf(c[4 * (w % 2) + e] * r));
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
                    by_token[b] = pack4(static_cast<int>(rintf(c[0] * r)), static_cast<int>(rintf(c[1] * r)),
                                        static_cast<int>(rintf(c[2] * r)), static_cast<int>(rintf(c[3] * r)));
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
template <int D, typename T>
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
            append_block<D, T>(a, s, i, head, first, st);
            __syncthreads();
        }
    }
    append_block<D, T>(a, s, i, head, block, st);
}

// a.q_rows rows (token, query head) of q, kEach per group of D / 8 lanes in flight.
template <int D, typename T>
__device__ void turn_q(const AppendArgs &a, uint32_t unit) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes, kEach = 4;
    const int lane = threadIdx.x % kLanes;
    const bool interleaved = a.d.interleaved != 0;
    const Place at = place_of<D>(lane, a.d.rotary, interleaved);
    const uint32_t heads = a.d.q_heads;
    const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * heads, row_first = static_cast<uint64_t>(unit) * a.q_rows;
    // The workgroup's tokens are mostly of one sequence: the first one's.
    const Seq s0 = seq_of(a.batch, a.cache, token_seq(a.batch, static_cast<uint32_t>(row_first / heads)));
    for (uint32_t x0 = threadIdx.x / kLanes; x0 < a.q_rows; x0 += kEach * kRows) {
        Row r[kEach];
        Turn turn[kEach];
        uint32_t n[kEach], head[kEach];
        bool live[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const uint64_t row = row_first + x0 + x * kRows;
            live[x] = x0 + x * kRows < a.q_rows && row < rows;
            n[x] = live[x] ? static_cast<uint32_t>(row / heads) : 0;
            head[x] = live[x] ? static_cast<uint32_t>(row - static_cast<uint64_t>(n[x]) * heads) : 0;
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
            if (live[x]) load_turn(turn[x], at, a.d, s.past + static_cast<int>(n[x]) - s.first);
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            if (!live[x]) continue;
            if (a.d.q_norm != nullptr) norm_row<D>(r[x], at, a.d.q_norm, a.d.eps);
            turn_row(r[x], at, turn[x], interleaved);
            T *out = static_cast<T *>(a.d.q_out.data) + static_cast<int64_t>(n[x]) * a.d.q_out.token_stride +
                     head[x] * a.d.q_out.head_stride;
            store_floats<T, 4>(out + at.a_at, a.wide != 0, r[x].a);
            store_floats<T, 4>(out + at.b_at, a.wide != 0, r[x].b);
        }
    }
}

template <int D, typename T>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
    __shared__ AppendStage<D> stage;
    if (blockIdx.x < a.kv_units)
        append_place<D, T>(a, blockIdx.x, stage);
    else
        turn_q<D, T>(a, blockIdx.x - a.kv_units);
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

hipError_t launch_append(const AppendArgs &a, hipStream_t stream) {
    const uint32_t grid = a.kv_units + a.q_units;
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a); };
    if (a.cache.head_dim == 64)
        a.d.dtype == Q4RDNA_F32 ? go(append_kernel<64, float>) : a.d.dtype == Q4RDNA_F16 ? go(append_kernel<64, _Float16>) : go(append_kernel<64, __bf16>);
    else
        a.d.dtype == Q4RDNA_F32 ? go(append_kernel<128, float>) : a.d.dtype == Q4RDNA_F16 ? go(append_kernel<128, _Float16>) : go(append_kernel<128, __bf16>);
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
