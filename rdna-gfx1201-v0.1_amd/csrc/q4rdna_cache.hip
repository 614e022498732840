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
__device__ __forceinline__ Row load_row(const T *row, const Place &p, bool wide) {
    Row r;
    load_floats<T, 4>(row + p.a_at, wide, r.a);
    load_floats<T, 4>(row + p.b_at, wide, r.b);
    return r;
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
__device__ __forceinline__ void turn_pair(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
    const float x = a * c - b * s;
    const float y = b * c + a * s;
    a = x;
    b = y;
}
__device__ __forceinline__ void turn_row(Row &r, const Place &p, const float *cos, const float *sin, size_t at,
                                         bool interleaved) {
    if (!p.turned) return;
    float c[4], s[4];
    load_floats<float, 4>(cos + at + p.pair, true, c);
    load_floats<float, 4>(sin + at + p.pair, true, s);
    if (interleaved) {
        turn_pair(r.a[0], r.a[1], c[0], s[0]);
        turn_pair(r.a[2], r.a[3], c[1], s[1]);
        turn_pair(r.b[0], r.b[1], c[2], s[2]);
        turn_pair(r.b[2], r.b[3], c[3], s[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) turn_pair(r.a[e], r.b[e], c[e], s[e]);
    }
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

    // Rows: the block's K rows, then its V rows, a group of D / 8 lanes each.
    const int lane = tid % kLanes;
    const bool interleaved = a.d.interleaved != 0;
    for (int row = tid / kLanes; row < 2 * fresh; row += kRows) {
        const bool is_v = row >= fresh;
        const int t = from + (is_v ? row - fresh : row);
        const size_t n = static_cast<size_t>(s.first) + (start + t - s.past);
        const q4rdna_kv_rows &src = is_v ? a.d.v : a.d.k;
        const T *p = static_cast<const T *>(src.data) + n * src.token_stride + head * src.head_stride;
        const Place at = place_of<D>(lane, is_v ? 0 : a.d.rotary, interleaved);
        Row r = load_row(p, at, a.wide != 0);
        if (!is_v) {
            if (a.d.k_norm != nullptr) norm_row<D>(r, at, a.d.k_norm, a.d.eps);
            turn_row(r, at, a.d.cos, a.d.sin, static_cast<size_t>(start + t) * (a.d.rotary / 2), interleaved);
        }
        // The largest magnitude by its bits: infinities and NaN come out on top.
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            top = max(top, max(__float_as_uint(r.a[e]) & 0x7fffffffu, __float_as_uint(r.b[e]) & 0x7fffffffu));
        top = lanes_max<kLanes>(top);
        const float largest = __uint_as_float(top);
        const bool finite = top < 0x7f800000u, some = finite && largest >= kKvZero;
        const float inv = some ? kKvCode16 / largest : 0.0f;
        short *out = &st.code[is_v][t * kRow<D>];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            out[at.a_at + e] = some ? static_cast<short>(static_cast<int>(rintf(r.a[e] * inv))) : 0;
            out[at.b_at + e] = some ? static_cast<short>(static_cast<int>(rintf(r.b[e] * inv))) : 0;
        }
        if (lane == 0) st.scale[is_v][t] = some ? largest / kKvCode16 : finite ? 0.0f : __builtin_nanf("");
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
    for (int piece = tid; piece < kPieces; piece += 256) {
        i32x4 k, v;
        const int t = k_token<D>(piece);
        const short *row = &st.code[0][t * kRow<D> + k_number<D>(piece)];
        const float r = st.ratio[0][t];
        const int number = v_number(piece);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t kw = 0, vw = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int vt = v_token(piece, 4 * w + e);
                kw |= (static_cast<uint32_t>(static_cast<int>(rintf(row[4 * w + e] * r))) & 255u) << (8 * e);
                vw |= (static_cast<uint32_t>(static_cast<int>(rintf(st.code[1][vt * kRow<D> + number] * st.ratio[1][vt]))) & 255u)
                      << (8 * e);
            }
            k[w] = static_cast<int>(kw);
            v[w] = static_cast<int>(vw);
        }
        store16(tile + 16 * piece, k);
        store16(tile + kPlane + 16 * piece, v);
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

// kAppendQRows rows (token, query head) of q.
template <int D, typename T>
__device__ void turn_q(const AppendArgs &a, uint32_t unit) {
    constexpr int kLanes = D / 8;
    const int lane = threadIdx.x % kLanes;
    const bool interleaved = a.d.interleaved != 0;
    const Place at = place_of<D>(lane, a.d.rotary, interleaved);
    const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * a.d.q_heads;
    for (uint32_t x = threadIdx.x / kLanes; x < kAppendQRows; x += 256 / kLanes) {
        const uint64_t row = static_cast<uint64_t>(unit) * kAppendQRows + x;
        if (row >= rows) return;
        const uint32_t n = static_cast<uint32_t>(row / a.d.q_heads), head = static_cast<uint32_t>(row - static_cast<uint64_t>(n) * a.d.q_heads);
        Row r = load_row(static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(n) * a.d.q.token_stride +
                             head * a.d.q.head_stride, at, a.wide != 0);
        const Seq s = seq_of(a.batch, a.cache, token_seq(a.batch, n));
        const int position = s.past + static_cast<int>(n) - s.first;
        if (!s.ok || static_cast<int>(n) < s.first || static_cast<int>(n) >= s.first + s.count ||
            (a.d.rotary != 0 && static_cast<uint32_t>(s.length) > a.d.positions))
            continue;  // its sequence is refused (and counted) as a whole
        if (a.d.q_norm != nullptr) norm_row<D>(r, at, a.d.q_norm, a.d.eps);
        turn_row(r, at, a.d.cos, a.d.sin, static_cast<size_t>(position) * (a.d.rotary / 2), interleaved);
        T *out = static_cast<T *>(a.d.q_out.data) + static_cast<int64_t>(n) * a.d.q_out.token_stride +
                 head * a.d.q_out.head_stride;
        store_floats<T, 4>(out + at.a_at, a.wide != 0, r.a);
        store_floats<T, 4>(out + at.b_at, a.wide != 0, r.b);
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

// One (sequence, block, kv head): its tokens past .. length - 1 as numbers.
template <int D, typename T>
__global__ __launch_bounds__(256) void read_kernel(const ReadArgs a) {
    constexpr int kPieces = kKvBlock * D / 16;
    __shared__ float values[kKvBlock * (D + 1)];
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
    constexpr size_t kPlane = kKvBlock * D;
    for (int which = 0; which < 2; ++which) {
        const int8_t *high = tile + (full ? which : 2 * which) * kPlane;
        __syncthreads();
        for (int piece = tid; piece < kPieces; piece += 256) {
            const i32x4 h = load16(high + 16 * piece);
            i32x4 l = {0, 0, 0, 0};
            if (!full) l = load16(high + kPlane + 16 * piece);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int t = which == 0 ? k_token<D>(piece) : v_token(piece, e);
                const int number = which == 0 ? k_number<D>(piece) + e : v_number(piece);
                const float x = full ? static_cast<float>(static_cast<int8_t>(static_cast<uint32_t>(h[e / 4]) >> (8 * (e % 4))))
                                     : static_cast<float>(join16(h, l, e));
                // An open block's scales past its length are not there.
                if (t >= from && t < to) values[t * (D + 1) + number] = x * (full ? scales[which] + bad : scales[which * 64 + t]);
            }
        }
        __syncthreads();
        const q4rdna_kv_rows &dst = which == 0 ? a.k : a.v;
        for (int x = tid; x < (to - from) * D; x += 256) {
            const int t = from + x / D, number = x % D;
            const int64_t n = static_cast<int64_t>(s.first) + (start + t - s.past);
            static_cast<T *>(dst.data)[n * dst.token_stride + head * dst.head_stride + number] =
                static_cast<T>(values[t * (D + 1) + number]);
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
