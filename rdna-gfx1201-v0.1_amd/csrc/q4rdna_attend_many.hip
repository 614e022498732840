// Attention over the 8-bit paged cache for many rows (q4rdna_kv_attend on
// prompts): attend_many_kernel.
//
// A workgroup takes 128 rows (query token, query head of one kv head), 32 per
// wave, and walks the blocks they see.  Each block's int8 codes are loaded once
// per workgroup, become fp16 on their way into LDS (exact: |code| <= 127), and
// are multiplied by 32x32x16 fp16 matrix instructions:
//
//  * S^T = K q^T, then O^T += V^T p^T.  A lane holds one row of q: its scores
//    (32 of a block's 64; lane ^ 32 has the others) come out of the first
//    product in the registers that the second takes as its operand, since V^T
//    is laid into LDS in that order of tokens.  The row's maximum, sum and
//    rescaling are the lane's own, with one exchange between the halves.
//  * q is scaled by a power of two per row, so fp16 and bf16 rows are exact in
//    fp16.  Their weights are rounded to fp16 (11 bits), which the matrix
//    instruction needs, while their sum keeps them whole: each weight is off by as
//    much as an fp16 output is rounded by, an eighth of a bf16 output's rounding
//    (2048 tokens behind 6100 in bf16: 8 % of the outputs are a last place off those
//    of a plain fp32 form, the error against 64 bits is 1.67e-3, that one's 1.66e-3).
//    fp32 rows take two fp16 parts of q and of the weights each (SPLIT = 2, 22 bits)
//    and twice the products: the error is half of a plain fp32 form's (5.7e-7 and
//    1.1e-6 of the output at 2047 tokens).
//  * V's scale per block goes into the weights: they are relative to the largest
//    product of a weight and a V scale that the row has had, not to the largest
//    weight, so fp16's range is spent on what counts in the row's output, however
//    far the blocks' scales lie apart.  That largest and the scores' maximum are
//    the lane's own, followed lazily, by steps of at least 2^8.
//  * The open block's two planes are two tiles, high and low / 256, both exact in
//    fp16; so its codes are as large as a full block's, and its scales 256 times
//    the tokens' own.  Its weights refer to the largest product of a weight and a
//    scale among the tokens that the row sees.
//
// Row groups are split over several workgroups along the blocks when there are
// too few of them; the last to arrive joins the parts in a fixed order.
//
// 2048 tokens behind 6100 (bf16, 8 kv heads of four query heads of 128 numbers)
// take 271 us, 0.9 PFLOP/s where a large matrix product of the library reaches
// 1.2; 2047 tokens from the start in fp32, twice the products, 88 us.  Two
// workgroups share a CU (72 KB of LDS, 241 to 255 registers).  The matrix unit is busy
// 37 % of the time, the vector unit 54 %, the LDS 28 % without bank conflicts:
// a wave's products and its softmax follow each other, and two waves per SIMD
// overlap in part; one alone takes 1.5 us a block, two 2.15.  Of a block's 1500
// vector cycles 512 are exponentials, 320 the codes' conversion.  Reading the
// LDS right before each product, not D / 16 products ahead, cost a tenth.
// Without gain: the two products of half a block interleaved with the other
// half's softmax (spills), conversions between the second products, the sum by
// two-element dot products, wave priorities, long row groups in two parts.
#include "q4rdna_rows_device.h"

namespace q4rdna {
namespace {

constexpr int kRowsMany = kAttendManyRows;

// LDS tiles of a block in fp16: K [64 tokens][D + 8], V^T [D][64 + 8].  Rows
// are 272 (144) and 144 bytes: 16 lanes' 16-byte reads of 16 rows cover all
// 64 banks once.
template <int D>
struct ManyTile {
    _Float16 k[kKvBlock * (D + 8)];
    _Float16 v[D * (kKvBlock + 8)];
};

template <bool LOW>
__device__ __forceinline__ void piece_to_lds(_Float16 *at, i32x4 piece) {
    h16x2 x[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) codes_to_half(static_cast<uint32_t>(piece[w]), x[2 * w], x[2 * w + 1]);
    if (LOW) {
        const h16x2 f = {static_cast<_Float16>(0x1p-8f), static_cast<_Float16>(0x1p-8f)};
#pragma unroll
        for (int w = 0; w < 8; ++w) x[w] *= f;
    }
    h16x8 a, b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a[e] = x[e / 2][e % 2];
        b[e] = x[4 + e / 2][e % 2];
    }
    *reinterpret_cast<h16x8 *>(at) = a;
    *reinterpret_cast<h16x8 *>(at + 8) = b;
}
// A block's pieces `tid`, `tid + 256`, ... of K and V.
template <int D>
struct Raw {
    i32x4 k[D / 64], v[D / 64];
};
template <int D>
__device__ __forceinline__ void load_raw(Raw<D> &r, const int8_t *k, const int8_t *v) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        r.k[i] = load16(k + 16 * (threadIdx.x + 256 * i));
        r.v[i] = load16(v + 16 * (threadIdx.x + 256 * i));
    }
}
template <bool LOW, int D>
__device__ __forceinline__ void stage_raw(ManyTile<D> &t, const Raw<D> &r) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const int piece = threadIdx.x + 256 * i, c = piece % 16, g = piece / 16 % 4;
        const int token = piece / (64 * (D / 64)) * 16 + c, number = piece / 64 % (D / 64) * 64 + g * 16;
        piece_to_lds<LOW>(t.k + token * (D + 8) + number, r.k[i]);
        // Row d: [half of the wave][product][8 tokens]; a piece is one half's two products.
        piece_to_lds<LOW>(t.v + (piece / 64 * 16 + c) * (kKvBlock + 8) + (g & 1) * 32 + (g >> 1) * 16, r.v[i]);
    }
}

// One block from LDS.  OPEN: two tiles (high, low / 256), scales per token (kt,
// vt, of 16-bit codes); otherwise k_scale and v_scale.
template <bool OPEN, int D, int SPLIT>
__device__ __forceinline__ void many_block(ManyState<D, SPLIT> &st, const ManyTile<D> *tile, float k_scale, float v_scale,
                                           const float *token_scales, int start, uint32_t window, bool masked) {
    constexpr int KF = D / 16, VF = D / 32;  // fragments per product's tile
    const int lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
    const int k_at = column * (D + 8) + 8 * half, v_at = column * (kKvBlock + 8) + 32 * half;
    // The tile's fragments in the order of their use, the first DEPTH of them
    // under way: the registers of each are refilled once its product is issued.
    constexpr int ALL = 2 * KF + 4 * VF, DEPTH = SPLIT == 1 ? KF : KF / 2;
    const auto fragment = [&](int y, int j) {
        const _Float16 *k = tile[y].k + k_at + j / KF * 32 * (D + 8) + j % KF * 16;
        const _Float16 *v = tile[y].v + v_at + (j - 2 * KF) % VF * 32 * (kKvBlock + 8) + (j - 2 * KF) / VF * 8;
        return *reinterpret_cast<const h16x8 *>(j < 2 * KF ? k : v);
    };
    h16x8 f[DEPTH];
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) f[j] = fragment(0, j);
    const auto use = [&](int j, const h16x8 (&operand)[SPLIT], f32x16 &sum) {
#pragma unroll
        for (int x = 0; x < SPLIT; ++x) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[j % DEPTH], operand[x], sum, 0, 0, 0);
        if (j + DEPTH < ALL) f[j % DEPTH] = fragment(0, j + DEPTH);
        tile_end();
        if (OPEN) {
            const h16x8 low = fragment(1, j);
#pragma unroll
            for (int x = 0; x < SPLIT; ++x) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(low, operand[x], sum, 0, 0, 0);
        }
    };
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KF; ++k) use(t * KF + k, st.q[k], s[t]);
    }
    if (OPEN) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const f32x4 kt = *(gptr_f32x4)(uintptr_t)(token_scales + 8 * x + 4 * half);
#pragma unroll
            for (int b = 0; b < 4; ++b) s[x / 4][4 * (x % 4) + b] *= kt[b];
        }
    }
    // Token of s[t][i]: 32 t + 8 (i / 4) + 4 half + i % 4.
    // Of the lane's 32 tokens in this order, 8 x + b from start + 4 half on, the
    // first few are at or before a position: bit masks, a word for each score
    // (bit operations only; compares would take a pair of scalar registers each).
    uint32_t seen = 0xffffffffu;
    if (masked) {
        const int ahead = st.position - start - 4 * half;
        seen = first_tokens(ahead);
        if (window != 0) seen &= ~first_tokens(static_cast<int>(max(static_cast<int64_t>(ahead) - window, static_cast<int64_t>(-1))));
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t m = bit_mask(seen, 16 * t + i);
                s[t][i] = __uint_as_float((__float_as_uint(s[t][i]) & m) | (__float_as_uint(kNegInf) & ~m));
            }
    }
    const float unit = OPEN ? 256.0f * st.q_scale : st.q_scale * k_scale;
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    top = max_xor32(top);
    const bool none = top == kNegInf;
    const float now = none ? kNegInf : top * unit;

    auto hide = [&] {  // whatever the unit and the scales are
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = __uint_as_float(__float_as_uint(s[t][i]) & bit_mask(seen, 16 * t + i));
    };
    const auto exponentials = [&](float shift) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], unit, shift));
        if (masked) hide();
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += s[t][i];
        return sum;
    };
    if (OPEN) {
        // Weights of 2^8 at most times the scales, under 2^114, in fp32; the
        // largest of them is what the row refers to.
        const float m = now > st.m + kLazy ? now : st.m;
        const float sum = exponentials(m == kNegInf ? 0.0f : -m);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const f32x4 vt = *(gptr_f32x4)(uintptr_t)(token_scales + kKvBlock + 8 * x + 4 * half);
#pragma unroll
            for (int b = 0; b < 4; ++b) s[x / 4][4 * (x % 4) + b] *= vt[b] + (vt[b] - vt[b]);  // an infinite scale is made NaN
        }
        hide();
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, s[t][i]);
        refer(st, now, m + __builtin_amdgcn_logf(max_xor32(most)) + 8.0f);
        st.l += __builtin_amdgcn_ldexpf(sum, static_cast<int>(kWeight));
        // From units of 2^(m + 8) to the accumulators'.
        const int up = st.e == kNegInf ? 0 : 8 + static_cast<int>(kWeight) - static_cast<int>(st.e);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_ldexpf(s[t][i], up);
    } else {
        // The block's scale of V, 2^(v_exp + v_log), goes into the exponent, and comes out of the sum.
        const bool finite = v_scale < __builtin_inff();
        const float v_exp = static_cast<float>(__builtin_amdgcn_frexp_expf(v_scale));
        const float v_log = finite ? __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v_scale)) : __builtin_nanf("");
        refer(st, now, now + (v_exp + v_log));
        const float ratio = none ? 0.0f : finite ? fmaxf(v_log + (v_exp - st.e), kLeast) : __builtin_nanf("");
        const float sum = exponentials(kWeight - (st.m == kNegInf ? 0.0f : st.m) + ratio);
        st.l += sum * __builtin_amdgcn_exp2f(-ratio);
    }
    tile_end();
    // Products 2 parity + pair: tokens 16 a + 8 parity + 4 half + b, a = 2 pair, 2 pair + 1.
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        h16x8 p[SPLIT];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int a = 2 * (x & 1) + e / 4, eight = 2 * a + (x >> 1);
            const float w = s[eight / 4][4 * (eight % 4) + e % 4];
            p[0][e] = static_cast<_Float16>(w);
            if (SPLIT == 2) p[SPLIT - 1][e] = static_cast<_Float16>(w - static_cast<float>(p[0][e]));
        }
#pragma unroll
        for (int d = 0; d < VF; ++d) use(2 * KF + x * VF + d, p, st.o[d]);
    }
}

template <int D, int SPLIT, typename T>
__device__ __forceinline__ void load_q_many(ManyState<D, SPLIT> &st, const AttendArgs &a, const Seq &s, uint32_t head, int row,
                                            bool live) {
    const int half = (threadIdx.x & 63) >> 5;
    const int token = live ? row / static_cast<int>(a.group) : 0;
    const uint32_t h = head * a.group + (live ? row - token * a.group : 0);
    st.position = s.past + token;
    const T *p = static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(s.first + token) * a.d.q.token_stride +
                 h * a.d.q.head_stride + 8 * half;
    float x[D / 16][8];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
        load_floats<T, 8>(p + 16 * k, a.wide != 0, x[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
    }
    top = __float_as_uint(max_xor32(__uint_as_float(min(top, 0x7f800000u))));  // NaN as infinity
    const bool finite = top < 0x7f800000u;
    // The largest number of the row to 2^13 .. 2^14: small ones stay normal in fp16.
    const int up = finite && top != 0 ? 14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = finite ? __builtin_amdgcn_ldexpf(x[k][e], up) : 0.0f;
            st.q[k][0][e] = static_cast<_Float16>(v);
            if (SPLIT == 2) st.q[k][SPLIT - 1][e] = static_cast<_Float16>(v - static_cast<float>(st.q[k][0][e]));
        }
    st.q_scale = finite ? __builtin_amdgcn_ldexpf(a.d.scale * kLog2e, -up) : __builtin_nanf("");
    st.m = kNegInf;
    st.l = 0.0f;
    st.e = kNegInf;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[d][i] = 0.0f;
}

template <int D, int SPLIT, typename T>
__global__ __launch_bounds__(256, 2) void attend_many_kernel(const AttendArgs a) {
    __shared__ __align__(16) ManyTile<D> tiles[2];
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid & 63, column = lane & 31, half = lane >> 5, wave = wave_id();
    const uint32_t heads = a.cache.kv_heads;
    // Neighbouring workgroups take different heads: with eight of them, each
    // XCD's L2 holds one head's cache.  Late rows, which see most, go first;
    // the second workgroup of each CU (workgroups are placed in turn: i and
    // i + 256 share one) comes in the opposite order, so that the longest ones
    // share their CU with the shortest: 2047 tokens from the start 104 us, not 108.
    const uint32_t head = blockIdx.x % heads, units = gridDim.x / heads;
    uint32_t unit = blockIdx.x / heads;
    if (unit >= a.cu_units && unit < 2 * a.cu_units) unit = a.cu_units + min(2 * a.cu_units, units) - 1 - unit;
    const uint32_t late = unit / a.splits, place = units / a.splits - 1 - late;

    // The sequence and the rows of the place: sequence i has the places from
    // cu[i] * group / 128 + i on (attend_many_places).
    auto first_place = [&](uint32_t i) {
        return static_cast<int64_t>(a.batch.cu_tokens ? a.batch.cu_tokens[i] : static_cast<int>(i)) * a.group / kRowsMany + i;
    };
    const uint32_t seq = __builtin_amdgcn_readfirstlane(last_not_past(a.batch.sequences, place, first_place));
    const int64_t seq_place = first_place(seq);
    const uint32_t base = seq_place < 0 || seq_place > place ? place : static_cast<uint32_t>(seq_place);
    const Seq s = seq_of(a.batch, a.cache, seq);
    if (!s.ok) {
        // (With several sequences attend_few_kernel, which is launched too, counts them all.)
        if (a.few_rows == 0 && head == 0 && place == base && unit == late * a.splits && tid == 0) count_fault(a.cache);
        return;
    }
    const int rows = s.count * static_cast<int>(a.group);
    const int64_t first_row64 = static_cast<int64_t>(place - base) * kRowsMany;
    if (first_row64 >= rows || static_cast<uint32_t>(rows) <= a.few_rows) return;
    const int first_row = static_cast<int>(first_row64);
    const int last_row = min(first_row + kRowsMany, rows) - 1;
    const int group = static_cast<int>(a.group), block_size = static_cast<int>(kKvBlock);
    const int first_position = s.past + first_row / group, end = s.past + last_row / group + 1;
    const int begin = a.d.window != 0 && static_cast<uint32_t>(first_position) >= a.d.window
                          ? first_position - static_cast<int>(a.d.window) + 1 : 0;
    const int block0 = begin / block_size, blocks = (end + block_size - 1) / block_size - block0;
    // A part costs the joining workgroup about as long as a block costs a part:
    // blocks / splits + splits is least at the root.
    const int splits = min(static_cast<int>(a.splits), max(1, static_cast<int>(__builtin_amdgcn_sqrtf(static_cast<float>(blocks)))));
    const int split = static_cast<int>(unit - late * a.splits);
    if (split >= splits) return;
    const int from = block0 + static_cast<int>(mul_div(split, blocks, splits));
    const int to = block0 + static_cast<int>(mul_div(split + 1, blocks, splits));
    // The open block, where this workgroup has it, comes last.
    const bool has_open = s.length % block_size != 0 && to - 1 == s.length / block_size;
    const int to_full = has_open ? to - 1 : to;

    // This wave's rows.
    const int row = first_row + 32 * wave + column;
    ManyState<D, SPLIT> st;
    load_q_many<D, SPLIT, T>(st, a, s, head, row, row < rows);
    const int wave_first = s.past + min(first_row + 32 * wave, rows - 1) / group;
    const int wave_last = s.past + min(first_row + 32 * wave + 31, rows - 1) / group;

    const int32_t *table = a.batch.table + static_cast<size_t>(seq) * a.batch.table_width;
    constexpr size_t kPlane = kKvBlock * D;
    // Lane x keeps the page of the x-th of the next 64 blocks, so no load waits
    // for another one inside the loop.
    Raw<D> raw;
    f32x2 scale_next;
    bool bad_next;
    int pages = 0;
    auto load = [&](int b) {
        if ((b - from) % 64 == 0) pages = table[min(b + lane, to - 1)];
        int page = __builtin_amdgcn_readlane(pages, (b - from) % 64);
        bad_next = static_cast<uint32_t>(page) >= a.cache.page_count;
        if (bad_next) {
            if (tid == 0) count_fault(a.cache);
            page = 0;
        }
        const int8_t *t = a.cache.pages + page_tile(a.cache, page, head);
        scale_next = *(gptr_f32x2)(uintptr_t)(a.cache.scales + (static_cast<size_t>(page) * heads + head) * 2);
        load_raw<D>(raw, t, t + kPlane);
    };
    if (from < to_full) {
        load(from);
        stage_raw<false, D>(tiles[0], raw);
    }
    __syncthreads();
    for (int b = from; b < to_full; ++b) {
        const int buffer = (b - from) & 1, start = b * block_size;
        f32x2 scale = scale_next;
        if (bad_next) scale[0] = scale[1] = __builtin_nanf("");
        if (b + 1 < to_full) load(b + 1);
        const bool away = start > wave_last ||
                          (a.d.window != 0 && wave_first - (start + block_size - 1) >= static_cast<int64_t>(a.d.window));
        if (!away) {
            const bool masked = start + block_size - 1 > wave_first ||
                                (a.d.window != 0 && static_cast<uint32_t>(wave_last - start) >= a.d.window);
            many_block<false, D, SPLIT>(st, &tiles[buffer], scale[0], scale[1], nullptr, start, a.d.window, masked);
        }
        if (b + 1 < to_full) stage_raw<false, D>(tiles[buffer ^ 1], raw);
        __syncthreads();
    }
    if (has_open) {
        const int8_t *planes = a.cache.open + open_tile(a.cache, s.slot, to - 1, head);
        load_raw<D>(raw, planes, planes + 2 * kPlane);
        stage_raw<false, D>(tiles[0], raw);
        load_raw<D>(raw, planes + kPlane, planes + 3 * kPlane);
        stage_raw<true, D>(tiles[1], raw);
        __syncthreads();
        const int start = (to - 1) * block_size;
        if (start <= wave_last)
            many_block<true, D, SPLIT>(st, tiles, 0.0f, 0.0f,
                                       a.cache.open_scales + open_scale_row(a.cache, s.slot, to - 1, head), start,
                                       a.d.window, true);
    }

    // The row's sum over both halves; results in units of one.
    const float l = add_xor32(st.l);
    const bool live = row < rows;
    const int token = live ? row / group : 0;
    const uint32_t h = head * a.group + (live ? row - token * group : 0);
    const uint32_t job = place * heads + head;
    // Parts lie as [number][row]: a lane's row, so neighbouring lanes side by side.
    // The result's unit is 2^(factor's logarithm + up).
    float m_row = st.m, l_row = l, factor = 1.0f, up = st.e;
    if (splits > 1) {
        const size_t first_slot = static_cast<size_t>(job) * a.splits;
        float *stats = a.partials + static_cast<size_t>(gridDim.x) * kRowsMany * D;
        const int r = 32 * wave + column;
        float *part = a.partials + (first_slot + split) * kRowsMany * D + r;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                store_agent(part + (32 * d + 8 * (i / 4) + 4 * half + i % 4) * kRowsMany, st.o[d][i]);
        float *stat = stats + first_slot * 3 * kRowsMany + r;  // of part i: m, l and e at i * 3 * kRowsMany
        if (half == 0) {
            store_agent(stat + split * 3 * kRowsMany, st.m);
            store_agent(stat + split * 3 * kRowsMany + kRowsMany, l);
            store_agent(stat + split * 3 * kRowsMany + 2 * kRowsMany, st.e);
        }
        wait_stores();
        __syncthreads();
        if (tid == 0) ticket = add_agent(a.arrived + job, 1u);
        __syncthreads();
        if (ticket != static_cast<uint32_t>(splits - 1)) return;
        if (tid == 0) store_agent(a.arrived + job, 0u);
        // The last to arrive reads all parts, its own too, in their order: the
        // result does not depend on which one it was.
        m_row = kNegInf;
        up = kNegInf;
        float m_up = 0.0f;  // the part with the largest unit has m_up and up
        for (int i = 0; i < splits; ++i) {
            const float m = load_agent(stat + i * 3 * kRowsMany), e = load_agent(stat + i * 3 * kRowsMany + 2 * kRowsMany);
            m_row = fmaxf(m_row, m);
            if (m + e > m_up + up) {
                m_up = m;
                up = e;
            }
        }
        const float ref = m_row == kNegInf ? 0.0f : m_row;
        l_row = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[d][i] = 0.0f;
        for (int y = 0; y < splits; ++y) {
            const float m = load_agent(stat + y * 3 * kRowsMany), e = load_agent(stat + y * 3 * kRowsMany + 2 * kRowsMany);
            l_row += load_agent(stat + y * 3 * kRowsMany + kRowsMany) * __builtin_amdgcn_exp2f(m - ref);
            const float f = e == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((m - m_up) + (e - up));  // (such a part is zero)
            const float *from_part = a.partials + (first_slot + y) * kRowsMany * D + r;
            float v[D / 32][16];
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) v[d][i] = load_agent(from_part + (32 * d + 8 * (i / 4) + 4 * half + i % 4) * kRowsMany);
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) st.o[d][i] = fmaf(v[d][i], f, st.o[d][i]);
        }
        if (up != kNegInf) {  // m_up <= m_row: the difference's whole part goes to `up`
            const float whole = rintf(m_up - m_row);
            factor = __builtin_amdgcn_exp2f((m_up - m_row) - whole);
            up += whole;
        }
    }
    if (!live) return;
    const float inv = l_row == 0.0f ? 0.0f : factor / l_row;
    const int places = static_cast<int>(fminf(fmaxf(up, -400.0f), 400.0f));
    T *out = static_cast<T *>(a.d.out.data) + static_cast<int64_t>(s.first + token) * a.d.out.token_stride + h * a.d.out.head_stride;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(st.o[d][4 * x + e] * inv, places);
            store_floats<T, 4>(out + 32 * d + 8 * x + 4 * half, a.wide_out != 0, v);
        }
    if (a.d.lse != nullptr && half == 0)
        a.d.lse[static_cast<size_t>(s.first + token) * a.d.q_heads + h] = (m_row + log2f(l_row) - kWeight) * (1.0f / kLog2e);
}

}  // namespace

uint64_t attend_many_places(const q4rdna_kv_batch &b, uint32_t group) {
    return static_cast<uint64_t>(b.tokens) * group / kRowsMany + b.sequences;
}

hipError_t launch_attend_many(const AttendArgs &a, uint32_t places, hipStream_t stream) {
    const uint32_t grid = places * a.cache.kv_heads * a.splits;
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a); };
    if (a.cache.head_dim == 64)
        a.d.dtype == Q4RDNA_F32 ? go(attend_many_kernel<64, 2, float>) : a.d.dtype == Q4RDNA_F16 ? go(attend_many_kernel<64, 1, _Float16>) : go(attend_many_kernel<64, 1, __bf16>);
    else
        a.d.dtype == Q4RDNA_F32 ? go(attend_many_kernel<128, 2, float>) : a.d.dtype == Q4RDNA_F16 ? go(attend_many_kernel<128, 1, _Float16>) : go(attend_many_kernel<128, 1, __bf16>);
    return hipGetLastError();
}

}  // namespace q4rdna
