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
// So no wave waits for another before the end.  Up to 32 rows the workgroup's
// four waves take different blocks, up to 64 two and two of them, and with more
// rows each has its own 32 and they read the same blocks side by side.
//
// The drafted tokens are one more block.  The workgroup lays their rows into LDS
// in fp16, scaled by a power of two for each token, fp32 ones in two parts; a
// row's mask is 64 bits.
//
// A sequence's blocks are split over workgroups, dealt by the sequences' lengths,
// and joined by the last one to arrive, in a fixed order.
#include "q4rdna_rows_device.h"

namespace q4rdna {
namespace {

constexpr int kWaves = 4, kTreeThreads = 64 * kWaves;
constexpr int kBlock = static_cast<int>(kKvBlock);

template <int D>
struct TreeTile {  // as attend_many_kernel's
    _Float16 k[kKvBlock * (D + 8)];
    _Float16 v[D * (kKvBlock + 8)];
};
template <int D, int SPLIT>
struct TreeStage {
    TreeTile<D> part[SPLIT];
    float k_scale[kKvBlock], v_scale[kKvBlock];
};
template <int D>
struct TreeJoin {
    float o[kWaves][32][D + 4];
    float m[kWaves][32], l[kWaves][32], e[kWaves][32];
};

// Rows of K and V of a block as they lie in memory.
template <int D>
struct TreeRaw {
    i32x4 k[2][D / 32];  // [32 tokens][32 numbers]
    i32x4 v[D / 32][2];  // [32 numbers][tokens with bit 3 clear, set]
};
template <int D>
__device__ __forceinline__ void load_k(TreeRaw<D> &r, const int8_t *tile) {
    const int lane = threadIdx.x & 63;
    const int8_t *p = tile + (lane & 31) / 16 * (D / 64 * 1024) + (lane >> 5) * 256 + (lane & 15) * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) r.k[t][x] = load16(p + t * (D / 64 * 2048) + x / 2 * 1024 + x % 2 * 512);
}
template <int D>
__device__ __forceinline__ void load_v(TreeRaw<D> &r, const int8_t *tile) {
    const int lane = threadIdx.x & 63;
    const int8_t *p = tile + (lane & 31) / 16 * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int y = 0; y < 2; ++y) r.v[d][y] = load16(p + d * 2048 + y * 512);
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
template <int D, int SPLIT, typename K>
__device__ __forceinline__ void add_scores(const ManyState<D, SPLIT> &st, f32x16 (&s)[2], K fragment) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int f = 0; f < D / 16; ++f) {
            const h16x8 k = fragment(t, f);
#pragma unroll
            for (int x = 0; x < SPLIT; ++x) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, st.q[f][x], s[t], 0, 0, 0);
        }
}
// o += the products of V's fragments (32 numbers d; tokens 16 a + 8 y + 4 half + b,
// a = 2 pair, 2 pair + 1) with the weights.
template <int D, int SPLIT, typename V>
__device__ __forceinline__ void add_rows(ManyState<D, SPLIT> &st, const f32x16 (&s)[2], V fragment) {
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
            h16x8 p[SPLIT];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int eight = 2 * (2 * pair + e / 4) + y;
                const float w = s[eight / 4][4 * (eight % 4) + e % 4];
                p[0][e] = static_cast<_Float16>(w);
                if (SPLIT == 2) p[SPLIT - 1][e] = static_cast<_Float16>(w - static_cast<float>(p[0][e]));
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const h16x8 v = fragment(d, y, pair);
#pragma unroll
                for (int x = 0; x < SPLIT; ++x) st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[x], st.o[d], 0, 0, 0);
            }
        }
}
__device__ __forceinline__ void clear(f32x16 (&s)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
}
// `instead` where a bit is clear.
__device__ __forceinline__ void hide(f32x16 (&s)[2], uint32_t seen, float instead) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t m = bit_mask(seen, 16 * t + i);
            s[t][i] = __uint_as_float((__float_as_uint(s[t][i]) & m) | (__float_as_uint(instead) & ~m));
        }
}
__device__ __forceinline__ float largest(const f32x16 (&s)[2]) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    return max_xor32(top);
}
// Scores to weights: s = 2^(s * unit + shift), zero where hidden; their sum.
__device__ __forceinline__ float exponentials(f32x16 (&s)[2], float unit, float shift, uint32_t seen, bool masked) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], unit, shift));
    if (masked) hide(s, seen, 0.0f);
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += s[t][i];
    return sum;
}

// The softmax of a full block: integer products to weights in the accumulators'
// units, V's scale among them.
template <int D, int SPLIT>
__device__ __forceinline__ void soften_block(ManyState<D, SPLIT> &st, f32x16 (&s)[2], float k_scale, float v_scale, uint32_t seen,
                                             bool masked) {
    if (masked) hide(s, seen, kNegInf);
    const float unit = st.q_scale * k_scale, top = largest(s);
    const bool none = top == kNegInf;
    const float now = none ? kNegInf : top * unit;
    // The block's scale of V, 2^(v_exp + v_log), goes into the exponent, and comes out of the sum.
    const bool finite = v_scale < __builtin_inff();
    const float v_exp = static_cast<float>(__builtin_amdgcn_frexp_expf(v_scale));
    const float v_log = finite ? __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v_scale)) : __builtin_nanf("");
    refer(st, now, now + (v_exp + v_log));
    const float ratio = none ? 0.0f : finite ? fmaxf(v_log + (v_exp - st.e), kLeast) : __builtin_nanf("");
    const float sum = exponentials(s, unit, kWeight - (st.m == kNegInf ? 0.0f : st.m) + ratio, seen, masked);
    st.l += sum * __builtin_amdgcn_exp2f(-ratio);
}
// The same with scales per token: `unit_log` is 8 for 16-bit codes, whose tiles
// are in units of 256 times the scales.
template <int D, int SPLIT, typename Scales>
__device__ __forceinline__ void soften_tokens(ManyState<D, SPLIT> &st, f32x16 (&s)[2], int unit_log, uint32_t seen, Scales scales) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const f32x4 kt = scales(0, x);
#pragma unroll
        for (int b = 0; b < 4; ++b) s[x / 4][4 * (x % 4) + b] *= kt[b];
    }
    hide(s, seen, kNegInf);
    const float unit = __builtin_amdgcn_ldexpf(st.q_scale, unit_log), top = largest(s);
    const float now = top == kNegInf ? kNegInf : top * unit;
    // Weights of 2^8 at most times the scales, under 2^122, in fp32; the largest
    // of them is what the row refers to.
    const float m = now > st.m + kLazy ? now : st.m;
    const float sum = exponentials(s, unit, m == kNegInf ? 0.0f : -m, seen, true);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const f32x4 vt = scales(1, x);
#pragma unroll
        for (int b = 0; b < 4; ++b) s[x / 4][4 * (x % 4) + b] *= vt[b] + (vt[b] - vt[b]);  // an infinite scale is made NaN
    }
    hide(s, seen, 0.0f);
    float most = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[t][i]);
    refer(st, now, m + __builtin_amdgcn_logf(max_xor32(most)) + static_cast<float>(unit_log));
    st.l += __builtin_amdgcn_ldexpf(sum, static_cast<int>(kWeight));
    // From units of 2^(m + unit_log) to the accumulators'.
    const int up = st.e == kNegInf ? 0 : unit_log + static_cast<int>(kWeight) - static_cast<int>(st.e);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_ldexpf(s[t][i], up);
}

// Rows of q, the numbers of a fragment f in the order in which K's pieces have
// them: 64 (f / 4) + 32 (f / 2 % 2) + 16 half + 8 (f % 2) and on.
__device__ __forceinline__ int fragment_number(int f, int half) { return f / 4 * 64 + f / 2 % 2 * 32 + 16 * half + f % 2 * 8; }
template <int D, int SPLIT, typename T>
__device__ __forceinline__ void load_rows(ManyState<D, SPLIT> &st, const T *row, bool wide, float scale) {
    const int half = (threadIdx.x & 63) >> 5;
    float x[D / 16][8];
    uint32_t top = 0;
#pragma unroll
    for (int f = 0; f < D / 16; ++f) {
        load_floats<T, 8>(row + fragment_number(f, half), wide, x[f]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[f][e]) & 0x7fffffffu);
    }
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

// The drafted tokens' K and V into LDS: a thread takes eight numbers of four
// tokens, D / 8 threads side by side a row.
template <int D, int SPLIT, typename T>
__device__ __forceinline__ void stage_drafts(TreeStage<D, SPLIT> &stage, const TreeArgs &a, int first, int count, uint32_t head) {
    constexpr int kOctets = D / 8;
    const int tid = threadIdx.x, octet = tid % kOctets, quad = tid / kOctets;
    if (quad >= kBlock / 4) return;
    float x[2][4][8];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const q4rdna_kv_rows &rows = which == 0 ? a.d.k : a.d.v;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (4 * quad + b < count) {
                load_floats<T, 8>(static_cast<const T *>(rows.data) + static_cast<int64_t>(first + 4 * quad + b) * rows.token_stride +
                                      head * rows.head_stride + 8 * octet, a.wide != 0, x[which][b]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[which][b][e] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[which][b][e]) & 0x7fffffffu);
            top = lanes_max<kOctets>(top);
            const bool finite = top < 0x7f800000u;
            // The largest to 2^13 .. 2^14, but for numbers under 2^-96: the scale stays a normal number.
            const int up = finite && top != 0 ? min(14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)), 110) : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[which][b][e] = finite ? __builtin_amdgcn_ldexpf(x[which][b][e], up) : 0.0f;
            if (octet == 0) (which == 0 ? stage.k_scale : stage.v_scale)[4 * quad + b] = finite ? __builtin_amdgcn_ldexpf(1.0f, -up) : __builtin_nanf("");
        }
    typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int part = 0; part < SPLIT; ++part) {
        TreeTile<D> &tile = stage.part[part];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            h16x8 k;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[e] = static_cast<_Float16>(x[0][b][e]);
                x[0][b][e] -= static_cast<float>(k[e]);
            }
            *reinterpret_cast<h16x8 *>(tile.k + (4 * quad + b) * (D + 8) + 8 * octet) = k;
        }
        // Row d of V: the tokens in the order of the lanes' scores.
        const int at = (quad & 1) * 32 + (quad >> 1 & 1) * 16 + (quad >> 2) * 4;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h16x4 v;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                v[b] = static_cast<_Float16>(x[1][b][e]);
                x[1][b][e] -= static_cast<float>(v[b]);
            }
            *reinterpret_cast<h16x4 *>(tile.v + (8 * octet + e) * (kBlock + 8) + at) = v;
        }
    }
}

// One sequence of a step: as seq_of, but its tokens are not in the cache.
__device__ __forceinline__ Seq draft_seq(const TreeArgs &a, uint32_t i) {
    Seq s;
    s.first = a.batch.cu_tokens ? a.batch.cu_tokens[i] : static_cast<int>(i);
    const int end = a.batch.cu_tokens ? a.batch.cu_tokens[i + 1] : static_cast<int>(i) + 1;
    s.past = a.batch.past[i];
    s.slot = a.batch.slots ? a.batch.slots[i] : static_cast<int>(i);
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

// What a sequence's workgroups take: each row group of each head is cut into
// parts of about `chunk` of its units, the cached blocks and the drafts.
struct TreeWork {
    Seq s;
    uint32_t jobs, units;
};
__device__ __forceinline__ TreeWork tree_work(const TreeArgs &a, uint32_t rows, uint32_t i) {
    TreeWork w;
    w.jobs = w.units = 0;
    w.s = draft_seq(a, min(i, a.batch.sequences - 1));
    if (i >= a.batch.sequences || !w.s.ok || w.s.count == 0) return w;
    w.jobs = (w.s.count * a.group + rows - 1) / rows * a.cache.kv_heads;
    w.units = (w.s.past + kBlock - 1) / kBlock - first_block(a, w.s.past) + 1;
    return w;
}
__device__ __forceinline__ uint32_t tree_parts(const TreeArgs &a, uint32_t units, uint32_t chunk) {
    chunk = max(chunk, a.least);
    return min((units + chunk - 1) / chunk, a.splits);
}

struct TreeItem {
    int seq;  // -1: nothing
    Seq s;
    uint32_t head, row_group;
    int split, splits;
    uint32_t first, step;  // workgroup of part 0; part i is `step` * i further on
};
// The item of workgroup x: the device knows the lengths, the host does not, so
// every wave adds up the sequences' parts, 64 at a time.
__device__ __forceinline__ TreeItem find_tree_item(const TreeArgs &a, uint32_t rows, uint32_t x) {
    TreeItem it;
    it.seq = -1;
    const int lane = threadIdx.x & 63;
    const uint32_t heads = a.cache.kv_heads;
    if (a.splits == 1) {  // as many workgroups as there may be row groups
        const uint32_t per = a.row_groups * heads;
        it.seq = static_cast<int>(x / per);
        it.s = draft_seq(a, x / per);
        it.row_group = x % per / heads;
        it.head = x % heads;
        it.split = 0;
        it.splits = 1;
        it.first = x;
        it.step = 1;
        return it;
    }
    TreeWork w;
    uint32_t all = 0;  // jobs * units, fewer than 2^32 by the host's bound
    for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
        w = tree_work(a, rows, i + lane);
        all += __builtin_amdgcn_readlane(wave_scan(w.jobs * w.units), 63);
    }
    const uint32_t chunk = (all - 1) / a.target + 1;
    uint32_t base = 0;
    for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
        if (a.batch.sequences > 64) w = tree_work(a, rows, i + lane);
        const uint32_t parts = tree_parts(a, w.units, chunk), end = base + wave_scan(w.jobs * parts);
        const uint64_t later = __builtin_amdgcn_ballot_w64(end > x);
        if (later != 0) {
            const int owner = __builtin_ctzll(later);
            const uint32_t mine = __builtin_amdgcn_readlane(parts, owner);
            const uint32_t local = x - __builtin_amdgcn_readlane(end - w.jobs * parts, owner);  // (row group, part, head)
            it.seq = static_cast<int>(i) + owner;
            it.s.first = __builtin_amdgcn_readlane(w.s.first, owner);
            it.s.count = __builtin_amdgcn_readlane(w.s.count, owner);
            it.s.past = __builtin_amdgcn_readlane(w.s.past, owner);
            it.s.slot = __builtin_amdgcn_readlane(w.s.slot, owner);
            it.s.length = it.s.past;
            it.s.ok = true;
            it.head = local % heads;
            it.split = static_cast<int>(local / heads % mine);
            it.row_group = local / heads / mine;
            it.splits = static_cast<int>(mine);
            it.step = heads;
            it.first = x - it.split * heads;
            return it;
        }
        base = __builtin_amdgcn_readlane(end, 63);
    }
    return it;
}

// Parts of one row joined: its maximum m, the accumulators' exponent e (a whole
// number) and its sum l, in units of 2^(m - 7).
struct Joined {
    float m, l, e;
};
__device__ __forceinline__ float part_factor(const Joined &j, float m, float e) {  // (a part without e is zero, or NaN)
    return e == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((m - j.m) + (e - j.e));
}
template <typename Stat>
__device__ __forceinline__ Joined join(int parts, Stat stat) {
    Joined j = {kNegInf, 0.0f, kNegInf};
    for (int i = 0; i < parts; ++i) j.m = fmaxf(j.m, stat(i).m);
    const float ref = j.m == kNegInf ? 0.0f : j.m;
    for (int i = 0; i < parts; ++i) {
        const Joined s = stat(i);
        if (s.e != kNegInf) j.e = fmaxf(j.e, ceilf((s.m - ref) + s.e));
        j.l += s.l * __builtin_amdgcn_exp2f(s.m - ref);
    }
    return j;
}

// RW of the four waves have different rows, 4 / RW different blocks.
template <int D, int SPLIT, int RW, typename T>
__global__ __launch_bounds__(kTreeThreads, SPLIT == 1 ? 2 : 1) void attend_tree_kernel(const TreeArgs a) {
    constexpr int BW = kWaves / RW, ROWS = 32 * RW;
    __shared__ __align__(16) union Shared {
        TreeStage<D, SPLIT> stage;
        TreeJoin<D> join;
    } shared;
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid & 63, column = lane & 31, half = lane >> 5, wave = wave_id();
    const int row_wave = wave % RW, block_wave = wave / RW;
    const TreeItem it = find_tree_item(a, ROWS, blockIdx.x);
    if (blockIdx.x == 0)  // bad entries, once
        for (uint32_t i = tid; i < a.batch.sequences; i += kTreeThreads)
            if (!draft_seq(a, i).ok) count_fault(a.cache);
    if (it.seq < 0 || !it.s.ok) return;
    const uint32_t head = it.head;
    const Seq &s = it.s;
    const int group = static_cast<int>(a.group), rows = s.count * group;
    const int first_row = static_cast<int>(it.row_group) * ROWS;
    if (first_row >= rows) return;
    // Units: the cached blocks from block0 on, full ones, then the open one, then the drafts.
    const int block0 = first_block(a, s.past), full_blocks = s.past / kBlock;
    const int units = (s.past + kBlock - 1) / kBlock - block0 + 1;
    const int splits = min(it.splits, units), split = it.split;
    if (split >= splits) return;
    const int from = block0 + static_cast<int>(mul_div(split, units, splits));
    const int to = block0 + static_cast<int>(mul_div(split + 1, units, splits));
    const int drafts = block0 + units - 1;
    const bool has_drafts = drafts < to;
    const auto mine = [&](int unit) { return unit >= from && unit < to && (unit - from) % BW == block_wave; };

    // This wave's rows.
    const int row = first_row + 32 * row_wave + column;
    const bool live = row < rows;
    const int token = live ? row / group : 0;
    const uint32_t h = head * a.group + (live ? row - token * group : 0);
    ManyState<D, SPLIT> st;

    // The wave's full blocks: from + block_wave + BW n.  Lane x keeps the page of
    // the x-th of the next 64.
    const int32_t *table = a.batch.table + static_cast<size_t>(it.seq) * a.batch.table_width;
    const int start = from + block_wave, full_to = min(to, full_blocks);
    const int full = full_to > start ? (full_to - start + BW - 1) / BW : 0;
    constexpr size_t kPlane = kKvBlock * D;
    TreeRaw<D> raw;
    f32x2 scale_next = {0.0f, 0.0f};
    bool bad_next = false;
    int pages = 0;
    const int8_t *tile = nullptr;
    const auto next = [&](int n) {
        if (n % 64 == 0) pages = table[min(start + BW * (n + lane), full_to - 1)];
        int page = __builtin_amdgcn_readlane(pages, n % 64);
        bad_next = static_cast<uint32_t>(page) >= a.cache.page_count;
        if (bad_next) {
            if (lane == 0) count_fault(a.cache);
            page = 0;
        }
        tile = a.cache.pages + page_tile(a.cache, page, head);
        scale_next = *(gptr_f32x2)(uintptr_t)(a.cache.scales + (static_cast<size_t>(page) * a.cache.kv_heads + head) * 2);
    };
    if (full > 0) next(0);
    // What the row sees of the drafts, and where it stands.
    const uint64_t there = s.count >= 64 ? ~0ull : (1ull << s.count) - 1;
    uint64_t seen = a.d.seen[s.first + token] & there;
    const int depth = __builtin_popcountll(seen);
    load_rows<D, SPLIT, T>(st, static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(s.first + token) * a.d.q.token_stride +
                                   h * a.d.q.head_stride, a.wide != 0, a.d.scale);
    st.position = s.past - 1 + depth;
    if (full > 0) {
        load_k(raw, tile);
        load_v(raw, tile + kPlane);
    }
    if (has_drafts) {  // the same for the whole workgroup
        stage_drafts<D, SPLIT, T>(shared.stage, a, s.first, s.count, head);
        __syncthreads();
    }
    // Of the lane's 32 tokens of a block, in the order of its scores: those cached and within the window.
    const auto seen_from = [&](int first) {
        const int ahead = s.past - 1 - first - 4 * half;
        uint32_t bits = first_tokens(ahead);
        if (a.d.window != 0) {
            const int64_t behind = static_cast<int64_t>(st.position) - first - 4 * half - a.d.window;
            bits &= ~first_tokens(static_cast<int>(max(behind, static_cast<int64_t>(-1))));
        }
        return bits;
    };

    f32x16 sc[2];
    for (int n = 0; n < full; ++n) {
        const int first = (start + BW * n) * kBlock;
        const f32x2 scale = scale_next;
        const float k_scale = bad_next ? __builtin_nanf("") : scale[0], v_scale = bad_next ? __builtin_nanf("") : scale[1];
        // No row stands behind past + 63.
        const bool masked = a.d.window != 0 && static_cast<int64_t>(s.past) + 63 - first >= static_cast<int64_t>(a.d.window);
        clear(sc);
        add_scores(st, sc, [&](int t, int f) { return half_piece<false>(raw.k[t][f / 2], f % 2); });
        tile_end();
        if (n + 1 < full) {
            next(n + 1);
            load_k(raw, tile);
        }
        tile_end();
        soften_block(st, sc, k_scale, v_scale, masked ? seen_from(first) : 0xffffffffu, masked);
        tile_end();
        add_rows(st, sc, [&](int d, int y, int pair) { return half_piece<false>(raw.v[d][y], pair); });
        tile_end();
        if (n + 1 < full) load_v(raw, tile + kPlane);
        tile_end();
    }
    if (s.past % kBlock != 0 && mine(full_blocks)) {
        const int8_t *planes = a.cache.open + open_tile(a.cache, s.slot, full_blocks, head);
        const float *scales = a.cache.open_scales + open_scale_row(a.cache, s.slot, full_blocks, head);
        clear(sc);
        load_k(raw, planes);
        add_scores(st, sc, [&](int t, int f) { return half_piece<false>(raw.k[t][f / 2], f % 2); });
        load_k(raw, planes + kPlane);
        load_v(raw, planes + 2 * kPlane);
        add_scores(st, sc, [&](int t, int f) { return half_piece<true>(raw.k[t][f / 2], f % 2); });
        soften_tokens(st, sc, 8, seen_from(full_blocks * kBlock), [&](int which, int x) {
            return *(gptr_f32x4)(uintptr_t)(scales + kBlock * which + 8 * x + 4 * half);
        });
        add_rows(st, sc, [&](int d, int y, int pair) { return half_piece<false>(raw.v[d][y], pair); });
        load_v(raw, planes + 3 * kPlane);
        add_rows(st, sc, [&](int d, int y, int pair) { return half_piece<true>(raw.v[d][y], pair); });
    }
    if (mine(drafts)) {
        if (a.d.window != 0 && a.d.window < 64) {  // drafted tokens that lie too far above
            const int depths = __builtin_popcountll(a.d.seen[s.first + min(lane, s.count - 1)] & there);
            for (int j = 0; j < s.count; ++j)
                if (__builtin_amdgcn_readlane(depths, j) + static_cast<int>(a.d.window) <= depth) seen &= ~(1ull << j);
        }
        uint32_t bits = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) bits |= (static_cast<uint32_t>(seen >> (8 * x + 4 * half)) & 15u) << (4 * x);
        clear(sc);
#pragma unroll
        for (int part = 0; part < SPLIT; ++part)
            add_scores(st, sc, [&](int t, int f) {
                return *reinterpret_cast<const h16x8 *>(shared.stage.part[part].k + (32 * t + column) * (D + 8) + fragment_number(f, half));
            });
        soften_tokens(st, sc, 0, bits, [&](int which, int x) {
            return *reinterpret_cast<const f32x4 *>((which == 0 ? shared.stage.k_scale : shared.stage.v_scale) + 8 * x + 4 * half);
        });
#pragma unroll
        for (int part = 0; part < SPLIT; ++part)
            add_rows(st, sc, [&](int d, int y, int pair) {
                return *reinterpret_cast<const h16x8 *>(shared.stage.part[part].v + (32 * d + column) * (kBlock + 8) + 32 * half + 16 * y + 8 * pair);
            });
    }

    // The waves' rows meet in LDS.
    __syncthreads();
    TreeJoin<D> &j = shared.join;
    const float l_row = add_xor32(st.l);
    if (half == 0) {
        j.m[wave][column] = st.m;
        j.l[wave][column] = l_row;
        j.e[wave][column] = st.e;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4 *>(&j.o[wave][column][32 * d + 8 * x + 4 * half]) =
                f32x4{st.o[d][4 * x], st.o[d][4 * x + 1], st.o[d][4 * x + 2], st.o[d][4 * x + 3]};
    __syncthreads();
    const int live_rows = min(ROWS, rows - first_row);
    const auto finish = [&](int r, int d, const Joined &w, f32x4 o) {
        const int of = first_row + r, n = s.first + of / group;
        const uint32_t to_head = head * a.group + of % group;
        const float inv = w.l == 0.0f ? 0.0f : 1.0f / w.l;
        const int places = static_cast<int>(fminf(fmaxf(w.e, -400.0f), 400.0f));
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(o[e] * inv, places);
        store_floats<T, 4>(static_cast<T *>(a.d.out.data) + static_cast<int64_t>(n) * a.d.out.token_stride + to_head * a.d.out.head_stride + d,
                           a.wide_out != 0, v);
        if (d == 0 && a.d.lse != nullptr)
            a.d.lse[static_cast<size_t>(n) * a.d.q_heads + to_head] = (w.m + log2f(w.l) - kWeight) * (1.0f / kLog2e);
    };
    float *stats = a.partials + static_cast<size_t>(gridDim.x) * ROWS * D;  // [workgroup][row][m, l, e]
    for (int x = tid; x < live_rows * (D / 4); x += kTreeThreads) {
        const int r = x / (D / 4), d = x % (D / 4) * 4, rw = r / 32, c = r % 32;
        const Joined w = join(BW, [&](int i) { return Joined{j.m[RW * i + rw][c], j.l[RW * i + rw][c], j.e[RW * i + rw][c]}; });
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < BW; ++i)
            o += *reinterpret_cast<const f32x4 *>(&j.o[RW * i + rw][c][d]) * part_factor(w, j.m[RW * i + rw][c], j.e[RW * i + rw][c]);
        if (splits == 1) {
            finish(r, d, w, o);
            continue;
        }
        float *to_part = a.partials + (static_cast<size_t>(blockIdx.x) * ROWS + r) * D + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) store_agent(to_part + e, o[e]);
        if (d == 0) {
            float *stat = stats + (static_cast<size_t>(blockIdx.x) * ROWS + r) * 3;
            store_agent(stat, w.m);
            store_agent(stat + 1, w.l);
            store_agent(stat + 2, w.e);
        }
    }
    if (splits == 1) return;

    // The last workgroup of the row group joins the parts, in their order.
    wait_stores();
    __syncthreads();
    uint32_t *arrived = a.arrived + (static_cast<size_t>(it.seq) * a.row_groups + it.row_group) * a.cache.kv_heads + head;
    if (tid == 0) ticket = add_agent(arrived, 1u);
    __syncthreads();
    if (ticket != static_cast<uint32_t>(splits - 1)) return;
    if (tid == 0) store_agent(arrived, 0u);
    const auto slot = [&](int i, int r) { return (static_cast<size_t>(it.first) + static_cast<size_t>(i) * it.step) * ROWS + r; };
    for (int x = tid; x < live_rows * (D / 4); x += kTreeThreads) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        const auto stat = [&](int i) {
            const float *p = stats + slot(i, r) * 3;
            return Joined{load_agent(p), load_agent(p + 1), load_agent(p + 2)};
        };
        const Joined w = join(splits, stat);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < splits; ++i) {
            const float *p = a.partials + slot(i, r) * D + d;
            const f32x2 lo = load_agent2(p), hi = load_agent2(p + 2);
            const Joined q = stat(i);
            o += f32x4{lo[0], lo[1], hi[0], hi[1]} * part_factor(w, q.m, q.e);
        }
        finish(r, d, w, o);
    }
}

}  // namespace

template <int SPLIT, int RW, typename T>
static void launch_tree_as(const TreeArgs &a, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<a.workgroups, kTreeThreads, 0, stream>>>(a); };
    a.cache.head_dim == 64 ? go(attend_tree_kernel<64, SPLIT, RW, T>) : go(attend_tree_kernel<128, SPLIT, RW, T>);
}
template <int SPLIT, typename T>
static void launch_tree_as(const TreeArgs &a, hipStream_t stream) {
    a.row_waves == 1 ? launch_tree_as<SPLIT, 1, T>(a, stream)
                     : a.row_waves == 2 ? launch_tree_as<SPLIT, 2, T>(a, stream) : launch_tree_as<SPLIT, 4, T>(a, stream);
}
hipError_t launch_attend_tree(const TreeArgs &a, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_tree_as<2, float>(a, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_tree_as<1, _Float16>(a, stream);
    else launch_tree_as<1, __bf16>(a, stream);
    return hipGetLastError();
}

}  // namespace q4rdna
