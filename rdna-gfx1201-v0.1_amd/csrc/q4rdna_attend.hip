// Attention over the 8-bit paged cache (q4rdna_kv_attend).
//
// attend_few_kernel: few rows (query token, query head) per kv head, the
// decode form.  It streams the cache once and multiplies by the int8 codes as
// they lie in memory, with no conversion:
//
//  * A row of q becomes 32-bit fixed point relative to its largest number, as
//    four balanced base-256 digits, so q . k is four int8 dot products, exact
//    in int32.  The digits of four rows fill the 16 columns of a 16x16x64 int8
//    matrix instruction (column 4 r + digit), which is what a group of four
//    query heads needs; a tile of K is its other operand straight from memory.
//  * Its results S^T lie as (token, column): the four lanes of a quad hold a
//    row's digits, two DPP adds join them, and each lane then holds 16 of the
//    64 scores of its row -- in the k order that the second product's operand
//    has, so the weights p never leave their lanes.  They become 30-bit fixed
//    point relative to the block's largest and the lane keeps its digit's byte.
//  * O^T += V^T p by the same instruction, and each lane scales its digit's
//    int32 sums into fp32 accumulators (the digits are joined once at the end).
//
// Each wave keeps its own running maximum and sum (base 2) over the blocks it
// takes; a workgroup's four waves, then the workgroups that share a row group,
// are joined by those.  The last workgroup to arrive joins them, in a fixed
// order, so results do not depend on the order of arrival.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kWaves = 4;

// Four int32 values as balanced base-256 digits: byte d of (x + 0x808080) ^
// 0x808080 is digit d in [-128, 127].  Returns byte `digit` of each, packed;
// `pick` is digit | (4 + digit) << 8.
__device__ __forceinline__ int digits4(int x0, int x1, int x2, int x3, uint32_t pick) {
    constexpr int kBias = 0x00808080;
    const uint32_t w0 = static_cast<uint32_t>((x0 + kBias) ^ kBias), w1 = static_cast<uint32_t>((x1 + kBias) ^ kBias);
    const uint32_t w2 = static_cast<uint32_t>((x2 + kBias) ^ kBias), w3 = static_cast<uint32_t>((x3 + kBias) ^ kBias);
    const uint32_t lo = __builtin_amdgcn_perm(w1, w0, pick), hi = __builtin_amdgcn_perm(w3, w2, pick);
    return static_cast<int>(__builtin_amdgcn_perm(hi, lo, 0x05040100u));
}

__device__ __forceinline__ float quad_sum(float v) {
    v += dpp<kDppXor1>(v);
    v += dpp<kDppXor2>(v);
    return v;
}

// Keeps the scheduler from moving instructions across: it would issue the
// loads or products of many tiles ahead and run out of registers.
__device__ __forceinline__ void tile_end() { __builtin_amdgcn_sched_barrier(0); }

// Element `digit` (the lane's place in its quad) of the quad's sum of v.
__device__ __forceinline__ float quad_sum_pick(f32x4 v, int digit) {
    const bool b0 = digit & 1, b1 = digit & 2;
    float x = b0 ? v[1] : v[0], y = b0 ? v[3] : v[2];
    x += dpp<kDppXor1>(b0 ? v[0] : v[1]);
    y += dpp<kDppXor1>(b0 ? v[2] : v[3]);
    float z = b1 ? y : x;
    z += dpp<kDppXor2>(b1 ? x : y);
    return z;
}

template <int D, int QT>
struct FewState {
    static constexpr int KS = D / 64, DT = D / 16;
    i32x4 q[QT][KS];     // q digits
    float q_scale[QT];   // base-2 score = q_scale * (k scale) * integer product
    int position[QT];    // of the lane's row
    float m[QT], l[QT];  // running maximum; the lane's part of the running sum
    f32x4 o[QT][DT];
    float weight;        // 256^digit
    uint32_t pick;
};

// Softmax weights of a block from the lane's raw scores (times f: base-2
// scores) and the state's rescale.  s: [tile][token]; hidden tokens hold -inf
// where MASKED.  On return s holds p * 2^30 relative to the block's maximum,
// and the result is the block's factor relative to the new running maximum
// (with the 2^-30), zero where the row sees nothing of the block.
template <bool MASKED, int DT>
__device__ __forceinline__ float softmax_block(float (&s)[4][4], float f, float &m, float &l, f32x4 (&o)[DT]) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    top = max_xor32(max_xor16(top));
    const bool none = MASKED && top == kNegInf;
    const float bmax = none ? kNegInf : top * f;
    const float next = fmaxf(m, bmax);
    const float ref = next == kNegInf ? 0.0f : next;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    const float factor = none ? 0.0f : __builtin_amdgcn_exp2f(bmax - ref) * 0x1p-30f;
    const float shift = 30.0f - (none ? 0.0f : bmax);
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[t][i], f, shift));
            s[t][i] = MASKED && s[t][i] == kNegInf ? 0.0f : p;
            sum += s[t][i];
        }
    l = l * alpha + sum * factor;
    m = next;
    // The maximum seldom moves after the first blocks.
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
    return factor;
}

// Whether the lane's row at `position` sees token t.
__device__ __forceinline__ bool sees(int position, int t, uint32_t window) {
    return t <= position && (window == 0 || static_cast<uint32_t>(position - t) < window);
}

// A full block whose K and V codes are in registers.
template <bool MASKED, int D, int QT>
__device__ __forceinline__ void few_block(FewState<D, QT> &st, const i32x4 (&k)[4][D / 64], const i32x4 (&v)[D / 16],
                                          float k_scale, float v_scale, int start, uint32_t window) {
    constexpr int KS = D / 64, DT = D / 16;
    const int group = (threadIdx.x & 63) >> 4;
    const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 c = zero;
#pragma unroll
            for (int x = 0; x < KS; ++x) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][x], st.q[qt][x], c, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = quad_sum(static_cast<float>(c[i]) * st.weight);
                if (MASKED && !sees(st.position[qt], start + 16 * t + 4 * group + i, window)) s[t][i] = kNegInf;
            }
        }
        tile_end();
        const float factor = softmax_block<MASKED, DT>(s, st.q_scale[qt] * k_scale, st.m[qt], st.l[qt], st.o[qt]);
        i32x4 p;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            p[t] = digits4(static_cast<int>(s[t][0]), static_cast<int>(s[t][1]), static_cast<int>(s[t][2]),
                           static_cast<int>(s[t][3]), st.pick);
        // A row that sees nothing of the block takes nothing of it, a NaN scale included.
        const float w = MASKED && factor == 0.0f ? 0.0f : v_scale * factor * st.weight;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const i32x4 c = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[d], p, zero, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) st.o[qt][d][i] = fmaf(static_cast<float>(c[i]), w, st.o[qt][d][i]);
            if (d % 4 == 3) tile_end();
        }
    }
}

// The open block: codes in two planes, scales per token.  K's token scales
// multiply the scores; V's are folded into the weights.
template <int D, int QT>
__device__ __forceinline__ void few_open_block(FewState<D, QT> &st, const int8_t *planes, const float *scales, int start,
                                               uint32_t window) {
    constexpr int KS = D / 64, DT = D / 16;
    constexpr size_t kPlane = kKvBlock * D;
    const int lane = threadIdx.x & 63, group = lane >> 4;
    const i32x4 zero = {0, 0, 0, 0};
    f32x4 ks[4], vs[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        ks[t] = *(gptr_f32x4)(uintptr_t)(scales + 16 * t + 4 * group);
        vs[t] = *(gptr_f32x4)(uintptr_t)(scales + 64 + 16 * t + 4 * group);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        float s[4][4];
        float v_top = 0.0f, poison = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 high = zero, low = zero;
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const int at = ((t * KS + x) * 64 + lane) * 16;
                high = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(planes + at), st.q[qt][x], high, 0, 0, 0);
                low = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(planes + kPlane + at), st.q[qt][x], low, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float c = fmaf(static_cast<float>(high[i]), 256.0f, static_cast<float>(low[i]));
                const bool seen = sees(st.position[qt], start + 16 * t + 4 * group + i, window);
                s[t][i] = seen ? quad_sum(c * st.weight) * ks[t][i] : kNegInf;
                v_top = fmaxf(v_top, seen ? vs[t][i] : 0.0f);
                poison += seen ? vs[t][i] - vs[t][i] : 0.0f;  // NaN where a seen scale is not finite
            }
            tile_end();
        }
        v_top = max_xor32(max_xor16(v_top));
        poison = add_xor32(add_xor16(poison));
        const float factor = softmax_block<true, DT>(s, st.q_scale[qt], st.m[qt], st.l[qt], st.o[qt]);
        const float inv = v_top > 0.0f ? 1.0f / v_top : 0.0f;
        i32x4 p;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            int x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = s[t][i] > 0.0f ? static_cast<int>(s[t][i] * (vs[t][i] * inv)) : 0;
            p[t] = digits4(x[0], x[1], x[2], x[3], st.pick);
        }
        const float w = factor == 0.0f ? 0.0f : v_top * factor * st.weight + poison;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int at = (d * 64 + lane) * 16;
            const i32x4 high = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(planes + 2 * kPlane + at), p, zero, 0, 0, 0);
            const i32x4 low = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(planes + 3 * kPlane + at), p, zero, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                st.o[qt][d][i] = fmaf(fmaf(static_cast<float>(high[i]), 256.0f, static_cast<float>(low[i])), w, st.o[qt][d][i]);
            if (d % 2 == 1) tile_end();
        }
    }
}

// The lanes' digits of the rows' q: four rows per tile, column 4 r + digit.
template <int D, int QT, typename T>
__device__ __forceinline__ void load_q(FewState<D, QT> &st, const AttendArgs &a, const Seq &s, uint32_t head, int first_row,
                                       int rows) {
    constexpr int KS = D / 64;
    const int lane = threadIdx.x & 63, column = lane & 15, group = lane >> 4;
    st.pick = (column & 3) | ((4 + (column & 3)) << 8);
    st.weight = static_cast<float>(1u << (8 * (column & 3)));
    const float c = a.d.scale * kLog2e;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = first_row + 4 * qt + (column >> 2);
        const bool live = row < rows;
        const int token = live ? row / static_cast<int>(a.group) : 0;
        const uint32_t h = head * a.group + (live ? row - token * a.group : 0);
        st.position[qt] = s.past + token;
        const T *p = static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(s.first + token) * a.d.q.token_stride +
                     h * a.d.q.head_stride + 16 * group;
        float x[KS][16];
#pragma unroll
        for (int k = 0; k < KS; ++k) load_floats<T, 16>(p + 64 * k, a.wide != 0, x[k]);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
        top = __float_as_uint(max_xor32(max_xor16(__uint_as_float(min(top, 0x7f800000u)))));  // NaN as infinity
        const bool finite = top < 0x7f800000u;
        // largest = f * 2^e, f in [0.5, 1): q * 2^(30 - e) stays below 2^30.
        const int e2 = __builtin_amdgcn_frexp_expf(__uint_as_float(top));
        const int up = finite && top != 0 ? 30 - e2 : 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                int v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = finite ? static_cast<int>(__builtin_amdgcn_ldexpf(x[k][4 * w + e], up)) : 0;
                st.q[qt][k][w] = digits4(v[0], v[1], v[2], v[3], st.pick);
            }
        st.q_scale[qt] = finite ? __builtin_amdgcn_ldexpf(c, -up) : __builtin_nanf("");
        st.m[qt] = kNegInf;
        st.l[qt] = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[qt][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

template <int D, int QT, typename T>
__global__ __launch_bounds__(256, D * QT <= 128 ? 2 : 1) void attend_few_kernel(const AttendArgs a) {
    constexpr int KS = D / 64, DT = D / 16, ROWS = 4 * QT;
    // The waves' results, then (in the last workgroup) the splits' factors.
    __shared__ float part[kWaves][ROWS][D];
    __shared__ float stat[kWaves][ROWS][2];
    __shared__ uint32_t ticket;

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t head = blockIdx.y / a.row_groups, row_group = blockIdx.y - head * a.row_groups;
    const uint32_t seq = blockIdx.z;
    const Seq s = seq_of(a.batch, a.cache, seq);
    if (!s.ok) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) count_fault(a.cache);
        return;
    }
    const int rows = s.count * static_cast<int>(a.group);
    const int first_row = row_group * ROWS;
    if (first_row >= rows || static_cast<uint32_t>(rows) > a.few_rows) return;

    // Blocks that some row of the group sees.
    const int last_row = min(first_row + ROWS, rows) - 1;
    const int end = s.past + last_row / static_cast<int>(a.group) + 1;
    const int first_position = s.past + first_row / static_cast<int>(a.group);
    const int begin = a.d.window != 0 && static_cast<uint32_t>(first_position) >= a.d.window
                          ? first_position - static_cast<int>(a.d.window) + 1 : 0;
    const int block0 = begin / static_cast<int>(kKvBlock);
    const int blocks = (end + static_cast<int>(kKvBlock) - 1) / static_cast<int>(kKvBlock) - block0;
    // A workgroup gets at least a block for each of its waves.
    const int splits = min(static_cast<int>(a.splits), (blocks + kWaves - 1) / kWaves);
    const int split = blockIdx.x;
    if (split >= splits) return;
    const int from = block0 + static_cast<int>(static_cast<int64_t>(split) * blocks / splits);
    const int to = block0 + static_cast<int>(static_cast<int64_t>(split + 1) * blocks / splits);
    const int open_block = s.length % static_cast<int>(kKvBlock) != 0 ? s.length / static_cast<int>(kKvBlock) : -1;

    FewState<D, QT> st;
    load_q<D, QT, T>(st, a, s, head, first_row, rows);

    const int32_t *table = a.batch.table + static_cast<size_t>(seq) * a.batch.table_width;
    const int last_position = s.past + last_row / static_cast<int>(a.group);
    for (int b = from + wave; b < to; b += kWaves) {
        const int start = b * static_cast<int>(kKvBlock);
        if (b == open_block) {
            few_open_block<D, QT>(st, a.cache.open + open_tile(a.cache, s.slot, b, head),
                                  a.cache.open_scales + open_scale_row(a.cache, s.slot, b, head), start, a.d.window);
            continue;
        }
        int page = __builtin_amdgcn_readfirstlane(table[b]);
        float bad = 0.0f;
        if (static_cast<uint32_t>(page) >= a.cache.page_count) {
            if (lane == 0) count_fault(a.cache);
            page = 0;
            bad = __builtin_nanf("");
        }
        const int8_t *tile = a.cache.pages + page_tile(a.cache, page, head);
        const float *scales = a.cache.scales + (static_cast<size_t>(page) * a.cache.kv_heads + head) * 2;
        const f32x2 sc = *(gptr_f32x2)(uintptr_t)scales;
        i32x4 k[4][KS], v[DT];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int x = 0; x < KS; ++x) k[t][x] = load16(tile + ((t * KS + x) * 64 + lane) * 16);
#pragma unroll
        for (int d = 0; d < DT; ++d) v[d] = load16(tile + kKvBlock * D + (d * 64 + lane) * 16);
        const bool masked = start + static_cast<int>(kKvBlock) - 1 > first_position ||
                            (a.d.window != 0 && static_cast<uint32_t>(last_position - start) >= a.d.window);
        if (masked)
            few_block<true, D, QT>(st, k, v, sc[0] + bad, sc[1] + bad, start, a.d.window);
        else
            few_block<false, D, QT>(st, k, v, sc[0] + bad, sc[1] + bad, start, a.d.window);
    }

    // Join the digits and the lanes' sums, then the four waves.
    const int column = lane & 15, group = lane >> 4, digit = column & 3;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = 4 * qt + (column >> 2);
        const float l = add_xor32(add_xor16(st.l[qt]));
        if (group == 0 && digit == 0) {
            stat[wave][r][0] = st.m[qt];
            stat[wave][r][1] = l;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) part[wave][r][16 * d + 4 * group + digit] = quad_sum_pick(st.o[qt][d], digit);
    }
    __syncthreads();

    const int live_rows = min(ROWS, rows - first_row);
    const uint32_t job = blockIdx.z * gridDim.y + blockIdx.y;
    const size_t slot = static_cast<size_t>(job) * a.splits + split;
    const size_t jobs = static_cast<size_t>(gridDim.y) * gridDim.z;
    float *stats = a.partials + jobs * a.splits * ROWS * D;
    for (int x = tid; x < live_rows * D; x += 256) {
        const int r = x / D, d = x % D;
        float m = kNegInf;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stat[w][r][0]);
        const float ref = m == kNegInf ? 0.0f : m;
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat[w][r][0] - ref);
            l += stat[w][r][1] * f;
            o += part[w][r][d] * f;
        }
        if (splits > 1) {
            store_agent(a.partials + (slot * ROWS + r) * D + d, o);
            if (d == 0) {
                store_agent(stats + (slot * ROWS + r) * 2, m);
                store_agent(stats + (slot * ROWS + r) * 2 + 1, l);
            }
        } else {
            const int row = first_row + r, token = row / static_cast<int>(a.group);
            const uint32_t h = head * a.group + (row - token * a.group);
            static_cast<T *>(a.d.out.data)[static_cast<int64_t>(s.first + token) * a.d.out.token_stride +
                                           h * a.d.out.head_stride + d] = static_cast<T>(l == 0.0f ? 0.0f : o / l);
            if (d == 0 && a.d.lse != nullptr)
                a.d.lse[static_cast<size_t>(s.first + token) * a.d.q_heads + h] = (m + log2f(l)) * (1.0f / kLog2e);
        }
    }
    if (splits == 1) return;

    // The last workgroup of the row group joins the splits.
    wait_stores();
    __syncthreads();
    if (tid == 0) ticket = add_agent(a.arrived + job, 1u);
    __syncthreads();
    if (ticket != static_cast<uint32_t>(splits - 1)) return;
    if (tid == 0) store_agent(a.arrived + job, 0u);
    const size_t first_slot = static_cast<size_t>(job) * a.splits;
    for (int x = tid; x < live_rows * D; x += 256) {
        const int r = x / D, d = x % D;
        float m = kNegInf;
        for (int i = 0; i < splits; ++i) m = fmaxf(m, load_agent(stats + ((first_slot + i) * ROWS + r) * 2));
        const float ref = m == kNegInf ? 0.0f : m;
        float l = 0.0f, o = 0.0f;
        for (int i = 0; i < splits; ++i) {
            const float f = __builtin_amdgcn_exp2f(load_agent(stats + ((first_slot + i) * ROWS + r) * 2) - ref);
            l += load_agent(stats + ((first_slot + i) * ROWS + r) * 2 + 1) * f;
            o += load_agent(a.partials + ((first_slot + i) * ROWS + r) * D + d) * f;
        }
        const int row = first_row + r, token = row / static_cast<int>(a.group);
        const uint32_t h = head * a.group + (row - token * a.group);
        static_cast<T *>(a.d.out.data)[static_cast<int64_t>(s.first + token) * a.d.out.token_stride +
                                       h * a.d.out.head_stride + d] = static_cast<T>(l == 0.0f ? 0.0f : o / l);
        if (d == 0 && a.d.lse != nullptr)
            a.d.lse[static_cast<size_t>(s.first + token) * a.d.q_heads + h] = (m + log2f(l)) * (1.0f / kLog2e);
    }
}

template <typename T>
void launch_few(const AttendArgs &a, uint32_t rows, hipStream_t stream) {
    const dim3 grid(a.splits, a.cache.kv_heads * a.row_groups, a.batch.sequences);
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a); };
    if (a.cache.head_dim == 64)
        rows == 4 ? go(attend_few_kernel<64, 1, T>) : go(attend_few_kernel<64, 2, T>);
    else
        rows == 4 ? go(attend_few_kernel<128, 1, T>) : go(attend_few_kernel<128, 2, T>);
}

}  // namespace

uint32_t attend_few_rows(uint32_t rows) { return rows <= 4 ? 4 : 8; }

hipError_t launch_attend_few(const AttendArgs &a, uint32_t rows, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_few<float>(a, rows, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_few<_Float16>(a, rows, stream);
    else launch_few<__bf16>(a, rows, stream);
    return hipGetLastError();
}

}  // namespace q4rdna
