// Drafted tokens on their way to the attention: positions and ancestors from
// their parents (q4rdna_kv_tree), queries and keys normalised and rotated by
// given positions (q4rdna_rotate).
#include "q4rdna_layer_device.h"
#include "q4rdna_rotate_device.h"

namespace q4rdna {
namespace {

// A wave per sequence, a lane per token.  In step s a lane has the tokens up to
// 2^s above its own and the next one up, `up`, and takes what that one has:
// six steps for 64 tokens.  A token below a bad one is bad.  Two dependent loads
// and a launch: 1.8 us for one sequence, 3.0 for 96.
__global__ __launch_bounds__(256) void tree_kernel(const q4rdna_kv_batch b, const int32_t *parents, int32_t *positions,
                                                   uint64_t *seen) {
    const uint32_t i = blockIdx.x * 4 + wave_id();
    const int lane = threadIdx.x & 63;
    if (i >= b.sequences) return;
    const int first = b.cu_tokens ? b.cu_tokens[i] : static_cast<int>(i);
    const int end = b.cu_tokens ? b.cu_tokens[i + 1] : static_cast<int>(i) + 1;
    const int past = b.past[i];
    if (first < 0 || end < first || static_cast<uint32_t>(end) > b.tokens) return;
    const int count = end - first;
    if (count > static_cast<int>(min(b.max_tokens, kTreeMax)) || past < 0 || past > (1 << 30)) {
        for (int n = first + lane; n < end; n += 64) {
            positions[n] = -1;
            seen[n] = 0;
        }
        return;
    }
    int up = lane < count ? parents[first + lane] : -1;
    uint32_t bad = up < -1 || up >= lane;
    if (bad) up = -1;
    uint32_t low = lane < 32 ? 1u << lane : 0u, high = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int s = 0; s < 6; ++s) {
        const int from = 4 * max(up, 0);
        const uint32_t l = __builtin_amdgcn_ds_bpermute(from, low), h = __builtin_amdgcn_ds_bpermute(from, high);
        const uint32_t bd = __builtin_amdgcn_ds_bpermute(from, bad);
        const int next = __builtin_amdgcn_ds_bpermute(from, up);
        if (up >= 0) {
            low |= l;
            high |= h;
            bad |= bd;
            up = next;
        }
    }
    if (lane >= count) return;
    positions[first + lane] = bad ? -1 : past + __builtin_popcount(low) + __builtin_popcount(high) - 1;
    seen[first + lane] = bad ? 0 : static_cast<uint64_t>(high) << 32 | low;
}

// a.unit_rows rows (token, head of q and then of k), one at a time for a group of
// D / 8 lanes.  A row is read and written once: 16 tokens of 32 and 8 heads by 128
// in fp32 3.5 us, a chain of loads (position, cosines); 61 MB in bf16 16.1 us, 3.8
// TB/s (two rows of a group in flight 16.6, with fewer waves on a CU).
template <int D, bool INTERLEAVED, typename T>
__global__ __launch_bounds__(256) void rotate_kernel(const RotateArgs a) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    const Place at = place_of<INTERLEAVED>(lane, a.d.rotary);
    Weights q_weights, k_weights;
    load_weights(q_weights, a.d.q_norm, at);
    load_weights(k_weights, a.d.k_norm, at);
    const uint32_t row_first = blockIdx.x * a.unit_rows, row_end = min(a.rows - row_first, a.unit_rows);
    // One division per workgroup, a multiplication per row.
    const uint32_t n_first = row_first / a.heads, head_first = row_first - n_first * a.heads;
    for (uint32_t x = threadIdx.x / kLanes; x < row_end; x += kRows) {
        const uint32_t local = head_first + x, token = div_split(local, a.heads, a.heads_magic);
        const uint32_t n = n_first + token, h = local - token * a.heads;
        const bool is_k = h >= a.d.q_heads;
        const uint32_t head = is_k ? h - a.d.q_heads : h;
        const q4rdna_kv_rows &in = is_k ? a.d.k : a.d.q, &to = is_k ? a.d.k_out : a.d.q_out;
        const int position = a.d.rotary != 0 ? a.d.position[n] : 0;
        Row r;
        load_row(r, static_cast<const T *>(in.data) + static_cast<int64_t>(n) * in.token_stride + head * in.head_stride, at, a.wide != 0);
        const bool there = static_cast<uint32_t>(position) < a.d.positions;
        Turn turn;
        load_turn(turn, at, a.d.cos, a.d.sin, a.d.rotary, there ? position : 0);
        if (a.d.rotary != 0 && !there)
#pragma unroll
            for (int e = 0; e < 4; ++e) r.a[e] = r.b[e] = __builtin_nanf("");
        if (is_k ? a.d.k_norm != nullptr : a.d.q_norm != nullptr) norm_row<D>(r, is_k ? k_weights : q_weights, a.d.eps);
        turn_row<INTERLEAVED>(r, at, turn);
        T *out = static_cast<T *>(to.data) + static_cast<int64_t>(n) * to.token_stride + head * to.head_stride;
        store_floats<T, 4>(out + at.a_at, a.wide != 0, r.a);
        store_floats<T, 4>(out + at.b_at, a.wide != 0, r.b);
    }
}

}  // namespace

hipError_t launch_tree(const q4rdna_kv_batch &batch, const int32_t *parents, int32_t *positions, uint64_t *seen,
                       hipStream_t stream) {
    tree_kernel<<<(batch.sequences + 3) / 4, 256, 0, stream>>>(batch, parents, positions, seen);
    return hipGetLastError();
}

template <bool INTERLEAVED, typename T>
static void launch_rotate_as(const RotateArgs &a, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<(a.rows + a.unit_rows - 1) / a.unit_rows, 256, 0, stream>>>(a); };
    a.d.head_dim == 64 ? go(rotate_kernel<64, INTERLEAVED, T>) : go(rotate_kernel<128, INTERLEAVED, T>);
}
template <typename T>
static void launch_rotate_as(const RotateArgs &a, hipStream_t stream) {
    a.d.interleaved != 0 ? launch_rotate_as<true, T>(a, stream) : launch_rotate_as<false, T>(a, stream);
}
hipError_t launch_rotate(const RotateArgs &a, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_rotate_as<float>(a, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_rotate_as<_Float16>(a, stream);
    else launch_rotate_as<__bf16>(a, stream);
    return hipGetLastError();
}

}  // namespace q4rdna
