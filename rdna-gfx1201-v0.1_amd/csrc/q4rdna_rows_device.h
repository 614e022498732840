// Rows of queries on fp16 matrix instructions: what attend_many_kernel and
// attend_tree_kernel share.  A lane holds one row; its state is what the comment
// of q4rdna_attend_many.hip describes.
#pragma once

#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLazy = 8.0f;    // the maximum may trail by this much (base 2)
constexpr float kWeight = 7.0f;  // weights are 2^7 relative to their reference, at most 2^15, within fp16's range
constexpr float kLeast = -90.0f; // a block's V scale counts as 2^-90 of the reference at least
// Four codes as fp16: 0x6400 | (code + 128) is 1024 + code + 128.
__device__ __forceinline__ void codes_to_half(uint32_t w, h16x2 &lo, h16x2 &hi) {
    const uint32_t u = w ^ 0x80808080u;
    const h16x2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    lo = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
    hi = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
}
template <int D, int SPLIT>
struct ManyState {
    h16x8 q[D / 16][SPLIT];
    float q_scale;    // base-2 score = q_scale * (k scale) * product
    int position;     // of the lane's row
    float m, l;       // the maximum that the sum refers to; the lane's part of the sum, in units of 2^(m - 7)
    float e;          // a whole number, -inf while nothing was added: accumulators are in units of 2^(m + e - 7)
    f32x16 o[D / 32];
};

// Bits of the tokens 8 x + b (bit 4 x + b, b < 4) that are at most `ahead`.
__device__ __forceinline__ uint32_t first_tokens(int ahead) {
    const int count = ahead < 0 ? 0 : ahead >= 63 ? 32 : ahead / 8 * 4 + min(ahead % 8 + 1, 4);
    return count == 32 ? 0xffffffffu : (1u << count) - 1u;
}
__device__ __forceinline__ uint32_t bit_mask(uint32_t bits, int i) {
    return static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - i)) >> 31);
}

// Moves the references where the row's next block needs it: m to its maximum
// `now` and m + e to its largest weight times V scale, `top` (both base 2).
template <int D, int SPLIT>
__device__ __forceinline__ void refer(ManyState<D, SPLIT> &st, float now, float top) {
    const bool grown = now > st.m + kLazy, more = top > st.m + st.e + kLazy;
    if (__builtin_amdgcn_ballot_w64(grown || more) == 0) return;
    if (!(grown || more)) return;
    const float m = grown ? now : st.m, most = fmaxf(st.m + st.e, top);
    const float e = most == kNegInf ? kNegInf : ceilf(most - m);
    st.l *= __builtin_amdgcn_exp2f(st.m - m);  // 0 from -inf
    const float f = st.e == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((st.m - m) + (st.e - e));  // (o is zero there)
#pragma unroll
    for (int d = 0; d < D / 32; ++d) st.o[d] *= f;
    st.m = m;
    st.e = e;
}

}  // namespace
}  // namespace q4rdna
