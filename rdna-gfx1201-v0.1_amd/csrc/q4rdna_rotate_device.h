// The norm of a head's row and its rotation by position (q4rdna_cache.hip,
// q4rdna_draft.hip).
#pragma once

#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

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

template <bool INTERLEAVED>
__device__ __forceinline__ Place place_of(int lane, uint32_t rotary) {
    const int half = static_cast<int>(rotary) / 2;
    Place p;
    p.pair = 4 * lane;
    p.turned = p.pair < half;  // rotary is a multiple of 8: a lane's pairs lie on one side
    if (p.turned && !INTERLEAVED) {
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
__device__ __forceinline__ void load_turn(Turn &t, const Place &p, const float *cos, const float *sin, uint32_t rotary,
                                          int position) {
    if (!p.turned) return;
    const size_t at = static_cast<size_t>(position) * (rotary / 2) + p.pair;
    load_floats<float, 4>(cos + at, true, t.c);
    load_floats<float, 4>(sin + at, true, t.s);
}

// The lane's norm weights, once per workgroup.
struct Weights {
    float a[4], b[4];
};
__device__ __forceinline__ void load_weights(Weights &w, const float *weight, const Place &p) {
    if (weight == nullptr) return;
    load_floats<float, 4>(weight + p.a_at, true, w.a);
    load_floats<float, 4>(weight + p.b_at, true, w.b);
}
// Which products are fused is written out here and in turn_pair: the compiler
// would choose anew for each copy of an unrolled loop, and the cache's bytes
// would depend on a token's place in its step.
template <int D>
__device__ __forceinline__ void norm_row(Row &r, const Weights &w, float eps) {
#pragma clang fp contract(off)
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fmaf(r.a[e], r.a[e], fmaf(r.b[e], r.b[e], sum));
    const float inv = inverse_root(fmaf(lanes_sum<D / 8>(sum), 1.0f / D, eps), eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r.a[e] = r.a[e] * inv * w.a[e];
        r.b[e] = r.b[e] * inv * w.b[e];
    }
}
__device__ __forceinline__ void turn_pair(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
    const float bs = b * s, as = a * s;
    const float x = fmaf(a, c, -bs);
    b = fmaf(b, c, as);
    a = x;
}
template <bool INTERLEAVED>
__device__ __forceinline__ void turn_row(Row &r, const Place &p, const Turn &t) {
    if (!p.turned) return;
    if (INTERLEAVED) {
        turn_pair(r.a[0], r.a[1], t.c[0], t.s[0]);
        turn_pair(r.a[2], r.a[3], t.c[1], t.s[1]);
        turn_pair(r.b[0], r.b[1], t.c[2], t.s[2]);
        turn_pair(r.b[2], r.b[3], t.c[3], t.s[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) turn_pair(r.a[e], r.b[e], t.c[e], t.s[e]);
    }
}

}  // namespace
}  // namespace q4rdna
