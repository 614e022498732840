// Residual add with the norms before and after it (q4rdna_add_norm).
//
//   h = residual + scale * gate * post(y),   n = rms(h) * weight
//
// One pass over memory: a workgroup keeps its row in registers between the two
// sums (mean y^2, then mean h^2), so every input is read once and every output
// written once.  Products are in fp32, sums of squares in fp32 over 64 neighbours, as
// one tree of pairs, and in 64 bits from there on: so the factor does not depend on
// how many numbers a thread takes, which differs between aligned and unaligned rows.
// With 1024 threads a row the 64 bits cost a few percent (64 rows of 8192 in fp16,
// both norms: 3.9 us, in fp32 alone 3.75; 77 rows of 1111 3.4 and 3.5).  The weights
// stay fp32, since models keep them so and they come from the L2.
//
// Many rows are bound by the memory: 8192 rows of 4096 in bf16 (residual and y
// in, h and n out, 268 MB) take 39 us where the inputs are in the Infinity
// Cache and 55 us where they are not, 4.9 TB/s; a plain copy reaches 5.2 TB/s.
// Few rows are bound by the launch and one trip to memory: 2.4 us for one row.
#include "q4rdna_layer_device.h"

#include <algorithm>

namespace q4rdna {
namespace {

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t low = dpp<CTRL>(static_cast<uint32_t>(b)), high = dpp<CTRL>(static_cast<uint32_t>(b >> 32));
    return __builtin_bit_cast(double, high << 32 | low);
}
// v + v of lane ^ 16 and of lane ^ 32.
__device__ __forceinline__ double sum_rows(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const auto low = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(b), static_cast<uint32_t>(b), false, false);
    const auto high = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(b >> 32), static_cast<uint32_t>(b >> 32), false, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) +
           __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
}
__device__ __forceinline__ double sum_halves(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const auto low = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(b), static_cast<uint32_t>(b), false, false);
    const auto high = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(b >> 32), static_cast<uint32_t>(b >> 32), false, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) +
           __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
}

// The sums of four v over the wave's rows of 16 lanes, v[i] in row i: two sums for
// each swap.  Its pairs are those of add_xor32(add_xor16(v)).
__device__ __forceinline__ float sum_rows4(float v0, float v1, float v2, float v3) {
    const auto p01 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v0), __float_as_uint(v1), false, false);
    const auto p23 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v2), __float_as_uint(v3), false, false);
    const float s01 = __uint_as_float(p01[0]) + __uint_as_float(p01[1]);
    const float s23 = __uint_as_float(p23[0]) + __uint_as_float(p23[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(s01), __float_as_uint(s23), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// The wave's sum of squares of VEC numbers a lane in CH runs: 64 neighbours in
// fp32, always as the same tree of pairs, whether eight, four or one of them lie in
// a lane; the sums of 64 in 64 bits.
template <int CH, int VEC>
__device__ __forceinline__ double wave_squares(const float (&x)[CH][VEC]) {
#pragma clang fp contract(off)
    static_assert(VEC == 1 || VEC == 4 || VEC == 8);
    float v[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float tree[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) tree[e] = x[c][e] * x[c][e];
#pragma unroll
        for (int step = 1; step < VEC; step *= 2)
#pragma unroll
            for (int e = 0; e < VEC; e += 2 * step) tree[e] += tree[e + step];
        v[c] = tree[0];
        v[c] += dpp<kDppXor1>(v[c]);
        v[c] += dpp<kDppXor2>(v[c]);
        v[c] += dpp<kDppMirror8>(v[c]);
        if (VEC < 8) v[c] += dpp<kDppMirror16>(v[c]);
    }
    double sum = 0.0;
    if constexpr (VEC == 1 && CH % 4 == 0) {
#pragma unroll
        for (int c = 0; c < CH; c += 4) sum += sum_rows4(v[c], v[c + 1], v[c + 2], v[c + 3]);
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) sum += VEC == 1 ? add_xor32(add_xor16(v[c])) : v[c];
        if (VEC == 1) return sum;
        if (VEC == 8) sum += dpp64<kDppMirror16>(sum);
    }
    return sum_halves(sum_rows(sum));
}

// The workgroup's sum of v, the same in each wave's lanes; `slots` is the caller's
// own for each sum, so one barrier is enough.
template <int NT>
__device__ __forceinline__ double block_sum(double v, double *slots) {
    static_assert(NT == 64 || NT == 256 || NT == 512 || NT == 1024, "one, two or four lanes with four waves' sums each");
    if (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    const double *mine = slots + threadIdx.x % (NT / 256 ? NT / 256 : 1) * 4;
    v = (mine[0] + mine[1]) + (mine[2] + mine[3]);
    if (NT >= 512) v += dpp64<kDppXor1>(v);
    if (NT >= 1024) v += dpp64<kDppXor2>(v);
    return v;
}

// The norm's factor, 1 / sqrt(sum / width + eps), rounded once: the sum is in 64
// bits and so is the remainder of the step of Newton's iteration on the
// instruction's result (1 ulp).  The instruction takes no subnormal number, so
// small ones are scaled by 2^128; above fp32's range it gives zero, and infinity
// for zero.
__device__ __forceinline__ float norm_factor(double sum, double per_width, float eps) {
    const double mean = fma(sum, per_width, static_cast<double>(eps));
    const bool tiny = mean < 0x1p-100;
    const double x = tiny ? mean * 0x1p128 : mean;
    const float y = __builtin_amdgcn_rsqf(static_cast<float>(x));
    const double y64 = y;
    const float rest = static_cast<float>(fma(-x * y64, y64, 1.0));
    const float root = y > 0.0f && y < __builtin_inff() ? fmaf(0.5f * y, rest, y) : y;
    return tiny ? root * 0x1p64f : root;
}

// NT threads a row, CH runs of VEC numbers per thread.
template <typename T, int VEC, int NT, int CH>
__global__ __launch_bounds__(NT) void add_norm_kernel(const q4rdna_add_norm_desc d, double per_width) {
    __shared__ __align__(16) double slots[2][NT / 64];
    const uint32_t row = blockIdx.x;
    const T *res = static_cast<const T *>(d.residual) + row * d.residual_stride;
    const uint32_t width = d.width;
    const bool wide = VEC > 1;
    float h[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t at = (c * NT + threadIdx.x) * VEC;
        if (at < width) {
            load_floats<T, VEC>(res + at, wide, h[c]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[c][e] = 0.0f;
        }
    }
    if (d.y != nullptr) {
        const T *yrow = static_cast<const T *>(d.y) + row * d.y_stride;
        float y[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t at = (c * NT + threadIdx.x) * VEC;
            if (at < width) {
                load_floats<T, VEC>(yrow + at, wide, y[c]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[c][e] = 0.0f;
            }
        }
        if (d.post_weight != nullptr) {
            const double sum = block_sum<NT>(wave_squares(y), slots[0]);
            const float inv = norm_factor(sum, per_width, d.eps);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const uint32_t at = (c * NT + threadIdx.x) * VEC;
                if (at < width) {
                    float w[VEC];
                    load_floats<float, VEC>(d.post_weight + at, wide, w);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[c][e] = y[c][e] * inv * w[e];
                }
            }
        }
        if (d.gate != nullptr) {
            const T *gate = static_cast<const T *>(d.gate) + row * d.gate_stride;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const uint32_t at = (c * NT + threadIdx.x) * VEC;
                if (at < width) {
                    float g[VEC];
                    load_floats<T, VEC>(gate + at, wide, g);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[c][e] *= g[e];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[c][e] += d.scale * y[c][e];
    }
    if (d.h != nullptr) {
        T *out = static_cast<T *>(d.h) + row * d.h_stride;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t at = (c * NT + threadIdx.x) * VEC;
            if (at < width) store_floats<T, VEC>(out + at, wide, h[c]);
        }
    }
    if (d.n == nullptr) return;
    const double sum = block_sum<NT>(wave_squares(h), slots[1]);
    const float inv = norm_factor(sum, per_width, d.eps);
    T *out = static_cast<T *>(d.n) + row * d.n_stride;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t at = (c * NT + threadIdx.x) * VEC;
        if (at < width) {
            float w[VEC];
            load_floats<float, VEC>(d.weight + at, wide, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = h[c][e] * inv * w[e];
            store_floats<T, VEC>(out + at, wide, w);
        }
    }
}

// A matrix from one of its rows on.
template <typename T>
const void *from_row(const void *p, int64_t stride, uint32_t row) {
    return p == nullptr ? p : static_cast<const T *>(p) + row * stride;
}
template <typename T>
void *from_row(void *p, int64_t stride, uint32_t row) {
    return p == nullptr ? p : static_cast<T *>(p) + row * stride;
}

template <typename T, int VEC>
hipError_t launch(const q4rdna_add_norm_desc &d, uint32_t cus, hipStream_t stream) {
    // A launch holds fewer than 2^32 threads: more rows go in several.
    auto go = [&](auto kernel, uint32_t threads) {
        q4rdna_add_norm_desc part = d;
        for (uint32_t row = 0; row < d.rows; row += part.rows) {
            part.rows = std::min(d.rows - row, 0xffffffffu / threads);
            part.residual = from_row<T>(d.residual, d.residual_stride, row);
            part.y = from_row<T>(d.y, d.y_stride, row);
            part.gate = from_row<T>(d.gate, d.gate_stride, row);
            part.h = from_row<T>(d.h, d.h_stride, row);
            part.n = from_row<T>(d.n, d.n_stride, row);
            kernel<<<part.rows, threads, 0, stream>>>(part, 1.0 / d.width);
        }
    };
    const uint32_t runs = (d.width + VEC - 1) / VEC;  // per row
    // A run per thread is the shortest chain, and up to 512 threads the faster
    // one at any number of rows (fp16/bf16 rows of 4096, against two runs in
    // half the threads: 2.4 us, 2.8 us for one row; 39.2 us, 40.1 us for 8192).
    // 1024 threads fill a CU with two rows: with more rows than that, two runs
    // each in 512 (bf16 rows of 8192, 1024 threads against 512: 2.6 us, 3.0 us
    // for one row, 5.8 us, 6.1 us for 512, 9.8 us, 8.6 us for 768).
    const bool few = d.rows <= 2 * cus;
    if (runs <= 64) {
        go(add_norm_kernel<T, VEC, 64, 1>, 64);
    } else if (runs <= 256) {
        go(add_norm_kernel<T, VEC, 256, 1>, 256);
    } else if (runs <= 512) {
        go(add_norm_kernel<T, VEC, 512, 1>, 512);
    } else if (runs <= 1024) {
        few ? go(add_norm_kernel<T, VEC, 1024, 1>, 1024) : go(add_norm_kernel<T, VEC, 512, 2>, 512);
    } else if (runs <= 2048) {
        go(add_norm_kernel<T, VEC, 1024, 2>, 1024);
    } else if constexpr (VEC < 8) {  // at most Q4RDNA_NORM_MAX_WIDTH numbers
        if (VEC == 4 || runs <= 4096)
            go(add_norm_kernel<T, VEC, 1024, 4>, 1024);
        else if constexpr (VEC == 1)
            go(add_norm_kernel<T, VEC, 1024, 16>, 1024);
    }
    return hipGetLastError();
}

}  // namespace

// `wide`: every row starts at a multiple of the vector (16 bytes) and holds a
// whole number of vectors; the weights are 16-byte aligned.
hipError_t launch_add_norm(const q4rdna_add_norm_desc &d, bool wide, uint32_t cus, hipStream_t stream) {
    if (d.dtype == Q4RDNA_F32) return wide ? launch<float, 4>(d, cus, stream) : launch<float, 1>(d, cus, stream);
    if (d.dtype == Q4RDNA_F16) return wide ? launch<_Float16, 8>(d, cus, stream) : launch<_Float16, 1>(d, cus, stream);
    return wide ? launch<__bf16, 8>(d, cus, stream) : launch<__bf16, 1>(d, cus, stream);
}

}  // namespace q4rdna
