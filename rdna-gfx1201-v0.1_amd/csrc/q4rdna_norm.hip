// Residual add with the norms before and after it (q4rdna_add_norm).
//
//   h = residual + scale * gate * post(y),   n = rms(h) * weight
//
// One pass over memory: a workgroup keeps its row in registers between the two
// sums (mean y^2, then mean h^2), so every input is read once and every output
// written once.  Sums and products are in fp32; the weights stay fp32, since
// models keep them so and they come from the L2.
//
// Many rows are bound by the memory: 8192 rows of 4096 in bf16 (residual and y
// in, h and n out, 268 MB) take 39 us where the inputs are in the Infinity
// Cache and 55 us where they are not, 4.9 TB/s; a plain copy reaches 5.2 TB/s.
// Few rows are bound by the launch and one trip to memory: 2.4 us for one row.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

// The workgroup's sum of v; `slots` is the caller's own for each sum, so one
// barrier is enough.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float *slots) {
    v = lanes_sum<16>(v);
    v = add_xor32(add_xor16(v));
    if (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) sum += slots[w];
    return sum;
}

// NT threads a row, CH runs of VEC numbers per thread.
template <typename T, int VEC, int NT, int CH>
__global__ __launch_bounds__(NT) void add_norm_kernel(const q4rdna_add_norm_desc d) {
    __shared__ float slots[2][NT / 64];
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
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum += y[c][e] * y[c][e];
            sum = block_sum<NT>(sum, slots[0]);
            const float inv = 1.0f / sqrtf(sum / static_cast<float>(width) + d.eps);
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
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t at = (c * NT + threadIdx.x) * VEC;
        if (at < width) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += h[c][e] * h[c][e];
        }
    }
    sum = block_sum<NT>(sum, slots[1]);
    const float inv = 1.0f / sqrtf(sum / static_cast<float>(width) + d.eps);
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

template <typename T, int VEC>
hipError_t launch(const q4rdna_add_norm_desc &d, uint32_t cus, hipStream_t stream) {
    auto go = [&](auto kernel, uint32_t threads) { kernel<<<d.rows, threads, 0, stream>>>(d); };
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
