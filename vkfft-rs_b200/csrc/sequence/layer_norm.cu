// Layer normalisation over the last axis, forward and backward.
#include "device.cuh"

namespace b200fft {

namespace {

constexpr int kThreads = 256;

// Sum over the block, in every thread, in a fixed order.
__device__ __forceinline__ float block_sum(float v, float *buf) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0;
#pragma unroll
    for (int k = 0; k < kThreads / 32; k++) s += buf[k];
    return s;
}

// A row of any width: one CTA reads it three times (the second and third from L1 or L2).
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) norm_long_kernel(NormParams p) {
    __shared__ float buf[kThreads / 32];
    const P *w = static_cast<const P *>(p.w), *b = static_cast<const P *>(p.b);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(p.x) + row * p.xs;
        T *y = static_cast<T *>(p.y) + row * p.ys;
        float s = 0;
        for (int64_t i = threadIdx.x; i < p.features; i += kThreads) s += to_float(x[i]);
        const float mean = block_sum(s, buf) / (float)p.features;
        s = 0;
        for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
            const float d = to_float(x[i]) - mean;
            s += d * d;
        }
        const float rstd = 1.f / sqrtf(block_sum(s, buf) / (float)p.features + p.epsilon);
        for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
            float v = (to_float(x[i]) - mean) * rstd;
            if (w) v *= to_float(w[i]);
            if (b) v += to_float(b[i]);
            y[i] = from_float<T>(v);
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
    }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) norm_grad_long_kernel(NormGradParams p) {
    __shared__ float buf[kThreads / 32];
    const P *w = static_cast<const P *>(p.w);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(p.x) + row * p.xs, *dy = static_cast<const T *>(p.dy) + row * p.ys;
        T *dx = static_cast<T *>(p.dx) + row * p.xs;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s0 = 0, s1 = 0;
        for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
            const float g = to_float(dy[i]) * (w ? to_float(w[i]) : 1.f);
            s0 += g;
            s1 += g * ((to_float(x[i]) - mean) * rstd);
        }
        s0 = block_sum(s0, buf) / (float)p.features;
        s1 = block_sum(s1, buf) / (float)p.features;
        for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
            const float g = to_float(dy[i]) * (w ? to_float(w[i]) : 1.f);
            const float h = (to_float(x[i]) - mean) * rstd;
            dx[i] = from_float<T>(rstd * (g - s0 - h * s1));
        }
    }
}

// Column sums of dy xhat and dy over one strip of rows: 32 columns x 8 row lanes.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_columns_kernel(NormGradParams p) {
    __shared__ float sw[8][33], sb[8][33];
    const int c = threadIdx.x & 31, lane = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    const int64_t strip = (p.rows + p.partials - 1) / p.partials;
    const int64_t r0 = blockIdx.y * strip, r1 = min(p.rows, r0 + strip);
    float aw = 0, ab = 0;
    if (col < p.features)
        for (int64_t r = r0 + lane; r < r1; r += 8) {
            const float g = to_float(static_cast<const T *>(p.dy)[r * p.ys + col]);
            aw += g * ((to_float(static_cast<const T *>(p.x)[r * p.xs + col]) - p.mean[r]) * p.rstd[r]);
            ab += g;
        }
    sw[lane][c] = aw;
    sb[lane][c] = ab;
    __syncthreads();
    if (lane == 0 && col < p.features) {
        for (int k = 1; k < 8; k++) {
            aw += sw[k][c];
            ab += sb[k][c];
        }
        p.part_w[blockIdx.y * p.features + col] = aw;
        p.part_b[blockIdx.y * p.features + col] = ab;
    }
}

template <typename P>
__global__ void __launch_bounds__(kThreads) norm_grad_reduce_kernel(NormGradParams p) {
    const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (col >= p.features) return;
    float aw = 0, ab = 0;
    for (int k = 0; k < p.partials; k++) {
        aw += p.part_w[k * p.features + col];
        ab += p.part_b[k * p.features + col];
    }
    if (p.dw) static_cast<P *>(p.dw)[col] = from_float<P>(aw);
    if (p.db) static_cast<P *>(p.db)[col] = from_float<P>(ab);
}

int grid_of(int64_t n, int64_t most) { return (int)(n < most ? n : most); }

}  // namespace

cudaError_t launch_norm(const NormParams &p, Element e, Element param, cudaStream_t s) {
    return with_element(e, [&](auto t) {
        return with_element(param, [&](auto q) {
            using T = decltype(t);
            using P = decltype(q);
            before_launch();
            norm_long_kernel<T, P><<<grid_of(p.rows, 1 << 30), kThreads, 0, s>>>(p);
            return cudaGetLastError();
        });
    });
}

cudaError_t launch_norm_grad(const NormGradParams &p, Element e, Element param, cudaStream_t s) {
    return with_element(e, [&](auto t) {
        return with_element(param, [&](auto q) {
            using T = decltype(t);
            using P = decltype(q);
            // the sums first: dx may take the place of dy
            if (p.dw || p.db) {
                before_launch();
                norm_grad_columns_kernel<T><<<dim3((unsigned)((p.features + 31) / 32), p.partials), kThreads, 0, s>>>(p);
                before_launch();
                norm_grad_reduce_kernel<P><<<(unsigned)((p.features + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
            }
            if (p.dx) {
                before_launch();
                norm_grad_long_kernel<T, P><<<grid_of(p.rows, 1 << 30), kThreads, 0, s>>>(p);
            }
            return cudaGetLastError();
        });
    });
}

}  // namespace b200fft
