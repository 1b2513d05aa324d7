// Layer normalisation over the last axis, forward and backward.
#include <algorithm>

#include "launch.cuh"

namespace b200fft {

namespace {

constexpr int kThreads = 256;
template <int N>
using Int = std::integral_constant<int, N>;

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

// ---- rows in registers ----------------------------------------------------------------
// A row belongs to TPR threads of a block, each with VPT vectors of VEC elements (16 bytes, or single elements where
// rows or addresses are not aligned): one read, mean and centred variance from registers, one write.  Bound by HBM;
// the weight and bias come from L1 after the first row.

template <typename T, int VEC>
struct Vec {
    float f[VEC];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC == 1) {
            f[0] = to_float(*p);
        } else {
            static_assert(VEC * sizeof(T) == 16, "16 bytes");
            const uint4 w = *reinterpret_cast<const uint4 *>(p);
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int i = 0; i < VEC; i++) f[i] = to_float(e[i]);
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (VEC == 1) {
            *p = from_float<T>(f[0]);
        } else {
            uint4 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int i = 0; i < VEC; i++) e[i] = from_float<T>(f[i]);
            *reinterpret_cast<uint4 *>(p) = w;
        }
    }
};

// The raw 16 bytes (or one element) of a vector, as they wait for their turn.
template <typename T, int VEC>
struct Raw {
    uint4 w;
    __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ float at(int i) const { return to_float(reinterpret_cast<const T *>(&w)[i]); }
};
template <typename T>
struct Raw<T, 1> {
    T w;
    __device__ __forceinline__ void load(const T *p) { w = *p; }
    __device__ __forceinline__ float at(int) const { return to_float(w); }
};

// VEC parameters of whatever type, from an index that is a multiple of VEC; aligned where VEC > 1.
template <int VEC>
__device__ __forceinline__ void load_parameters(const void *p, Element type, int64_t at, float (&f)[VEC]) {
    if (type == Element::F32) {
        const float *q = static_cast<const float *>(p) + at;
        if constexpr (VEC == 1) {
            f[0] = *q;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const float4 w = *reinterpret_cast<const float4 *>(q + i);
                f[i] = w.x, f[i + 1] = w.y, f[i + 2] = w.z, f[i + 3] = w.w;
            }
        }
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(p) + at;
        uint32_t w[(VEC + 1) / 2];
        if constexpr (VEC == 1) {
            w[0] = *q;
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 4; i++) {
                const uint2 v = *reinterpret_cast<const uint2 *>(q + 4 * i);
                w[2 * i] = v.x, w[2 * i + 1] = v.y;
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const uint16_t bits = (uint16_t)(w[i / 2] >> (i % 2 * 16));
            f[i] = type == Element::F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
        }
    }
}

// Sums over the TPR threads of a row, the same in all of them.  `buf` has two halves for two calls in a row.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *buf) {
#pragma unroll
    for (int n = 0; n < N; n++) v[n] = warp_sum(v[n]);
    if constexpr (TPR > 32) {
        constexpr int WARPS = TPR / 32;
        float *mine = buf + threadIdx.x / TPR * WARPS * N;
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int n = 0; n < N; n++) mine[(threadIdx.x % TPR / 32) * N + n] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; n++) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; k++) s += mine[k * N + n];
            v[n] = s;
        }
    }
}

template <typename T, int VEC, int TPR, int VPT>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_kernel(const __grid_constant__ NormParams p) {
    constexpr int BLOCK = TPR < 128 ? 128 : TPR, ROWS = BLOCK / TPR;
    __shared__ float buf[2][BLOCK / 32];
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    const int at = threadIdx.x % TPR;
    if (TPR == 32 && row >= p.rows) return;  // (wider rows: a block is one row)
    const T *x = static_cast<const T *>(p.x) + row * p.xs;
    T *y = static_cast<T *>(p.y) + row * p.ys;
    const int units = (int)p.features / VEC;
    Vec<T, VEC> v[VPT];
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (at + k * TPR < units) v[k].load(x + (at + k * TPR) * VEC);
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (at + k * TPR < units) {
#pragma unroll
            for (int i = 0; i < VEC; i++) s[0] += v[k].f[i];
        }
    row_sums<TPR>(s, buf[0]);
    const float mean = s[0] / (float)p.features;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (at + k * TPR < units) {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                v[k].f[i] -= mean;
                s[0] = fmaf(v[k].f[i], v[k].f[i], s[0]);
            }
        }
    row_sums<TPR>(s, buf[1]);
    const float rstd = 1.f / sqrtf(s[0] / (float)p.features + p.epsilon);
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (at + k * TPR < units) {
            float w[VEC], b[VEC];
            if (p.w) load_parameters<VEC>(p.w, p.parameter, (at + k * TPR) * VEC, w);
            if (p.b) load_parameters<VEC>(p.b, p.parameter, (at + k * TPR) * VEC, b);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float f = v[k].f[i] * rstd;
                if (p.w) f *= w[i];
                if (p.b) f += b[i];
                v[k].f[i] = f;
            }
            v[k].store(y + (at + k * TPR) * VEC);
        }
    if (at == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
}

// dx of a row from its two sums; dw and db of the thread's columns over all rows of its group (partials groups of TPR
// threads, each with every partials-th row).  NEXT: the next row's loads stand ahead of this row's sums, and the columns'
// sums in registers.  Otherwise (rows of 1024 threads, whose 64 registers do not hold that) they stand in shared memory:
// 8 bytes read and written for each element, half of what the row takes from HBM at HBM's pace.
template <typename T, int VEC, int TPR, int VPT, bool NEXT>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR <= 256 ? 2 : 1) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, GROUPS = BLOCK / TPR;
    __shared__ float buf[2][BLOCK / 32 * 2];
    extern __shared__ __align__(16) float columns[];  // [2][VPT][VEC][TPR]
    const int at = threadIdx.x % TPR;
    const int64_t group = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;
    const int units = (int)p.features / VEC;
    const float scale = 1.f / (float)p.features;
    float w[VPT][VEC], dw[NEXT ? VPT : 1][VEC], db[NEXT ? VPT : 1][VEC];
    Raw<T, VEC> x[VPT], dy[VPT];
    float mean = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t row) {
        if (row >= p.rows || group >= p.partials) return;
        const T *xr = static_cast<const T *>(p.x) + row * p.xs, *dr = static_cast<const T *>(p.dy) + row * p.ys;
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (at + k * TPR < units) {
                x[k].load(xr + (at + k * TPR) * VEC);
                dy[k].load(dr + (at + k * TPR) * VEC);
            }
        mean = p.mean[row];
        rstd = p.rstd[row];
    };
    fetch(group);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            w[k][i] = 1.f;
            if constexpr (NEXT)
                dw[k][i] = db[k][i] = 0.f;
            else
                columns[(k * VEC + i) * TPR + at] = columns[((VPT + k) * VEC + i) * TPR + at] = 0.f;
        }
        if (p.w && at + k * TPR < units) load_parameters<VEC>(p.w, p.parameter, (at + k * TPR) * VEC, w[k]);
    }
    // every group of a block takes the same number of steps (they share its barriers)
    const int64_t steps = (p.rows + p.partials - 1) / p.partials;
    for (int64_t step = 0; step < steps; step++) {
        const int64_t row = group + step * p.partials;
        const bool live = row < p.rows && group < p.partials;
        const float m = mean, r = rstd;
        Raw<T, VEC> x0[VPT], dy0[VPT];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            x0[k] = x[k];
            dy0[k] = dy[k];
            if (live && at + k * TPR < units) {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = dy0[k].at(i), h = (x0[k].at(i) - m) * r, g = d * w[k][i];
                    if constexpr (NEXT) {
                        dw[k][i] = fmaf(d, h, dw[k][i]);
                        db[k][i] += d;
                    } else {
                        float &cw = columns[(k * VEC + i) * TPR + at], &cb = columns[((VPT + k) * VEC + i) * TPR + at];
                        cw = fmaf(d, h, cw);
                        cb += d;
                    }
                    s[0] += g;
                    s[1] = fmaf(g, h, s[1]);
                }
            }
        }
        if (NEXT) fetch(row + p.partials);
        row_sums<TPR>(s, buf[step & 1]);
        if (live && p.dx) {
            T *dx = static_cast<T *>(p.dx) + row * p.xs;
            const float a = s[0] * scale, b = s[1] * scale;
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (at + k * TPR < units) {
                    Vec<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        const float h = (x0[k].at(i) - m) * r, g = dy0[k].at(i) * w[k][i];
                        o.f[i] = r * (g - a - h * b);
                    }
                    o.store(dx + (at + k * TPR) * VEC);
                }
        }
        if (!NEXT) fetch(row + p.partials);
    }
    let_next_start();
    if (!p.part_w || group >= p.partials) return;
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (at + k * TPR < units) {
            const int64_t to = group * p.features + (at + k * TPR) * VEC;
            float a[VEC], b[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                a[i] = NEXT ? dw[NEXT ? k : 0][i] : columns[(k * VEC + i) * TPR + at];
                b[i] = NEXT ? db[NEXT ? k : 0][i] : columns[((VPT + k) * VEC + i) * TPR + at];
            }
            if constexpr (VEC == 1) {
                p.part_w[to] = a[0];
                p.part_b[to] = b[0];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i += 4) {
                    *reinterpret_cast<float4 *>(p.part_w + to + i) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
                    *reinterpret_cast<float4 *>(p.part_b + to + i) = make_float4(b[i], b[i + 1], b[i + 2], b[i + 3]);
                }
            }
        }
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

// Sums of the partials, in order: 32 columns x 8 lanes of partials, weight or bias by blockIdx.y.
template <typename P>
__global__ void __launch_bounds__(kThreads) norm_grad_reduce_kernel(NormGradParams p) {
    __shared__ float part[8][33];
    const int c = threadIdx.x & 31, lane = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    const float *src = blockIdx.y ? p.part_b : p.part_w;
    P *dst = static_cast<P *>(blockIdx.y ? p.db : p.dw);
    wait_for_previous();
    float s = 0.f;
    if (dst && col < p.features) {
#pragma unroll 8
        for (int k = lane; k < p.partials; k += 8) s += src[k * p.features + col];
    }
    part[lane][c] = s;
    __syncthreads();
    if (lane == 0 && dst && col < p.features) {
        for (int k = 1; k < 8; k++) s += part[k][c];
        dst[col] = from_float<P>(s);
    }
}

int grid_of(int64_t n, int64_t most) { return (int)(n < most ? n : most); }

template <typename T>
bool aligned_rows(const void *p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * sizeof(T) % 16 == 0;
}

// Threads and vectors for rows of `units` vectors: the fewest threads that keep a row in registers.
template <typename F>
bool with_row_shape(int64_t units, F &&f) {
    if (units <= 32)
        f(Int<32>(), Int<1>());
    else if (units <= 64)
        f(Int<32>(), Int<2>());
    else if (units <= 128)
        f(Int<32>(), Int<4>());
    else if (units <= 256)
        f(Int<128>(), Int<2>());
    else if (units <= 512)
        f(Int<128>(), Int<4>());
    else if (units <= 1024)
        f(Int<256>(), Int<4>());
    else if (units <= 2048)
        f(Int<512>(), Int<4>());
    else if (units <= 4096)
        f(Int<1024>(), Int<4>());
    else
        return false;
    return true;
}

// The same where a thread also keeps its columns' sums: 16 of them at most, and at 1024 threads in shared memory.
template <int VEC, typename F>
bool with_grad_shape(int64_t units, F &&f) {
    constexpr int MORE = VEC == 1 ? 4 : VEC == 4 ? 4 : 2;
    if (units <= 32)
        f(Int<32>(), Int<1>(), std::true_type());
    else if (units <= 64)
        f(Int<32>(), Int<2>(), std::true_type());
    else if (units <= 128 * MORE)
        f(Int<128>(), Int<MORE>(), std::true_type());
    else if (units <= 256 * MORE)
        f(Int<256>(), Int<MORE>(), std::true_type());
    else if (units <= 512 * MORE)
        f(Int<512>(), Int<MORE>(), std::true_type());
    else if (units <= 1024 * MORE)
        f(Int<1024>(), Int<MORE>(), std::false_type());
    else
        return false;
    return true;
}

}  // namespace

int norm_grad_groups(int64_t rows, int64_t features, int vec) {
    int threads = 0;
    const auto shape = [&](auto tpr, auto, auto) { threads = decltype(tpr)::value; };
    const bool kept = vec == 1   ? with_grad_shape<1>(features, shape)
                      : vec == 4 ? with_grad_shape<4>(features / 4, shape)
                                 : with_grad_shape<8>(features / 8, shape);
    if (!kept) return (int)std::clamp<int64_t>(rows / 64, 1, 64);
    // as many rows at a time as fill the SMs with 512 threads each, but 8 rows or more to a group: its sums cost
    // 8 bytes a column, written and read
    const int64_t most = (int64_t)kSms * std::max(1, std::min(8, 512 / threads));
    return (int)std::clamp<int64_t>(rows / 8, 1, most);
}

cudaError_t launch_norm(const NormParams &args, Element e, Element param, cudaStream_t s) {
    NormParams p = args;
    p.parameter = param;
    return with_element(e, [&](auto t) {
        using T = decltype(t);
        constexpr int VEC = 16 / sizeof(T);
        const auto in_registers = [&](auto vec) {
            return with_row_shape(p.features / decltype(vec)::value, [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value, ROWS = TPR < 128 ? 128 / TPR : 1;
                before_launch();
                norm_kernel<T, decltype(vec)::value, TPR, decltype(vpt)::value>
                    <<<(unsigned)((p.rows + ROWS - 1) / ROWS), TPR < 128 ? 128 : TPR, 0, s>>>(p);
            });
        };
        const bool wide = p.features % VEC == 0 && aligned_rows<T>(p.x, p.xs) && aligned_rows<T>(p.y, p.ys) &&
                          aligned_rows<T>(p.w, 0) && aligned_rows<T>(p.b, 0);
        const bool few = p.rows < (int64_t(1) << 31);  // a launch's CTAs
        if (!few || !(wide ? in_registers(Int<VEC>()) : in_registers(Int<1>())))
            with_element(param, [&](auto q) {
                before_launch();
                norm_long_kernel<T, decltype(q)><<<grid_of(p.rows, 1 << 30), kThreads, 0, s>>>(p);
                return cudaSuccess;
            });
        return cudaGetLastError();
    });
}

cudaError_t launch_norm_grad(const NormGradParams &args, Element e, Element param, cudaStream_t s) {
    NormGradParams p = args;
    p.parameter = param;
    const bool sums = p.dw || p.db;
    return with_element(e, [&](auto t) {
        using T = decltype(t);
        constexpr int VEC = 16 / sizeof(T);
        const bool wide = p.features % VEC == 0 && aligned_rows<T>(p.x, p.xs) && aligned_rows<T>(p.dy, p.ys) &&
                          aligned_rows<T>(p.dx, p.xs) && aligned_rows<T>(p.w, 0);
        p.partials = norm_grad_groups(p.rows, p.features, wide ? VEC : 1);
        p.part_b = p.part_w ? p.part_w + (size_t)p.partials * p.features : nullptr;
        cudaError_t started = cudaSuccess;
        const auto in_registers = [&](auto vec) {
            constexpr int V = decltype(vec)::value;
            return with_grad_shape<V>(p.features / V, [&](auto tpr, auto vpt, auto next) {
                constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value, GROUPS = TPR < 256 ? 256 / TPR : 1;
                constexpr bool NEXT = decltype(next)::value;
                started = launch(norm_grad_kernel<T, V, TPR, VPT, NEXT>, dim3((p.partials + GROUPS - 1) / GROUPS),
                                 TPR < 256 ? 256 : TPR, NEXT ? 0 : 2 * VPT * V * TPR * (int)sizeof(float), false, s, p);
            });
        };
        return with_element(param, [&](auto q) {
            using P = decltype(q);
            if (!(wide ? in_registers(Int<VEC>()) : in_registers(Int<1>()))) {
                // the sums first: dx may take the place of dy
                if (sums) {
                    before_launch();
                    norm_grad_columns_kernel<T><<<dim3((unsigned)((p.features + 31) / 32), p.partials), kThreads, 0, s>>>(p);
                }
                if (p.dx) {
                    before_launch();
                    norm_grad_long_kernel<T, P><<<grid_of(p.rows, 1 << 30), kThreads, 0, s>>>(p);
                }
            }
            cudaError_t err = started != cudaSuccess ? started : cudaGetLastError();
            if (err == cudaSuccess && sums)
                err = launch(norm_grad_reduce_kernel<P>, dim3((unsigned)((p.features + 31) / 32), 2), kThreads, 0, true, s, p);
            return err;
        });
    });
}

}  // namespace b200fft
