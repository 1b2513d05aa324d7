// Linear attention by chunks of tokens for everything that the tcgen05 kernels do not take: f32, head dimensions up to
// 256 of any size, any strides and addresses.
//
// The same products as there, on tf32 matrix instructions with every f32 operand in two parts of 11 bits: a b = ah bh +
// ah bl + al bh, off by 2^-22 (16-bit inputs are one part).  A CTA takes 64 value columns of one segment of one head of
// one sequence; the tile of the state that a warp updates stays in its registers as the accumulator of its products.
#include <algorithm>

#include "segments.cuh"

namespace b200fft {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSlice = 64;  // value columns of a CTA

// Row pitches in floats that keep the fragments' reads free of bank conflicts: rows by lane / 4 and columns by
// lane % 4 (pitch 20 mod 32: keys are also read the other way round), and the other way round (8 mod 32).
constexpr int pitch_by_row(int n) { return n / 32 * 32 + 20; }
constexpr int pitch_by_column(int n) { return n / 32 * 32 + 8; }
static_assert(pitch_by_row(32) >= 32 + 4, "pitch");

template <int DK>
struct BlockLayout {
    static constexpr int C = DK > 128 ? 32 : 64;  // tokens of a chunk
    static constexpr int key_pitch = pitch_by_row(DK), value_pitch = pitch_by_column(kSlice), score_pitch = pitch_by_row(C);
    static constexpr int q = 0, k = q + C * key_pitch, v = k + C * key_pitch, p = v + C * value_pitch,
                         s = p + C * score_pitch, pw = s + DK * value_pitch, weight = pw + C + 4, end = weight + C;
    static constexpr int bytes = end * 4;
};

// A fragment's elements: rounded to 11 bits, and what is left (of either sign), of which the instruction sees 11 bits:
// 2^-22 of the element is lost, to either side.  (cvt.rna.tf32 for both parts made 15 instructions for each matrix
// instruction, and 57 us of 2 x 1023 x 8 heads x 64 x 96 where this takes 48; cutting the first part off, too, one
// instruction less, left 7e-7 of the result, to one side.)
template <int N, bool WHOLE>
struct Parts {
    uint32_t hi[N], lo[WHOLE ? 1 : N];
    __device__ __forceinline__ void set(int i, float x) {
        if (WHOLE) {
            hi[i] = __float_as_uint(x);
        } else {
            hi[i] = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
            lo[i] = __float_as_uint(x - __uint_as_float(hi[i]));
        }
    }
};
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// c += the products of two steps of eight.  The instruction cuts sums off where f32 rounds; so those sixteen are added up
// by themselves, and to the rest in f32 (added to it by the instruction, 128 of them were off by 2e-6, to one side).
template <bool WA, bool WB>
__device__ __forceinline__ void multiply(float (&c)[4], const Parts<4, WA> (&a)[2], const Parts<2, WB> (&b)[2]) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if constexpr (!WA) mma_tf32(x, a[k].lo, b[k].hi);
        if constexpr (!WB) mma_tf32(x, a[k].hi, b[k].lo);
    }
#pragma unroll
    for (int k = 0; k < 2; k++) mma_tf32(x, a[k].hi, b[k].hi);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] += x[i];
}
// Fragments of two steps: A's rows by lane / 4, its eight columns by lane % 4 (or, for B, rows and columns changed).
template <bool W>
__device__ __forceinline__ void fragment_a(Parts<4, W> (&a)[2], const float *p, int pitch) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        a[k].set(0, p[8 * k]), a[k].set(1, p[8 * k + 8 * pitch]);
        a[k].set(2, p[8 * k + 4]), a[k].set(3, p[8 * k + 4 + 8 * pitch]);
    }
}
template <bool W>
__device__ __forceinline__ void fragment_b(Parts<2, W> (&b)[2], const float *p, int step) {  // `step` floats from k to k + 1
#pragma unroll
    for (int k = 0; k < 2; k++) b[k].set(0, p[8 * k * step]), b[k].set(1, p[(8 * k + 4) * step]);
}

// C rows x COLS columns into shared memory as f32; rows outside [first, end) and columns from `cols` on are zero.
// Tells whether this thread met an infinity or NaN.
template <typename T, int C, int COLS>
__device__ __forceinline__ bool load_tile(float *dst, int pitch, const T *src, int64_t stride, int first, int end, int cols) {
    constexpr int VEC = 16 / sizeof(T);
    bool odd = false;
    if (cols % VEC == 0 && stride % VEC == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        constexpr int PER = COLS / VEC;
        static_assert(C * PER % kThreads == 0, "whole rounds");
#pragma unroll 4
        for (int u = threadIdx.x; u < C * PER; u += kThreads) {
            const int r = u / PER, c = u % PER * VEC;
            float f[VEC];
            if (r >= first && r < end && c < cols) {
                const uint4 w = *reinterpret_cast<const uint4 *>(src + r * stride + c);
                const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (int i = 0; i < VEC; i++) f[i] = to_float(e[i]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) f[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                *reinterpret_cast<float4 *>(dst + r * pitch + c + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
                odd |= !(fabsf(f[i]) + fabsf(f[i + 1]) + fabsf(f[i + 2]) + fabsf(f[i + 3]) <= 3.4e38f);
            }
        }
    } else {
#pragma unroll 8
        for (int u = threadIdx.x; u < C * COLS; u += kThreads) {
            const int r = u / COLS, c = u % COLS;
            const float f = r >= first && r < end && c < cols ? to_float(src[r * stride + c]) : 0.f;
            dst[r * pitch + c] = f;
            odd |= !(fabsf(f) <= 3.4e38f);
        }
    }
    return odd;
}

// SUM: only the segment's own sum of the state, into the workspace.
template <typename T, int DK, bool SUM>
__global__ void __launch_bounds__(kThreads) block_kernel(const __grid_constant__ Passes all) {
    using L = BlockLayout<DK>;
    constexpr int C = L::C;
    constexpr bool WHOLE = sizeof(T) == 2;                 // the inputs fit one part
    constexpr int ROW_TILES = C / 16, ACROSS = kWarps / ROW_TILES;
    constexpr int SCORE_TILES = C / 8 / ACROSS, OUT_TILES = kSlice / 8 / ACROSS;
    constexpr int STATE_ROWS = DK >= 128 ? DK / 128 : 1;   // 16-row tiles of the state that a warp keeps
    constexpr int STATE_ACROSS = DK >= 128 ? 1 : 128 / DK, STATE_TILES = kSlice / 8 / STATE_ACROSS;
    extern __shared__ __align__(16) float shared[];
    float *const sq = shared + L::q, *const sk = shared + L::k, *const sv = shared + L::v, *const sp = shared + L::p,
                 *const ss = shared + L::s, *const pw = shared + L::pw, *const weight = shared + L::weight;
    __shared__ int first_odd;

    const int b = blockIdx.z % (unsigned)all.pass[0].p.batch;
    const MixPass &cp = all.pass[blockIdx.z / (unsigned)all.pass[0].p.batch];
    const MixParams &p = cp.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int slices = gridDim.y / p.heads;
    const int segment = blockIdx.x, h = blockIdx.y / slices, c0 = blockIdx.y % slices * kSlice;
    const int cols = min(kSlice, p.dv - c0);
    // (the pass after a sum: that has waited for the inputs)
    if (SUM || cp.count == 1) wait_for_previous();
    const Line line(cp, segment, h, b);
    if (!SUM && (segment > line.last || c0 >= p.dv)) wait_for_previous();
    if (SUM) let_next_start();
    if (c0 >= p.dv) return;  // the widest pass decides the grid
    if (segment > line.last || (SUM && ((segment == line.last && !p.s_out) || line.count == 0))) return;
    const int chunks = (line.tokens + C - 1) / C;  // none for an empty sequence, whose state passes through
    const float log_decay = p.log_decay[h];
    for (int i = tid; i <= C; i += kThreads) pw[i] = i ? (float)exp((double)log_decay * i) : 1.f;

    // this warp's tile of the state: rows state_row + g, + 8, columns state_col + 8 n + 2 t, + 1
    const int state_row = warp / STATE_ACROSS * 16 * STATE_ROWS, state_col = warp % STATE_ACROSS * STATE_TILES * 8;
    float s[STATE_ROWS][STATE_TILES][4];
    float *const own = segment_state(cp, b, h, segment);
    if (!SUM && cp.count > 1) wait_for_previous();
    if (!SUM) let_next_start();
    const float *in = SUM ? nullptr : cp.count > 1 ? own : p.s_in && line.kept ? p.s_in + line.user : nullptr;
    float *out = SUM ? own : cp.count == 1 && p.s_out && line.kept ? p.s_out + line.user : nullptr;
    const int64_t in_k = cp.count > 1 ? p.dv : p.state_k, in_v = cp.count > 1 ? 1 : p.state_v;  // of `out` too
#pragma unroll
    for (int m = 0; m < STATE_ROWS; m++)
#pragma unroll
        for (int n = 0; n < STATE_TILES; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = state_row + 16 * m + g + (e >> 1) * 8, c = state_col + 8 * n + 2 * t + (e & 1);
                s[m][n][e] = in && r < p.dk && c < cols ? in[r * in_k + (c0 + c) * in_v] : 0.f;
            }
    auto publish_state = [&] {
#pragma unroll
        for (int m = 0; m < STATE_ROWS; m++)
#pragma unroll
            for (int n = 0; n < STATE_TILES; n++)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    *reinterpret_cast<float2 *>(ss + (state_row + 16 * m + g + e * 4) * L::value_pitch + state_col + 8 * n + 2 * t) =
                        make_float2(s[m][n][e], s[m][n][e + 1]);
    };

    const T *q = static_cast<const T *>(p.q.p) + (p.offsets ? 0 : b * p.q.sb) + (h / p.q.per_head) * p.q.sh;
    const T *k = static_cast<const T *>(p.k.p) + (p.offsets ? 0 : b * p.k.sb) + (h / p.k.per_head) * p.k.sh;
    const T *v = static_cast<const T *>(p.v.p) + (p.offsets ? 0 : b * p.v.sb) + (h / p.v.per_head) * p.v.sh + c0;
    const int64_t out_at = (p.offsets ? 0 : b * p.osb) + h * p.osh + c0;
    auto write = [&](int64_t row, int col, float y) {
        if (cp.out_f32)
            static_cast<float *>(p.o)[out_at + row * p.ost + col] = y;
        else
            static_cast<T *>(p.o)[out_at + row * p.ost + col] = from_float<T>(y);
    };
    const int row0 = warp / ACROSS * 16;  // of the chunk, for scores and results
    const float inside = p.update * p.out;
    int powers_of = 0;
    Fade keep{1.f, 0.f};

    for (int c = 0; c < chunks; c++) {
        const int at = line.from + c * C, n = min(C, line.tokens - c * C);
        const int first = p.reverse ? C - n : 0, end = first + n;  // valid tile rows
        const int64_t start = line.start + (p.reverse ? line.count - at - C : at);
        __syncthreads();  // nobody reads the tiles any more
        if (n != powers_of) {
            powers_of = n;
            keep = fade_of((double)log_decay * n);
            for (int r = tid; r < C; r += kThreads)
                weight[r] = r >= first && r < end ? p.update * pw[p.reverse ? r + 1 - first : end - 1 - r] : 0.f;
        }
        load_tile<T, C, DK>(sk, L::key_pitch, k + start * p.k.st, p.k.st, first, end, p.dk);
        bool odd = load_tile<T, C, kSlice>(sv, L::value_pitch, v + start * p.v.st, p.v.st, first, end, cols);
        if (!SUM) {
            load_tile<T, C, DK>(sq, L::key_pitch, q + start * p.q.st, p.q.st, first, end, p.dk);
            publish_state();
        }
        const bool careful = __syncthreads_or(odd);

        if (!SUM) {
            // scores
            float x[SCORE_TILES][4] = {};
            const int col0 = warp % ACROSS * SCORE_TILES * 8;
            const bool none = p.reverse ? col0 + SCORE_TILES * 8 <= row0 : col0 >= row0 + 16;
            if (!none) {
#pragma unroll 2
                for (int d = 0; d < DK; d += 16) {
                    Parts<4, WHOLE> a[2];
                    fragment_a(a, sq + (row0 + g) * L::key_pitch + d + t, L::key_pitch);
#pragma unroll
                    for (int m = 0; m < SCORE_TILES; m++) {
                        Parts<2, WHOLE> w[2];
                        fragment_b(w, sk + (col0 + 8 * m + g) * L::key_pitch + d + t, 1);
                        multiply(x[m], a, w);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < SCORE_TILES; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = row0 + g + (e >> 1) * 8, j = col0 + 8 * m + 2 * t + (e & 1), gap = p.reverse ? j - i : i - j;
                    sp[i * L::score_pitch + j] = gap >= 0 ? x[m][e] * (inside * pw[max(gap, 0)]) : 0.f;
                }
        }

        // state
#pragma unroll
        for (int m = 0; m < STATE_ROWS; m++)
#pragma unroll
            for (int j = 0; j < STATE_TILES; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[m][j][e] = faded(s[m][j][e], keep);
        if (state_col < cols) {
#pragma unroll 1
            for (int r = 0; r < C; r += 16) {
                Parts<4, false> a[STATE_ROWS][2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int r0 = r + 8 * k + t;
                    const float w0 = weight[r0], w1 = weight[r0 + 4];
#pragma unroll
                    for (int m = 0; m < STATE_ROWS; m++) {
                        const float *ka = sk + r0 * L::key_pitch + state_row + 16 * m + g;
                        a[m][k].set(0, ka[0] * w0), a[m][k].set(1, ka[8] * w0);
                        a[m][k].set(2, ka[4 * L::key_pitch] * w1), a[m][k].set(3, ka[4 * L::key_pitch + 8] * w1);
                    }
                }
#pragma unroll
                for (int j = 0; j < STATE_TILES; j++) {
                    Parts<2, WHOLE> w[2];
                    fragment_b(w, sv + (r + t) * L::value_pitch + state_col + 8 * j + g, L::value_pitch);
#pragma unroll
                    for (int m = 0; m < STATE_ROWS; m++) multiply(s[m][j], a[m], w);
                }
            }
        }
        if (SUM) continue;
        __syncthreads();

        // Infinities and NaN among the values: a masked score of zero times them would spread them to tokens before
        // them.  The rows from the first of them on are summed one by one; the others' product goes without them.
        int stop = C;
        if (careful) {
            if (tid == 0) first_odd = C;
            __syncthreads();
            for (int u = tid; u < C * kSlice; u += kThreads)
                if (!(fabsf(sv[u / kSlice * L::value_pitch + u % kSlice]) <= 3.4e38f))
                    atomicMin(&first_odd, p.reverse ? C - 1 - u / kSlice : u / kSlice);
            __syncthreads();
            stop = first_odd;
            for (int u = tid; u < C * kSlice; u += kThreads) {
                const int i = u / kSlice, col = u % kSlice;
                if (i < first || i >= end || col >= cols || (p.reverse ? C - 1 - i : i) < stop) continue;
                float state = 0.f, sum = 0.f;
                for (int d = 0; d < DK; d++) state = fmaf(sq[i * L::key_pitch + d], ss[d * L::value_pitch + col], state);
                for (int j = p.reverse ? i : 0; j < (p.reverse ? C : i + 1); j++)
                    sum = fmaf(sp[i * L::score_pitch + j], sv[j * L::value_pitch + col], sum);
                if (p.o) write(start + i, col, fmaf(p.out * pw[p.reverse ? C - 1 - i : i + 1], state, sum));
            }
            __syncthreads();
            for (int u = tid; u < C * kSlice; u += kThreads) {
                float &f = sv[u / kSlice * L::value_pitch + u % kSlice];
                if (!(fabsf(f) <= 3.4e38f)) f = 0.f;
            }
            __syncthreads();
        }

        // results: the state's part, faded by row, and the part inside the chunk
        const int col0 = warp % ACROSS * OUT_TILES * 8;
        float y[OUT_TILES][4] = {};
        if (col0 >= cols) continue;  // columns past the last
#pragma unroll 2
        for (int d = 0; d < DK; d += 16) {
            Parts<4, WHOLE> a[2];
            fragment_a(a, sq + (row0 + g) * L::key_pitch + d + t, L::key_pitch);
#pragma unroll
            for (int m = 0; m < OUT_TILES; m++) {
                Parts<2, false> w[2];
                fragment_b(w, ss + (d + t) * L::value_pitch + col0 + 8 * m + g, L::value_pitch);
                multiply(y[m], a, w);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = row0 + g + (e >> 1) * 8;
            const float fade = p.out * pw[p.reverse ? C - 1 - i : i + 1];
#pragma unroll
            for (int m = 0; m < OUT_TILES; m++) y[m][e] *= fade;
        }
        const int from = p.reverse ? row0 : 0, to = p.reverse ? C : row0 + 16;  // columns of scores that this row tile has
#pragma unroll 1
        for (int j = from; j < to; j += 16) {
            Parts<4, false> a[2];
            fragment_a(a, sp + (row0 + g) * L::score_pitch + j + t, L::score_pitch);
#pragma unroll
            for (int m = 0; m < OUT_TILES; m++) {
                Parts<2, WHOLE> w[2];
                fragment_b(w, sv + (j + t) * L::value_pitch + col0 + 8 * m + g, L::value_pitch);
                multiply(y[m], a, w);
            }
        }
#pragma unroll
        for (int m = 0; m < OUT_TILES; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = row0 + g + (e >> 1) * 8, col = col0 + 8 * m + 2 * t + (e & 1);
                if (p.o && i >= first && i < end && (p.reverse ? C - 1 - i : i) < stop && col < cols) write(start + i, col, y[m][e]);
            }
    }

    if (!out) return;
#pragma unroll
    for (int m = 0; m < STATE_ROWS; m++)
#pragma unroll
        for (int j = 0; j < STATE_TILES; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = state_row + 16 * m + g + (e >> 1) * 8, col = state_col + 8 * j + 2 * t + (e & 1);
                if (r < p.dk && col < cols) out[r * in_k + (c0 + col) * in_v] = s[m][j][e];
            }
}

template <typename T, int DK>
cudaError_t launch_dims(const Passes &all, int passes, cudaStream_t s) {
    const MixPass &first = all.pass[0];
    int slices = 1;
    for (int k = 0; k < passes; k++) slices = std::max(slices, (all.pass[k].p.dv + kSlice - 1) / kSlice);
    const dim3 grid(first.count, first.p.heads * slices, (unsigned)first.p.batch * passes);
    if (first.count > 1) {
        cudaError_t e = launch(block_kernel<T, DK, true>, grid, kThreads, BlockLayout<DK>::bytes, s, all);
        if (e == cudaSuccess) e = launch_enter(all, passes, s);
        if (e != cudaSuccess) return e;
    }
    return launch(block_kernel<T, DK, false>, grid, kThreads, BlockLayout<DK>::bytes, s, all);
}

}  // namespace

bool chunked_tf32_takes(const MixPass &pass) {
    const MixParams &p = pass.p;
    const int64_t tokens = p.offsets ? p.packed_tokens : p.length;
    if ((int64_t)p.heads * 4 > 65535) return false;  // the grid's second axis: up to four slices of a head
    return p.length >= 2 && tokens > 0 && std::max(tokens, p.length) <= int64_t(1) << 30;  // rows are counted in 32 bits
}

int chunked_tf32_shape(const MixPass &pass) { return pass.p.dk <= 64 ? 64 : pass.p.dk <= 128 ? 128 : 256; }

cudaError_t launch_chunked_tf32(const MixPass *passes, int n, Element e, cudaStream_t s) {
    Passes all{};
    for (int k = 0; k < n; k++) all.pass[k] = passes[k];
    return with_element(e, [&](auto v) {
        using T = decltype(v);
        switch (chunked_tf32_shape(passes[0])) {
            case 64: return launch_dims<T, 64>(all, n, s);
            case 128: return launch_dims<T, 128>(all, n, s);
            default: return launch_dims<T, 256>(all, n, s);
        }
    });
}

}  // namespace b200fft
