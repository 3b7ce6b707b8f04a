// Layer norm over rows and its backward pass.
//
//   forward   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  y = (x - m) r w + b
//   backward  g = dL_dy w,  u = (x - m) r,  dx = r (g - mean g - u mean(g u)),  dw = sum of dL_dy u,  db = sum of dL_dy
//
// Both passes read each array once: a row stays in the registers of a group of GROUP threads (a part of a wave for
// narrow rows, a workgroup for wide ones) from the first sum to the result, and the variance is taken about the mean
// rather than as a difference of two large numbers.  The weight's and bias's gradients gather in registers over the
// rows a workgroup walks through; the workgroups' sums are joined in order by a second kernel.
//
// Bound by memory: 1920 x 1080 x 64 float32 there and back moves 2.65 GB (x is read by both passes) in 488 us, 5.4 TB/s;
// 8191 x 5001 float16 410 MB in 133 us, of which rows that start off a word's boundary cost a quarter (5000 wide: 101 us).
#include "decoder_common.h"

#define NORM_WAVE_BLOCKS 1024  // workgroups of the kernels that give a row to a wave or less: what fills the chip

template <int GROUP, int THREADS>
struct Groups {
    // sum over a group's threads, the same on all of them; `buf` holds a float per wave
    static __device__ __forceinline__ float sum(float v, float* buf)
    {
#pragma unroll
        for (int d = 1; d < (GROUP < 64 ? GROUP : 64); d <<= 1) v += __shfl_xor(v, d);
        if (GROUP > 64) {
            const int wave = threadIdx.x >> 6;
            __syncthreads();
            if ((threadIdx.x & 63) == 0) buf[wave] = v;
            __syncthreads();
            v = 0.0f;
#pragma unroll
            for (int k = 0; k < THREADS / 64; k++) v += buf[k];
        }
        return v;
    }
    // two sums at once
    static __device__ __forceinline__ void sum2(float& v, float& w, float* buf)
    {
#pragma unroll
        for (int d = 1; d < (GROUP < 64 ? GROUP : 64); d <<= 1) {
            v += __shfl_xor(v, d);
            w += __shfl_xor(w, d);
        }
        if (GROUP > 64) {
            const int wave = threadIdx.x >> 6;
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                buf[wave] = v;
                buf[THREADS / 64 + wave] = w;
            }
            __syncthreads();
            v = w = 0.0f;
#pragma unroll
            for (int k = 0; k < THREADS / 64; k++) {
                v += buf[k];
                w += buf[THREADS / 64 + k];
            }
        }
    }
};

// A chunk's weights as they lie in memory (N of them: one or two 16-byte pieces), `other` where there is none: they stay
// packed in registers between rows, which leaves room for the next row's loads.
template <typename W, int N>
struct Weights {
    W e[N];
    __device__ __forceinline__ void load(const W* p, long long at, long long valid, float other)
    {
#pragma unroll
        for (int i = 0; i < N; i++) e[i] = (W)other;
        if (!p || valid <= 0) return;
        if (valid >= N) {
            __builtin_memcpy(e, p + at, sizeof e);
        } else {
#pragma unroll
            for (int i = 0; i < N - 1; i++)
                if (i < valid) e[i] = p[at + i];
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)e[i]; }
};

// Whether a group has its next row on the way while it works on one: worth its registers for narrow rows and for groups
// of several waves, which stand at barriers together; a lone wave with much to hold makes room for other waves instead
// (100000 x 1024 bfloat16 there and back: 223 us ahead, 208 us not; 8191 x 5001 float16: 144 us and 172 us).  Four chunks of
// 16-bit types are more than the backward pass has registers for: 64 to 124 bytes a lane go to memory and back for every
// row (8191 x 6144 float16 there and back 116 us, 8192 wide 188 us; 4096 x 12288 120 us, 16384 wide 240 us).
template <int GROUP, int NC>
constexpr bool norm_reads_ahead() { return GROUP <= 64 ? NC == 1 : GROUP < 1024; }

template <typename T, typename W>
struct NormArgs {
    long long rows;
    int width;
    float eps, width_f;  // sums are divided, not multiplied by a rounded reciprocal: a constant row has its value as mean
    const T* x;
    long long ldx;
    const W *weight, *bias;
    T* y;
    float *mean, *rstd;
};

template <typename T, typename W, int GROUP, int NC, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_forward_kernel(NormArgs<T, W> a)
{
    constexpr int N = Chunk<T>::N, SLOTS = THREADS / GROUP;
    __shared__ float buf[THREADS / 64];
    const int me = threadIdx.x % GROUP, slot = threadIdx.x / GROUP;
    Weights<W, N> w[NC], b[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = (c * GROUP + me) * N;
        w[c].load(a.weight, col, a.width - col, 1.0f);
        b[c].load(a.bias, col, a.width - col, 0.0f);
    }
    // (a group without a row goes through the motions: the sums of a workgroup-wide group meet at barriers)
    u32x4 next[NC];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int col = (c * GROUP + me) * N;
            next[c] = load16_head(a.x + row * a.ldx + col, row < a.rows ? a.width - col : 0);
        }
    };
    constexpr bool AHEAD = norm_reads_ahead<GROUP, NC>();
    const long long stride = (long long)gridDim.x * SLOTS;
    long long first = (long long)blockIdx.x * SLOTS;
    if (AHEAD) fetch(first + slot);
    for (; first < a.rows; first += stride) {
        const long long row = first + slot;
        if (!AHEAD) fetch(row);
        float v[NC][N], s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            unpack<T>(next[c], v[c]);
#pragma unroll
            for (int i = 0; i < N; i++) s += v[c][i];
        }
        if (AHEAD && first + stride < a.rows) fetch(row + stride);
        const float mean = Groups<GROUP, THREADS>::sum(s, buf) / a.width_f;
        s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int valid = a.width - (c * GROUP + me) * N;
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[c][i] -= mean;
                s += i < valid ? v[c][i] * v[c][i] : 0.0f;
            }
        }
        const float rstd = 1.0f / sqrtf(Groups<GROUP, THREADS>::sum(s, buf) / a.width_f + a.eps);
        if (row >= a.rows) continue;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int col = (c * GROUP + me) * N;
            float y[N];
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = v[c][i] * rstd * w[c][i] + b[c][i];
            store16_head(a.y + row * a.width + col, pack<T>(y), a.width - col);
        }
        if (me == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// Rows that do not fit the registers of a workgroup: the row is read three times, the last two from cache if it fits.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_forward_wide_kernel(NormArgs<T, W> a)
{
    constexpr int N = Chunk<T>::N, STEP = 1024 * N;
    __shared__ float buf[16];
    const long long row = blockIdx.x;
    const T* const x = a.x + row * a.ldx;
    const int first = threadIdx.x * N;
    float s = 0.0f, f[N];
    for (long long col = first; col < a.width; col += STEP) {
        unpack<T>(load16_head(x + col, a.width - col), f);
#pragma unroll
        for (int i = 0; i < N; i++) s += f[i];
    }
    const float mean = Groups<1024, 1024>::sum(s, buf) / a.width_f;
    s = 0.0f;
    for (long long col = first; col < a.width; col += STEP) {
        unpack<T>(load16_head(x + col, a.width - col), f);
#pragma unroll
        for (int i = 0; i < N; i++) s += col + i < a.width ? (f[i] - mean) * (f[i] - mean) : 0.0f;
    }
    const float rstd = 1.0f / sqrtf(Groups<1024, 1024>::sum(s, buf) / a.width_f + a.eps);
    for (long long col = first; col < a.width; col += STEP) {
        const int valid = (int)(a.width - col < N ? a.width - col : N);
        Weights<W, N> w, b;
        w.load(a.weight, col, valid, 1.0f);
        b.load(a.bias, col, valid, 0.0f);
        unpack<T>(load16_head(x + col, valid), f);
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = (f[i] - mean) * rstd * w[i] + b[i];
        store16_head(a.y + row * a.width + col, pack<T>(f), valid);
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
}

template <typename T, typename W>
struct NormBackwardArgs {
    long long rows;
    int width;
    float width_f;
    const T *x, *dy;
    long long ldx, lddy;
    const W* weight;
    const float *mean, *rstd;
    T* dx;
    float* partial;  // [workgroup][2][width]: sums of dy u, then of dy; NULL: not wanted
};

template <typename T, typename W, int GROUP, int NC, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS <= 256 ? 2 : 1) void norm_backward_kernel(NormBackwardArgs<T, W> a)
{
    constexpr int N = Chunk<T>::N, SLOTS = THREADS / GROUP;
    __shared__ float buf[2 * (THREADS / 64)];
    __shared__ float join[SLOTS > 1 ? 2 * N * THREADS : 1];
    const int me = threadIdx.x % GROUP, slot = threadIdx.x / GROUP;
    Weights<W, N> w[NC];
    float dw[NC][N], db[NC][N];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = (c * GROUP + me) * N;
        w[c].load(a.weight, col, a.width - col, 1.0f);
#pragma unroll
        for (int i = 0; i < N; i++) dw[c][i] = db[c][i] = 0.0f;
    }
    u32x4 nx[NC], ng[NC];
    float nmean = 0.0f, nrstd = 0.0f;
    auto fetch = [&](long long row) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int col = (c * GROUP + me) * N, valid = row < a.rows ? a.width - col : 0;
            nx[c] = load16_head(a.x + row * a.ldx + col, valid);
            ng[c] = load16_head(a.dy + row * a.lddy + col, valid);
        }
        nmean = row < a.rows ? a.mean[row] : 0.0f;
        nrstd = row < a.rows ? a.rstd[row] : 0.0f;
    };
    constexpr bool AHEAD = norm_reads_ahead<GROUP, NC>();
    const long long stride = (long long)gridDim.x * SLOTS;
    long long first = (long long)blockIdx.x * SLOTS;
    if (AHEAD) fetch(first + slot);
    for (; first < a.rows; first += stride) {
        const long long row = first + slot;
        const bool there = row < a.rows;
        if (!AHEAD) fetch(row);
        const float mean = nmean, rstd = nrstd;
        float u[NC][N], g[NC][N], sg = 0.0f, sgu = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            unpack<T>(nx[c], u[c]);
            unpack<T>(ng[c], g[c]);
            // (behind the row's end dy is zero, and u is of no account)
#pragma unroll
            for (int i = 0; i < N; i++) {
                u[c][i] = (u[c][i] - mean) * rstd;
                dw[c][i] += g[c][i] * u[c][i];
                db[c][i] += g[c][i];
                g[c][i] *= w[c][i];
                sg += g[c][i];
                sgu += g[c][i] * u[c][i];
            }
        }
        if (AHEAD && first + stride < a.rows) fetch(row + stride);
        if (!a.dx) continue;
        Groups<GROUP, THREADS>::sum2(sg, sgu, buf);
        const float mg = sg / a.width_f, mgu = sgu / a.width_f;
        if (!there) continue;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int col = (c * GROUP + me) * N;
            float d[N];
#pragma unroll
            for (int i = 0; i < N; i++) d[i] = rstd * (g[c][i] - mg - u[c][i] * mgu);
            store16_head(a.dx + row * a.width + col, pack<T>(d), a.width - col);
        }
    }
    if (!a.partial) return;
    float* const out = a.partial + (long long)blockIdx.x * 2 * a.width;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = (c * GROUP + me) * N;
        if (SLOTS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; i++) {
                join[i * THREADS + threadIdx.x] = dw[c][i];
                join[(N + i) * THREADS + threadIdx.x] = db[c][i];
            }
            __syncthreads();
            if (slot != 0) continue;
#pragma unroll
            for (int i = 0; i < N; i++) {
                float sw = 0.0f, sb = 0.0f;
#pragma unroll 4
                for (int k = 0; k < SLOTS; k++) {
                    sw += join[i * THREADS + k * GROUP + me];
                    sb += join[(N + i) * THREADS + k * GROUP + me];
                }
                dw[c][i] = sw;
                db[c][i] = sb;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (col + i < a.width) {
                out[col + i] = dw[c][i];
                out[a.width + col + i] = db[c][i];
            }
        }
    }
}

// dx of rows that do not fit the registers of a workgroup
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_backward_wide_kernel(NormBackwardArgs<T, W> a)
{
    constexpr int N = Chunk<T>::N, STEP = 1024 * N;
    __shared__ float buf[32];
    const long long row = blockIdx.x;
    const T *const x = a.x + row * a.ldx, *const dy = a.dy + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    const int first = threadIdx.x * N;
    float sg = 0.0f, sgu = 0.0f, u[N], g[N];
    Weights<W, N> w;
    for (long long col = first; col < a.width; col += STEP) {
        w.load(a.weight, col, a.width - col, 1.0f);
        unpack<T>(load16_head(x + col, a.width - col), u);
        unpack<T>(load16_head(dy + col, a.width - col), g);
#pragma unroll
        for (int i = 0; i < N; i++) {
            sg += g[i] * w[i];
            sgu += g[i] * w[i] * ((u[i] - mean) * rstd);
        }
    }
    Groups<1024, 1024>::sum2(sg, sgu, buf);
    const float mg = sg / a.width_f, mgu = sgu / a.width_f;
    for (long long col = first; col < a.width; col += STEP) {
        w.load(a.weight, col, a.width - col, 1.0f);
        unpack<T>(load16_head(x + col, a.width - col), u);
        unpack<T>(load16_head(dy + col, a.width - col), g);
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = rstd * (g[i] * w[i] - mg - (u[i] - mean) * rstd * mgu);
        store16_head(a.dx + row * a.width + col, pack<T>(u), a.width - col);
    }
}

// Column sums of the same: a thread per chunk of columns, the workgroups (y) share the rows.
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormBackwardArgs<T, W> a)
{
    constexpr int N = Chunk<T>::N;
    const long long col = ((long long)blockIdx.x * 256 + threadIdx.x) * N;
    if (col >= a.width) return;
    float dw[N], db[N], u[N], g[N];
#pragma unroll
    for (int i = 0; i < N; i++) dw[i] = db[i] = 0.0f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        unpack<T>(load16_head(a.x + row * a.ldx + col, a.width - col), u);
        unpack<T>(load16_head(a.dy + row * a.lddy + col, a.width - col), g);
#pragma unroll
        for (int i = 0; i < N; i++) {
            dw[i] += g[i] * ((u[i] - mean) * rstd);
            db[i] += g[i];
        }
    }
    float* const out = a.partial + (long long)blockIdx.y * 2 * a.width;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (col + i < a.width) {
            out[col + i] = dw[i];
            out[a.width + col + i] = db[i];
        }
    }
}

// ---------------------------------------------------------------------------
// Launch shapes: threads per row and chunks per thread by the number of 16-byte chunks of a row
// ---------------------------------------------------------------------------
enum NormShape { G1, G2, G4, G8, G16, G32, G64, G64x2, G64x3, G64x4, G256x2, G256x3, G256x4, G512x3, G512x4, G1024x3, G1024x4, NORM_WIDE };

static NormShape norm_shape(long long width, int dtype)
{
    const long long n = 16 / (long long)ngs_decoder_size(dtype), c = (width + n - 1) / n;
    if (c <= 1) return G1;
    if (c <= 2) return G2;
    if (c <= 4) return G4;
    if (c <= 8) return G8;
    if (c <= 16) return G16;
    if (c <= 32) return G32;
    if (c <= 64) return G64;
    if (c <= 128) return G64x2;
    if (c <= 192) return G64x3;
    if (c <= 256) return G64x4;
    if (c <= 512) return G256x2;
    if (c <= 768) return G256x3;
    if (c <= 1024) return G256x4;
    if (c <= 1536) return G512x3;
    if (c <= 2048) return G512x4;
    // (16-bit types hold twice as many elements per chunk: no registers for more)
    if (dtype == NGS_FLOAT32 && c <= 3 * 1024) return G1024x3;
    if (dtype == NGS_FLOAT32 && c <= 4 * 1024) return G1024x4;
    return NORM_WIDE;
}

static int norm_slots(NormShape s) { return s <= G64 ? 256 >> s : s <= G64x4 ? 4 : 1; }

// workgroups of the backward pass, each of which leaves one row of sums
static long long norm_backward_blocks(long long rows, int width, int dtype)
{
    const NormShape s = norm_shape(width, dtype);
    const long long need = (rows + norm_slots(s) - 1) / norm_slots(s);
    const long long most = s <= G64x4 ? 4 * NGS_CUS : s <= G256x4 ? 2 * NGS_CUS : s == NORM_WIDE ? 64 : NGS_CUS;
    return need < most ? need : most;
}

#define NGS_NORM_DISPATCH(LAUNCH)                 \
    switch (norm_shape(a.width, dtype)) {         \
    case G1: LAUNCH(1, 1, 256); break;            \
    case G2: LAUNCH(2, 1, 256); break;            \
    case G4: LAUNCH(4, 1, 256); break;            \
    case G8: LAUNCH(8, 1, 256); break;            \
    case G16: LAUNCH(16, 1, 256); break;          \
    case G32: LAUNCH(32, 1, 256); break;          \
    case G64: LAUNCH(64, 1, 256); break;          \
    case G64x2: LAUNCH(64, 2, 256); break;        \
    case G64x3: LAUNCH(64, 3, 256); break;        \
    case G64x4: LAUNCH(64, 4, 256); break;        \
    case G256x2: LAUNCH(256, 2, 256); break;      \
    case G256x3: LAUNCH(256, 3, 256); break;      \
    case G256x4: LAUNCH(256, 4, 256); break;      \
    case G512x3: LAUNCH(512, 3, 512); break;      \
    case G512x4: LAUNCH(512, 4, 512); break;      \
    case G1024x3:                                 \
        if constexpr (sizeof(T) == 4) LAUNCH(1024, 3, 1024); \
        break;                                    \
    case G1024x4:                                 \
        if constexpr (sizeof(T) == 4) LAUNCH(1024, 4, 1024); \
        break;                                    \
    default: return ngs_set_error("ngs_layer_norm", "no kernel for this width"); \
    }

template <typename T, typename W>
static int norm_forward(hipStream_t st, int dtype, NormArgs<T, W> a)
{
    const NormShape s = norm_shape(a.width, dtype);
    if (s == NORM_WIDE) {
        if (ngs_decoder_grid("ngs_layer_norm_forward", a.rows, 1024)) return 1;
        hipLaunchKernelGGL((norm_forward_wide_kernel<T, W>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
        return ngs_decoder_launched("ngs_layer_norm_forward");
    }
    const long long need = (a.rows + norm_slots(s) - 1) / norm_slots(s);
    const unsigned blocks = (unsigned)(need < NORM_WAVE_BLOCKS ? need : NORM_WAVE_BLOCKS);
#define LAUNCH_FORWARD(G, C, THREADS) \
    hipLaunchKernelGGL((norm_forward_kernel<T, W, G, C, THREADS>), dim3(blocks), dim3(THREADS), 0, st, a)
    NGS_NORM_DISPATCH(LAUNCH_FORWARD)
    return ngs_decoder_launched("ngs_layer_norm_forward");
}

template <typename T, typename W>
static int norm_backward(hipStream_t st, int dtype, int weight_dtype, NormBackwardArgs<T, W> a, void* dw, void* db)
{
    const unsigned blocks = (unsigned)norm_backward_blocks(a.rows, a.width, dtype);
    if (norm_shape(a.width, dtype) == NORM_WIDE) {
        if (ngs_decoder_grid("ngs_layer_norm_backward", a.rows, 1024)) return 1;
        if (a.dx)
            hipLaunchKernelGGL((norm_backward_wide_kernel<T, W>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
        if (a.partial) {
            const int span = 256 * Chunk<T>::N;
            hipLaunchKernelGGL((norm_columns_kernel<T, W>), dim3((a.width + span - 1) / span, blocks), dim3(256), 0, st, a);
        }
    } else {
#define LAUNCH_BACKWARD(G, C, THREADS) \
    hipLaunchKernelGGL((norm_backward_kernel<T, W, G, C, THREADS>), dim3(blocks), dim3(THREADS), 0, st, a)
        NGS_NORM_DISPATCH(LAUNCH_BACKWARD)
    }
    if (a.partial) ngs_launch_column_finish(st, a.partial, blocks, a.width, a.width, dw, db, weight_dtype);
    return ngs_decoder_launched("ngs_layer_norm_backward");
}

static int check_norm(const char* what, long long rows, int width, int dtype, int weight_dtype)
{
    if (rows < 0 || width < 0) return ngs_set_error(what, "a size is negative");
    if (rows > (1LL << 40) || width > NGS_WIDEST || (double)rows * width > 281474976710656.0)
        return ngs_set_error(what, "too many elements for one launch");
    if (!ngs_decoder_dtype(dtype) || !ngs_decoder_dtype(weight_dtype)) return ngs_set_error(what, "unknown element type");
    if (weight_dtype != dtype && weight_dtype != NGS_FLOAT32)
        return ngs_set_error(what, "the weights must be of the rows' type or float32");
    return 0;
}

extern "C" int ngs_layer_norm_forward(long long rows, int width, int dtype, int weight_dtype, float eps, const void* x,
                                      long long x_stride, const void* weight, const void* bias, void* y, float* mean,
                                      float* rstd, void* stream)
{
    const char* const what = "ngs_layer_norm_forward";
    if (check_norm(what, rows, width, dtype, weight_dtype)) return 1;
    if (!(eps >= 0.0f)) return ngs_set_error(what, "eps must not be negative");
    if (rows == 0 || width == 0) return 0;
    if (ngs_decoder_operand("ngs_layer_norm_forward: x", x, rows, width, x_stride) ||
        ngs_decoder_operand("ngs_layer_norm_forward: y", y, rows, width, width))
        return 1;
    hipStream_t st = (hipStream_t)stream;
#define NGS_NORM(T, W)                                                                                              \
    norm_forward<T, W>(st, dtype, NormArgs<T, W>{rows, width, eps, (float)width, (const T*)x, x_stride,      \
                                                 (const W*)weight, (const W*)bias, (T*)y, mean, rstd})
    if (dtype == NGS_FLOAT32) return NGS_NORM(float, float);
    if (dtype == NGS_FLOAT16) return weight_dtype == dtype ? NGS_NORM(f16, f16) : NGS_NORM(f16, float);
    return weight_dtype == dtype ? NGS_NORM(bf16, bf16) : NGS_NORM(bf16, float);
#undef NGS_NORM
}

extern "C" size_t ngs_layer_norm_backward_workspace_bytes(long long rows, int width, int dtype)
{
    if (rows <= 0 || width <= 0 || rows > (1LL << 40) || !ngs_decoder_dtype(dtype)) return 0;
    return (size_t)norm_backward_blocks(rows, width, dtype) * 2 * (size_t)width * sizeof(float);
}

extern "C" int ngs_layer_norm_backward(long long rows, int width, int dtype, int weight_dtype, const void* x,
                                       long long x_stride, const void* weight, const float* mean, const float* rstd,
                                       const void* dL_dy, long long dL_dy_stride, void* dL_dx, void* dL_dweight,
                                       void* dL_dbias, char* workspace, void* stream)
{
    const char* const what = "ngs_layer_norm_backward";
    if (check_norm(what, rows, width, dtype, weight_dtype)) return 1;
    if (width == 0 || (!dL_dx && !dL_dweight && !dL_dbias)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const bool sums = dL_dweight || dL_dbias;
    if (sums && ngs_decoder_columns(what, 2LL * width)) return 1;
    if (rows == 0) {  // sums over nothing
        if (sums) ngs_launch_column_finish(st, nullptr, 0, width, width, dL_dweight, dL_dbias, weight_dtype);
        return ngs_decoder_launched(what);
    }
    if (ngs_decoder_operand("ngs_layer_norm_backward: x", x, rows, width, x_stride) ||
        ngs_decoder_operand("ngs_layer_norm_backward: dL_dy", dL_dy, rows, width, dL_dy_stride) ||
        ngs_decoder_operand("ngs_layer_norm_backward: mean", mean, rows, 1, 1) ||
        ngs_decoder_operand("ngs_layer_norm_backward: rstd", rstd, rows, 1, 1))
        return 1;
    if (sums && !workspace) return ngs_set_error("ngs_layer_norm_backward: workspace", "is NULL");
#define NGS_NORM(T, W)                                                                                                  \
    norm_backward<T, W>(st, dtype, weight_dtype,                                                                        \
                        NormBackwardArgs<T, W>{rows, width, (float)width, (const T*)x, (const T*)dL_dy, x_stride, \
                                               dL_dy_stride, (const W*)weight, mean, rstd, (T*)dL_dx,                   \
                                               sums ? (float*)workspace : nullptr},                                     \
                        dL_dweight, dL_dbias)
    if (dtype == NGS_FLOAT32) return NGS_NORM(float, float);
    if (dtype == NGS_FLOAT16) return weight_dtype == dtype ? NGS_NORM(f16, f16) : NGS_NORM(f16, float);
    return weight_dtype == dtype ? NGS_NORM(bf16, bf16) : NGS_NORM(bf16, float);
#undef NGS_NORM
}
