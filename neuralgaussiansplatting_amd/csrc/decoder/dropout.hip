// Dropout whose mask is a function of (seed, offset, element) and is never stored, with an optional residual sum.
//
// Eight neighbouring elements share one block of Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw: "Parallel
// Random Numbers: As Easy as 1, 2, 3", SC 2011; the paper's count of rounds that passes all of its statistical tests):
// four words, 16 bits an element.  Sixteen bits set a probability to within 2^-17 and halve the generator's share of a
// pass that moves 4 to 6 bytes an element.
//
// Bound by memory: 1920 x 1080 x 64 bfloat16 with residual there and back moves 1.33 GB in 226 us, 5.9 TB/s.
// Rows with gaps go element by element where a block crosses rows: y may be x, so each load stays behind the store before
// it and is waited for (400 x 400 x 39 of 64 float16: 25 MB in 12.7 us, the waves waiting 74 % of their cycles).
#include "decoder_common.h"

#define PHILOX_ROUNDS 7

__device__ __forceinline__ u32x4 philox(uint64_t counter, uint64_t stream, uint64_t key)
{
    uint32_t a = (uint32_t)counter, b = (uint32_t)(counter >> 32), c = (uint32_t)stream, d = (uint32_t)(stream >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < PHILOX_ROUNDS; r++) {
        const uint64_t l = (uint64_t)a * 0xD2511F53u, h = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(h >> 32) ^ b ^ k0;
        b = (uint32_t)h;
        c = (uint32_t)(l >> 32) ^ d ^ k1;
        d = (uint32_t)l;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return (u32x4){a, b, c, d};
}

template <typename T>
struct DropoutArgs {
    long long rows, cols, total;
    const T *x, *residual;
    long long ldx, ldr;
    T* y;
    uint32_t threshold;  // in 65536ths
    float scale;
    uint64_t seed, offset;
    const unsigned long long* seed_device;
};

// A thread per block of eight elements.  Where all eight lie in one row (always, when the rows follow each other
// without gaps: the host then passes the array as one row) they move as 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs<T> a)
{
    constexpr int N = Chunk<T>::N, PARTS = 8 / N;
    const long long block = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long e0 = block * 8;
    if (e0 >= a.total) return;
    const uint64_t key = a.seed_device ? (uint64_t)*a.seed_device : a.seed;
    const u32x4 bits = philox((uint64_t)block, a.offset, key);
    long long row = 0, col = e0;
    if (a.rows > 1) {
        row = e0 / a.cols;
        col = e0 - row * a.cols;
    }
    if (col + 8 <= a.cols) {
        const T* const x = a.x + row * a.ldx + col;
        u32x4 vx[PARTS], vr[PARTS];
#pragma unroll
        for (int h = 0; h < PARTS; h++) {
            vx[h] = load16(x + h * N);
            if (a.residual) vr[h] = load16(a.residual + row * a.ldr + col + h * N);
        }
#pragma unroll
        for (int h = 0; h < PARTS; h++) {
            float f[N], r[N];
            unpack<T>(vx[h], f);
            if (a.residual) unpack<T>(vr[h], r);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = h * N + i;
                const uint32_t mine = (e & 1) ? bits[e / 2] >> 16 : bits[e / 2] & 0xffffu;
                float v = mine >= a.threshold ? f[i] * a.scale : 0.0f;
                if (a.residual) v += r[i];
                f[i] = v;
            }
            const u32x4 out = pack<T>(f);
            __builtin_memcpy(a.y + e0 + h * N, &out, 16);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (e0 + e >= a.total) return;
        const uint32_t mine = (e & 1) ? bits[e / 2] >> 16 : bits[e / 2] & 0xffffu;
        float v = mine >= a.threshold ? (float)a.x[row * a.ldx + col] * a.scale : 0.0f;
        if (a.residual) v += (float)a.residual[row * a.ldr + col];
        a.y[e0 + e] = (T)v;
        if (++col == a.cols) {
            col = 0;
            row++;
        }
    }
}

template <typename T>
static int run_dropout(hipStream_t st, DropoutArgs<T> a)
{
    const bool flat = a.ldx == a.cols && (!a.residual || a.ldr == a.cols);
    if (flat) {
        a.cols = a.total;
        a.rows = 1;
    }
    const long long groups = ((a.total + 7) / 8 + 255) / 256;
    if (ngs_decoder_grid("ngs_dropout", groups, 256)) return 1;
    hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)groups), dim3(256), 0, st, a);
    return ngs_decoder_launched("ngs_dropout");
}

extern "C" int ngs_dropout(long long rows, long long cols, int dtype, double p, unsigned long long seed,
                           const unsigned long long* seed_device, unsigned long long offset, const void* x,
                           long long x_stride, const void* residual, long long residual_stride, void* y, void* stream)
{
    if (rows < 0 || cols < 0) return ngs_set_error("ngs_dropout", "a size is negative");
    if (!ngs_decoder_dtype(dtype)) return ngs_set_error("ngs_dropout", "unknown element type");
    if (!(p >= 0.0 && p <= 1.0)) return ngs_set_error("ngs_dropout", "p must lie in [0, 1]");
    if (rows == 0 || cols == 0) return 0;
    if (rows > (1LL << 58) / cols) return ngs_set_error("ngs_dropout", "too many elements");
    if (ngs_decoder_operand("ngs_dropout: x", x, rows, cols, x_stride) ||
        ngs_decoder_operand("ngs_dropout: residual", residual ? residual : y, rows, cols, residual ? residual_stride : cols) ||
        ngs_decoder_operand("ngs_dropout: y", y, rows, cols, cols))
        return 1;
    const uint32_t t = (uint32_t)floor(p * 65536.0 + 0.5);
    const float scale = t < 65536u ? (float)(65536.0 / (65536.0 - (double)t)) : 0.0f;  // t = 65536: nothing is kept
    hipStream_t st = (hipStream_t)stream;
#define NGS_DROPOUT(T)                                                                                              \
    run_dropout<T>(st, DropoutArgs<T>{rows, cols, rows * cols, (const T*)x, (const T*)residual, x_stride,          \
                                      residual_stride, (T*)y, t, scale, seed, offset, seed_device})
    if (dtype == NGS_FLOAT32) return NGS_DROPOUT(float);
    if (dtype == NGS_FLOAT16) return NGS_DROPOUT(f16);
    return NGS_DROPOUT(bf16);
}
