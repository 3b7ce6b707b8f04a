// The product for a few rows (queries of a network): the weight's way through the memory is what it takes, so every
// weight is read once, straight into the matrix instructions' layout, and multiplied with all rows there.
//
// A workgroup takes 16 rows of the weight and cuts the reduction among its waves, as many as keep the memory busy; their
// sums meet in shared memory, in the waves' order, and are finished there: one launch, no second pass.
//
// Measured: 1 x 1024 -> 4096 bfloat16 (8 MB) 5.4 us, close to an empty call; 1 x 4096 -> 4096 (34 MB) 9.1 us, 3.7 TB/s;
// 16 x 4096 -> 4096 10.9 us.
#include "linear_stream.h"

template <typename T>
struct FewRows {
    int rows, k, n, run;  // run: steps of four chunks that a wave takes
    const T *x, *w;
    long long ldx, ldw;
    Epilogue<T> e;
};

// QF: fragments of 16 rows of x.  ANY: some row starts in the middle of a word.  U: steps whose loads are on their way
// together.
template <typename T, int QF, bool ANY>
__global__ __launch_bounds__(1024) void few_rows_kernel(FewRows<T> a)
{
    constexpr int U = QF == 1 ? 8 : QF == 2 ? 4 : 2;
    extern __shared__ __attribute__((aligned(16))) f32x4 sums[];  // [wave][QF][lane]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, g = lane >> 4, i = lane & 15;
    const long long p = (long long)blockIdx.x * 16 + i;
    const RowChunks<T, false, ANY> chunks(a.k);
    const T* const pw = a.w + (p < a.n ? p : a.n - 1) * a.ldw;
    const T* px[QF];
#pragma unroll
    for (int f = 0; f < QF; f++) px[f] = a.x + (f * 16 + i < a.rows ? f * 16 + i : a.rows - 1) * a.ldx;
    const int steps = (a.k + 4 * Chunk<T>::N - 1) / (4 * Chunk<T>::N);
    const int first = wave * a.run, last = first + a.run < steps ? first + a.run : steps;
    f32x4 acc[QF];
#pragma unroll
    for (int f = 0; f < QF; f++) acc[f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = first; s0 < last; s0 += U) {
        u32x4 w[U], x[U][QF];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + u < last ? s0 + u : last - 1;  // (a step that is not there is read and not used)
            w[u] = chunks.fetch(pw, s * 4 + g);
#pragma unroll
            for (int f = 0; f < QF; f++) x[u][f] = chunks.fetch(px[f], s * 4 + g);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + u;
            if (s >= last) break;
            const u32x4 ws = chunks.settle(w[u], s * 4 + g, s * 4, true);
#pragma unroll
            for (int f = 0; f < QF; f++)
                acc[f] = mma(ws, chunks.settle(x[u][f], s * 4 + g, s * 4, true), acc[f], (const T*)nullptr);
        }
    }
    if (waves > 1) {
#pragma unroll
        for (int f = 0; f < QF; f++) sums[(wave * QF + f) * 64 + lane] = acc[f];
        __syncthreads();
    }
    // a lane holds four neighbouring columns of one row
    for (int f = wave; f < QF; f += waves) {
        f32x4 z = acc[0];
        if (waves > 1) {
            z = sums[f * 64 + lane];
            for (int v = 1; v < waves; v++) z += sums[(v * QF + f) * 64 + lane];
        } else {
#pragma unroll
            for (int h = 1; h < QF; h++) z = f == h ? acc[h] : z;
        }
        const long long col = (long long)blockIdx.x * 16 + g * 4;
        const int row = f * 16 + i;
        if (row >= a.rows || col >= a.n) continue;
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (a.e.bias) load4(a.e.bias + col, bias, a.n - (int)col);
        finish4(a.e, row, (int)col, z, bias);
    }
}

bool ngs_few_rows_takes(long long rows, int k, int n, int dtype)
{
    // (four fragments of rows and a long reduction: the tiles' second pass over the sums costs less than the waits here,
    // 64 x 3712 -> 1000 bfloat16 20 us against 15 us; 64 x 1000 -> 1000 6 us against 12 us)
    const int size = (int)ngs_decoder_size(dtype);
    return rows >= 1 && (rows <= 32 || (rows <= NGS_FEW_ROWS && k <= 4096 / size)) && k >= 16 / size && n >= 1;
}

template <typename T, int QF>
static int few_rows_launch(hipStream_t st, FewRows<T> a)
{
    const int steps = (a.k + 4 * Chunk<T>::N - 1) / (4 * Chunk<T>::N), groups = (a.n + 15) / 16;
    // waves: until the chip holds 16 to a compute unit, while each has four steps
    int waves = 1;
    while (waves < 16 && (long long)groups * waves < 16 * NGS_CUS && steps >= 8 * waves) waves *= 2;
    if (ngs_decoder_grid("ngs_linear_forward", groups, 64 * waves)) return 1;
    a.run = (steps + waves - 1) / waves;
    const size_t lds = waves > 1 ? (size_t)waves * QF * 64 * sizeof(f32x4) : 0;
    const bool any = sizeof(T) == 2 && (((uintptr_t)a.x | (uintptr_t)a.w) & 3 || (a.ldx | a.ldw) & 1);
    if constexpr (sizeof(T) == 2) {
        if (any) hipLaunchKernelGGL((few_rows_kernel<T, QF, true>), dim3(groups), dim3(64 * waves), lds, st, a);
    }
    if (!any) hipLaunchKernelGGL((few_rows_kernel<T, QF, false>), dim3(groups), dim3(64 * waves), lds, st, a);
    return ngs_decoder_launched("ngs_linear_forward");
}

template <typename T>
int ngs_few_rows(hipStream_t st, long long rows, int k, int n, const T* x, long long ldx, const T* w, long long ldw,
                 const Epilogue<T>& e)
{
    const FewRows<T> a = {(int)rows, k, n, 0, x, w, ldx, ldw, e};
    if (rows <= 16) return few_rows_launch<T, 1>(st, a);
    if (rows <= 32) return few_rows_launch<T, 2>(st, a);
    return few_rows_launch<T, 4>(st, a);
}

#define NGS_FEW_INSTANCE(T) \
    template int ngs_few_rows<T>(hipStream_t, long long, int, int, const T*, long long, const T*, long long, const Epilogue<T>&);
NGS_FEW_INSTANCE(float)
NGS_FEW_INSTANCE(f16)
NGS_FEW_INSTANCE(bf16)
