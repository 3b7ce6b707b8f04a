// Matrix product with bias, activation and residual in its epilogue, and its backward pass.
//
//   forward   y = act(z) + residual,  z = x W^T + b          x [M][K], W [N][K], y [M][N]
//   backward  dz = dL_dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum of dz over the rows
//
// All three products are one kernel: D[q][p] = sum over r of P(p, r) Q(q, r), with p the contiguous index of the
// result.  P and Q each lie in memory either with r contiguous ("along") or with p / q contiguous ("across"):
//   forward  P = W along,   Q = x along,   r = K
//   dx       P = W across,  Q = dz along,  r = N
//   dW       P = x across,  Q = dz across, r = M
#include "linear_common.h"

// ---------------------------------------------------------------------------
// The product kernel
// ---------------------------------------------------------------------------
template <typename T>
struct Product {
    const T *p, *q;
    long long ldp, ldq;  // elements between neighbouring rows of the array as it lies in memory
    int np;
    long long nq, nr;
    long long tiles_p, tiles_q;
    int splits;          // the reduction is cut into this many runs of `run` elements (a multiple of a step's)
    long long run;
    Epilogue<T> epi;
};

// A workgroup of WP x WQ waves computes a TP x TQ tile of one run of the reduction; each step's operands travel
// through registers into shared memory while the step before is multiplied.
template <typename T, bool P_ACROSS, bool Q_ACROSS, int TP, int TQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void product_kernel(Product<T> a)
{
    typedef Tile<T, P_ACROSS, TP> TileP;
    typedef Tile<T, Q_ACROSS, TQ> TileQ;
    constexpr int THREADS = 64 * WP * WQ, STEP = TileP::STEP;
    constexpr int FP = TileP::CHUNKS / THREADS, FQ = TileQ::CHUNKS / THREADS;
    constexpr int MP = TP / WP / 16, MQ = TQ / WQ / 16;
    static_assert(TileP::CHUNKS % THREADS == 0 && TileQ::CHUNKS % THREADS == 0, "chunks divide over the threads");
    __shared__ __attribute__((aligned(16))) char sp[TP * ROW_BYTES];
    __shared__ __attribute__((aligned(16))) char sq[TQ * ROW_BYTES];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wp = wave % WP, wq = wave / WP;
    // workgroups go to the dies in turn: each die takes a contiguous run of tiles, whose operands meet in its cache
    const long long tiles = a.tiles_p * a.tiles_q, groups = tiles * a.splits;
    const long long per = (groups + NGS_XCDS - 1) / NGS_XCDS;
    const long long t = (long long)(blockIdx.x % NGS_XCDS) * per + blockIdx.x / NGS_XCDS;
    if (t >= groups) return;
    const long long split = t / tiles, tile = t - split * tiles;
    const long long p0 = (tile % a.tiles_p) * TP, q0 = (tile / a.tiles_p) * TQ;
    const long long r_begin = split * a.run, r_end = r_begin + a.run < a.nr ? r_begin + a.run : a.nr;

    f32x4 acc[MP][MQ];
#pragma unroll
    for (int i = 0; i < MP; i++)
#pragma unroll
        for (int j = 0; j < MQ; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    u32x4 fp[FP], fq[FQ];
    auto fetch = [&](long long r0) {
#pragma unroll
        for (int k = 0; k < FP; k++) fp[k] = TileP::fetch(a.p, a.ldp, p0, a.np, r0, r_end, tid + k * THREADS);
#pragma unroll
        for (int k = 0; k < FQ; k++) fq[k] = TileQ::fetch(a.q, a.ldq, q0, a.nq, r0, r_end, tid + k * THREADS);
    };
    if (r_begin < r_end) fetch(r_begin);
    for (long long r0 = r_begin; r0 < r_end; r0 += STEP) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < FP; k++) TileP::put(sp, tid + k * THREADS, fp[k]);
#pragma unroll
        for (int k = 0; k < FQ; k++) TileQ::put(sq, tid + k * THREADS, fq[k]);
        __syncthreads();
        if (r0 + STEP < r_end) fetch(r0 + STEP);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            u32x4 f[MP], h[MQ];
#pragma unroll
            for (int i = 0; i < MP; i++) f[i] = TileP::fragment(sp, wp * MP + i, s, lane);
#pragma unroll
            for (int j = 0; j < MQ; j++) h[j] = TileQ::fragment(sq, wq * MQ + j, s, lane);
#pragma unroll
            for (int i = 0; i < MP; i++)
#pragma unroll
                for (int j = 0; j < MQ; j++) acc[i][j] = mma(f[i], h[j], acc[i][j], (const T*)nullptr);
        }
    }

    // a lane holds four neighbouring p of one q
#pragma unroll
    for (int i = 0; i < MP; i++) {
        const int p = (int)p0 + (wp * MP + i) * 16 + (lane >> 4) * 4;
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p < a.np && a.epi.bias && !a.epi.partial) load4(a.epi.bias + p, bias, a.np - p);
#pragma unroll
        for (int j = 0; j < MQ; j++) {
            const long long q = q0 + (wq * MQ + j) * 16 + (lane & 15);
            if (p >= a.np || q >= a.nq) continue;
            if (a.epi.partial) {
                float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                store4(a.epi.partial + (split * a.nq + q) * a.np + p, v, a.np - p);
            } else {
                finish4(a.epi, q, p, acc[i][j], bias);
            }
        }
    }
}

// Adds up the runs of a product that was cut along its reduction, in their order, and finishes it.
template <typename T>
__global__ __launch_bounds__(256) void product_finish_kernel(const float* __restrict__ partial, int splits, long long nq,
                                                             Epilogue<T> e)
{
    const long long per_row = (e.np + 3) / 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= per_row * nq) return;
    const long long q = i / per_row;
    const int p = (int)(i - q * per_row) * 4, valid = e.np - p;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < splits; s++) {
        float v[4];
        load4(partial + ((long long)s * nq + q) * e.np + p, v, valid);
#pragma unroll
        for (int k = 0; k < 4; k++) sum[k] += v[k];
    }
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e.bias) load4(e.bias + p, bias, valid);
    finish4(e, q, p, (f32x4){sum[0], sum[1], sum[2], sum[3]}, bias);
}

// ---------------------------------------------------------------------------
// dz = dL_dy * slope and the column sums of dz
// ---------------------------------------------------------------------------
// A workgroup is `across` threads wide (each owns a chunk of neighbouring columns) and 256 / across rows high; it
// walks down its share of the rows.  slope == NULL: dz is dL_dy and only summed.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(long long rows, int n, int across, const T* __restrict__ dy,
                                                        long long lddy, const typename Slope<T>::type* __restrict__ slope,
                                                        T* __restrict__ dz, float* __restrict__ partial)
{
    constexpr int N = Chunk<T>::N;
    __shared__ float sums[256 * N];
    const int tid = threadIdx.x, tx = tid % across, ty = tid / across, high = 256 / across;
    const int col = (blockIdx.y * across + tx) * N, valid = n - col;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.0f;
    if (valid > 0) {
        for (long long r = (long long)blockIdx.x * high + ty; r < rows; r += (long long)gridDim.x * high) {
            float g[N];
            unpack<T>(load16_head(dy + r * lddy + col, valid), g);
            if (slope) {
                if (valid >= N) {
                    typename Slope<T>::type s[N];
                    __builtin_memcpy(s, slope + r * n + col, sizeof s);
#pragma unroll
                    for (int i = 0; i < N; i++) g[i] *= (float)s[i];
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (i < valid) g[i] *= (float)slope[r * n + col + i];
                }
                if (dz) store16_head(dz + r * n + col, pack<T>(g), valid);
            }
#pragma unroll
            for (int i = 0; i < N; i++) acc[i] += g[i];
        }
    }
    if (!partial) return;
#pragma unroll
    for (int i = 0; i < N; i++) sums[i * 256 + tid] = acc[i];
    __syncthreads();
    // the rows of the workgroup are added up by its first row of threads, in order
    if (ty == 0 && valid > 0) {
        for (int i = 0; i < N && i < valid; i++) {
            float s = 0.0f;
            for (int k = 0; k < high; k++) s += sums[i * 256 + k * across + tx];
            partial[(long long)blockIdx.x * n + col + i] = s;
        }
    }
}

// 16 columns by 64 rows of threads: a thread adds every 64th row, the 64 sums are joined pairwise.
template <typename T>
__global__ __launch_bounds__(1024) void column_finish_kernel(const float* __restrict__ partial, long long blocks,
                                                             long long width0, long long width1, T* __restrict__ out0,
                                                             T* __restrict__ out1)
{
    __shared__ float sums[64][17];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const long long c = (long long)blockIdx.x * 16 + tx, pitch = width0 + width1;
    float s = 0.0f;
    if (c < pitch)
        for (long long b = ty; b < blocks; b += 64) s += partial[b * pitch + c];
    sums[ty][tx] = s;
    __syncthreads();
    for (int half = 32; half > 0; half >>= 1) {
        if (ty < half) sums[ty][tx] += sums[ty + half][tx];
        __syncthreads();
    }
    if (ty != 0 || c >= pitch) return;
    T* const out = c < width0 ? out0 : out1;
    if (out) out[c < width0 ? c : c - width0] = (T)sums[0][tx];
}

void ngs_launch_column_finish(hipStream_t s, const float* partial, long long blocks, long long width0, long long width1,
                              void* out0, void* out1, int dtype)
{
    const dim3 grid((unsigned)((width0 + width1 + 15) / 16)), threads(1024);
    if (dtype == NGS_FLOAT32)
        hipLaunchKernelGGL(column_finish_kernel<float>, grid, threads, 0, s, partial, blocks, width0, width1, (float*)out0, (float*)out1);
    else if (dtype == NGS_FLOAT16)
        hipLaunchKernelGGL(column_finish_kernel<f16>, grid, threads, 0, s, partial, blocks, width0, width1, (f16*)out0, (f16*)out1);
    else
        hipLaunchKernelGGL(column_finish_kernel<bf16>, grid, threads, 0, s, partial, blocks, width0, width1, (bf16*)out0, (bf16*)out1);
}

// ---------------------------------------------------------------------------
// Launch shapes
// ---------------------------------------------------------------------------
struct Shape {
    int tp, tq;
    long long tiles_p, tiles_q;
    int splits;
    long long run;
    long long groups() const { return (tiles_p * tiles_q * splits + NGS_XCDS - 1) / NGS_XCDS * NGS_XCDS; }
    size_t partial_bytes(long long np, long long nq) const { return splits > 1 ? (size_t)splits * np * nq * 4 : 0; }
};

// Tiles are 128 wide unless the matrix is 32 or narrower; a reduction is cut until the tiles and its runs fill the
// chip twice, each run at least four steps long.
static Shape product_shape(long long np, long long nq, long long nr, int dtype)
{
    Shape s;
    s.tp = np <= 32 ? 32 : 128;
    s.tq = nq <= 32 ? 32 : 128;
    s.tiles_p = (np + s.tp - 1) / s.tp;
    s.tiles_q = (nq + s.tq - 1) / s.tq;
    const long long step = ROW_BYTES / (long long)ngs_decoder_size(dtype), steps = (nr + step - 1) / step;
    const long long tiles = s.tiles_p * s.tiles_q;
    long long cut = 1;
    if (tiles > 0 && tiles < NGS_CUS) {
        cut = (2 * NGS_CUS + tiles - 1) / tiles;
        if (cut > steps / 4) cut = steps / 4;
        if (cut < 1) cut = 1;
    }
    const long long run = cut > 1 ? (steps + cut - 1) / cut : (steps > 0 ? steps : 1);
    s.run = run * step;
    s.splits = steps > 0 ? (int)((steps + run - 1) / run) : 1;
    return s;
}

template <typename T, bool PA, bool QA>
static int launch_product(hipStream_t st, const Shape& s, Product<T> a, float* partial)
{
    a.tiles_p = s.tiles_p;
    a.tiles_q = s.tiles_q;
    a.splits = s.splits;
    a.run = s.run;
    a.epi.np = a.np;
    a.epi.partial = s.splits > 1 ? partial : nullptr;
    if (s.groups() > 0x7fffffffLL) return ngs_set_error("ngs_linear", "too many rows");
    const dim3 grid((unsigned)s.groups());
    if (s.tp == 128 && s.tq == 128)
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 128, 128, 2, 2>), grid, dim3(256), 0, st, a);
    else if (s.tp == 128)
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 128, 32, 4, 1>), grid, dim3(256), 0, st, a);
    else if (s.tq == 128)
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 32, 128, 1, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 32, 32, 2, 2>), grid, dim3(256), 0, st, a);
    if (s.splits > 1) {
        Epilogue<T> e = a.epi;
        const long long items = (a.np + 3LL) / 4 * a.nq;
        hipLaunchKernelGGL(product_finish_kernel<T>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, partial,
                           s.splits, a.nq, e);
    }
    return ngs_decoder_launched("ngs_linear");
}

static inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Backward workspace: dz (when there is an activation), the column sums' partials, the cut products' partials (the
// two products run one after the other and share them).
struct BackwardPlan {
    Shape dx, dw;
    int across;
    long long col_blocks, row_blocks;
    size_t sums_at, partial_at, total;
};

static BackwardPlan backward_plan(long long rows, int k, int n, int dtype, int act)
{
    BackwardPlan b;
    const long long size = (long long)ngs_decoder_size(dtype), chunk = 16 / size;
    b.dx = product_shape(k, rows, n, dtype);
    b.dw = product_shape(k, n, rows, dtype);
    const long long chunks = (n + chunk - 1) / chunk;
    b.across = 1;
    while (b.across < 64 && b.across < chunks) b.across *= 2;
    b.col_blocks = (chunks + b.across - 1) / b.across;
    const long long high = 256 / b.across;
    b.row_blocks = 2048 / (b.col_blocks > 0 ? b.col_blocks : 1);
    if (b.row_blocks > (rows + 4 * high - 1) / (4 * high)) b.row_blocks = (rows + 4 * high - 1) / (4 * high);
    if (b.row_blocks < 1) b.row_blocks = 1;
    b.sums_at = act == NGS_ACT_NONE ? 0 : align256((size_t)rows * n * size);
    b.partial_at = b.sums_at + align256((size_t)b.row_blocks * n * 4);
    const size_t p1 = b.dx.partial_bytes(k, rows), p2 = b.dw.partial_bytes(k, n);
    b.total = b.partial_at + align256(p1 > p2 ? p1 : p2) + 256;
    return b;
}

template <typename T>
static int linear_forward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const void* x, long long ldx,
                          const void* w, long long ldw, const void* bias, const void* res, long long ldr, void* y,
                          void* slope, char* workspace)
{
    Product<T> a = {};
    a.p = (const T*)w;
    a.q = (const T*)x;
    a.ldp = ldw;
    a.ldq = ldx;
    a.np = n;
    a.nq = rows;
    a.nr = k;
    a.epi.act = act;
    a.epi.bias = (const T*)bias;
    a.epi.residual = (const T*)res;
    a.epi.ldr = ldr;
    a.epi.y = (T*)y;
    a.epi.slope = act == NGS_ACT_NONE ? nullptr : (typename Slope<T>::type*)slope;
    a.epi.np = n;
    if (ngs_stream_forward_takes(rows, k, n, dtype))
        return ngs_stream_forward<T>(st, rows, k, n, dtype, a.q, ldx, a.p, ldw, a.epi);
    return launch_product<T, false, false>(st, product_shape(n, rows, k, dtype), a, (float*)workspace);
}

template <typename T>
static int linear_backward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const void* x, long long ldx,
                           const void* w, long long ldw, const void* bias, const void* slope, const void* dy, long long lddy,
                           void* dx, void* dw, void* db, char* workspace)
{
    if (ngs_stream_backward_takes(rows, k, n, dtype))
        return ngs_stream_backward<T>(st, rows, k, n, dtype, act, (const T*)x, ldx, (const T*)w, ldw, (const T*)bias,
                                      (const T*)dy, lddy, (T*)dx, (T*)dw, (T*)db, (float*)workspace);
    const BackwardPlan b = backward_plan(rows, k, n, dtype, act);
    const T* dz = (const T*)dy;
    long long lddz = lddy;
    float* sums = (float*)(workspace + b.sums_at);
    float* partial = (float*)(workspace + b.partial_at);
    const bool make_dz = act != NGS_ACT_NONE && (dx || dw) && rows > 0 && n > 0;
    if (make_dz || db) {
        const dim3 grid((unsigned)b.row_blocks, (unsigned)b.col_blocks);
        hipLaunchKernelGGL(linear_dz_kernel<T>, grid, dim3(256), 0, st, rows, n, b.across, (const T*)dy, lddy,
                           act == NGS_ACT_NONE ? nullptr : (const typename Slope<T>::type*)slope,
                           make_dz ? (T*)workspace : nullptr, db ? sums : nullptr);
        if (db) ngs_launch_column_finish(st, sums, b.row_blocks, n, 0, db, nullptr, dtype);
        if (ngs_decoder_launched("ngs_linear_backward")) return 1;
        if (make_dz) {
            dz = (const T*)workspace;
            lddz = n;
        }
    }
    if (dx) {
        Product<T> a = {};
        a.p = (const T*)w;
        a.q = dz;
        a.ldp = ldw;
        a.ldq = lddz;
        a.np = k;
        a.nq = rows;
        a.nr = n;
        a.epi.y = (T*)dx;
        if (launch_product<T, true, false>(st, b.dx, a, partial)) return 1;
    }
    if (dw) {
        Product<T> a = {};
        a.p = (const T*)x;
        a.q = dz;
        a.ldp = ldx;
        a.ldq = lddz;
        a.np = k;
        a.nq = n;
        a.nr = rows;
        a.epi.y = (T*)dw;
        if (launch_product<T, true, true>(st, b.dw, a, partial)) return 1;
    }
    return 0;
}

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
static int check_linear(const char* what, long long rows, int k, int n, int dtype, int act)
{
    if (rows < 0 || k < 0 || n < 0) return ngs_set_error(what, "a size is negative");
    if (rows > (1LL << 40)) return ngs_set_error(what, "too many rows");
    if (!ngs_decoder_dtype(dtype)) return ngs_set_error(what, "unknown element type");
    if (act < NGS_ACT_NONE || act > NGS_ACT_SIGMOID) return ngs_set_error(what, "unknown activation");
    return 0;
}

extern "C" size_t ngs_linear_forward_workspace_bytes(long long rows, int in_features, int out_features, int dtype)
{
    if (rows <= 0 || out_features <= 0 || in_features < 0 || rows > (1LL << 40) || !ngs_decoder_dtype(dtype)) return 0;
    if (ngs_stream_forward_takes(rows, in_features, out_features, dtype)) return 0;
    return product_shape(out_features, rows, in_features, dtype).partial_bytes(out_features, rows);
}

extern "C" int ngs_linear_forward(long long rows, int in_features, int out_features, int dtype, int activation,
                                  const void* x, long long x_stride, const void* weight, long long weight_stride,
                                  const void* bias, const void* residual, long long residual_stride, void* y,
                                  void* slope, char* workspace, void* stream)
{
    const int k = in_features, n = out_features;
    if (check_linear("ngs_linear_forward", rows, k, n, dtype, activation)) return 1;
    if (rows == 0 || n == 0) return 0;
    if (ngs_decoder_operand("ngs_linear_forward: x", x, rows, k, x_stride) ||
        ngs_decoder_operand("ngs_linear_forward: weight", weight, n, k, weight_stride) ||
        ngs_decoder_operand("ngs_linear_forward: residual", residual ? residual : y, rows, n, residual ? residual_stride : n) ||
        ngs_decoder_operand("ngs_linear_forward: y", y, rows, n, n))
        return 1;
    if (!workspace && ngs_linear_forward_workspace_bytes(rows, k, n, dtype))
        return ngs_set_error("ngs_linear_forward: workspace", "is NULL");
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NGS_FLOAT32)
        return linear_forward<float>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, residual,
                                     residual_stride, y, slope, workspace);
    if (dtype == NGS_FLOAT16)
        return linear_forward<f16>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, residual,
                                   residual_stride, y, slope, workspace);
    return linear_forward<bf16>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, residual,
                                residual_stride, y, slope, workspace);
}

extern "C" int ngs_linear_backward_reads_slope(long long rows, int in_features, int out_features, int dtype, int activation)
{
    if (rows <= 0 || out_features <= 0 || !ngs_decoder_dtype(dtype) || activation == NGS_ACT_NONE) return 0;
    return ngs_stream_backward_takes(rows, in_features, out_features, dtype) ? 0 : 1;
}

extern "C" size_t ngs_linear_backward_workspace_bytes(long long rows, int in_features, int out_features, int dtype,
                                                      int activation)
{
    if (rows < 0 || in_features < 0 || out_features < 0 || rows > (1LL << 40) || !ngs_decoder_dtype(dtype)) return 0;
    if (ngs_stream_backward_takes(rows, in_features, out_features, dtype))
        return (size_t)ngs_stream_backward_blocks(rows, in_features, out_features, dtype) *
               ((size_t)in_features * out_features + out_features) * sizeof(float);
    return backward_plan(rows, in_features, out_features, dtype, activation).total;
}

extern "C" int ngs_linear_backward(long long rows, int in_features, int out_features, int dtype, int activation,
                                   const void* x, long long x_stride, const void* weight, long long weight_stride,
                                   const void* bias, const void* slope, const void* dL_dy, long long dL_dy_stride,
                                   void* dL_dx, void* dL_dweight, void* dL_dbias, char* workspace, void* stream)
{
    const int k = in_features, n = out_features;
    if (check_linear("ngs_linear_backward", rows, k, n, dtype, activation)) return 1;
    if (rows == 0 || k == 0) dL_dx = nullptr;   // nothing to write
    if (n == 0 || k == 0) dL_dweight = nullptr;
    if (n == 0) dL_dbias = nullptr;
    if (!dL_dx && !dL_dweight && !dL_dbias) return 0;
    const bool reads_slope = ngs_linear_backward_reads_slope(rows, k, n, dtype, activation);
    const bool forms_z = activation != NGS_ACT_NONE && !reads_slope;
    if (((dL_dweight || forms_z) && ngs_decoder_operand("ngs_linear_backward: x", x, rows, k, x_stride)) ||
        ((dL_dx || forms_z) && ngs_decoder_operand("ngs_linear_backward: weight", weight, n, k, weight_stride)) ||
        ngs_decoder_operand("ngs_linear_backward: dL_dy", dL_dy, rows, n, dL_dy_stride))
        return 1;
    if (reads_slope && ngs_decoder_operand("ngs_linear_backward: slope", slope, rows, n, n)) return 1;
    if (!workspace) return ngs_set_error("ngs_linear_backward: workspace", "is NULL");
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NGS_FLOAT32)
        return linear_backward<float>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, slope, dL_dy,
                                      dL_dy_stride, dL_dx, dL_dweight, dL_dbias, workspace);
    if (dtype == NGS_FLOAT16)
        return linear_backward<f16>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, slope, dL_dy,
                                    dL_dy_stride, dL_dx, dL_dweight, dL_dbias, workspace);
    return linear_backward<bf16>(st, rows, k, n, dtype, activation, x, x_stride, weight, weight_stride, bias, slope, dL_dy,
                                 dL_dy_stride, dL_dx, dL_dweight, dL_dbias, workspace);
}
