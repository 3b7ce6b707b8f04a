// The product over many narrow rows (a layer of a decoder over the pixels of an image): the weight fits on the chip, so
// each workgroup keeps it in shared memory and the rows stream past, read and written once.  Bound by memory.
//
// Rows go straight from memory into the matrix instructions' layout: lane (g, i) = (lane / 16, lane % 16) holds, of row
// i of a group of 16, the 16-byte chunks 4 s + g.  A result comes out the same way: its 16 columns of a fragment are
// taken from the weight's rows in such an order that a lane's sums are neighbours and fill whole chunks -- so what one
// product writes is what the next would read, and the backward pass can form z again from x and the weight, chunk for
// chunk beside dL_dy, instead of reading a stored derivative (2 or 4 bytes an element, against a product that the
// matrix units have idle time for).
//
// The backward pass is one kernel: a workgroup walks over tiles of 16 rows per wave; dz goes through the product with the
// weight (dx) and, with x, through shared memory into the product over the rows (dW), whose sums stay in registers
// until the workgroup is done.
//
// Measured: 640000 rows 128 -> 128 bfloat16 with gelu and residual, kernel times: forward 494 MB in 103 us (4.8 TB/s, at a
// large copy's rate), backward 509 MB in 202 us (2.5 TB/s).  Without an activation the two together take 211 us instead
// of 280 us, of which the forward pass is 93 and 99 us: forming z and the derivative again is about 60 us of the backward
// pass; 241 registers a lane leave it two waves to a SIMD, too few to hide it under the loads.  1920 x 1080 rows 64 -> 128
// float32 forward with relu moves 1.59 GB in 358 us (4.5 TB/s).
//
// Widths count in steps of four chunks, rounded up to a power of two, and what of them is empty is left out only where
// there is much of it: unequal and odd widths are further from the memory's rate (292504 rows 14 -> 168 bfloat16 there and
// back 112 us for 213 MB; 893582 rows 40 -> 152 float32 926 us for 1.4 GB).  Widths of 129 to 256 beside narrow ones hold
// one wave a SIMD, and float32 of 17 to 32 against 129 to 256 spills 348 bytes a lane (893582 rows 20 -> 152: 1658 us).
#pragma once
#include "linear_common.h"

// ---------------------------------------------------------------------------
// Rows in chunks.  A chunk that the row's end cuts is read from the end backwards and shifted into place, so that every
// lane of a wave reads 16 bytes inside its row without a branch.  SHORT: rows of less than a chunk, read by elements.
// ANY: rows that start in the middle of a word, as load16_any reads them.
// ---------------------------------------------------------------------------
template <typename T, bool SHORT = false, bool ANY = false>
struct RowChunks {
    int width, whole, tail;  // whole chunks, elements behind them

    __device__ __forceinline__ explicit RowChunks(int w) : width(w), whole(w / Chunk<T>::N), tail(w % Chunk<T>::N) {}

    // raw bytes of chunk c: to be passed through settle() before use
    __device__ __forceinline__ u32x4 fetch(const T* row, int c) const
    {
        constexpr int N = Chunk<T>::N;
        if constexpr (SHORT) {
            union { u32x4 v; T e[N]; } u;
#pragma unroll
            for (int i = 0; i < N; i++) u.e[i] = row[i < width ? i : 0];
            return u.v;
        }
        const int at = c * N < width - N ? c * N : width - N;
        return ANY ? load16_any(row + at) : load16(row + at);
    }
    // chunks first .. first + 3 are those of a step: what lies behind the row's end, or in no row, becomes zero
    __device__ __forceinline__ u32x4 settle(u32x4 v, int c, int first, bool there) const
    {
        constexpr int N = Chunk<T>::N;
        if constexpr (SHORT) {
            union { u32x4 v; T e[N]; } u;
            u.v = v;
#pragma unroll
            for (int i = 0; i < N; i++) u.e[i] = there && c == 0 && i < width ? u.e[i] : (T)0.0f;
            return u.v;
        }
        if (first + 4 <= whole) {  // uniform: nothing is cut in this step
            if (!there) v = (u32x4){0, 0, 0, 0};
            return v;
        }
        if (tail) {  // uniform
            const int bytes = (N - tail) * (int)sizeof(T);
            u32x4 t = v;
            if (bytes & 8) t = (u32x4){t.z, t.w, 0, 0};
            if (bytes & 4) t = (u32x4){t.y, t.z, t.w, 0};
            if (bytes & 2) t = (u32x4){(t.x >> 16) | (t.y << 16), (t.y >> 16) | (t.z << 16), (t.z >> 16) | (t.w << 16), t.w >> 16};
            if (c == whole) v = t;
        }
        if (c >= whole + (tail ? 1 : 0) || !there) v = (u32x4){0, 0, 0, 0};
        return v;
    }
    // chunks first .. first + 3 of a row of results, `first` the same in all lanes
    static __device__ __forceinline__ void store(T* row, u32x4 v, int c, int first, int width)
    {
        constexpr int N = Chunk<T>::N;
        if ((first + 4) * N <= width) __builtin_memcpy(row + c * N, &v, 16);
        else if (c * N < width) store16_head(row + c * N, v, width - c * N);
    }
};

// ---------------------------------------------------------------------------
// The weight in shared memory: LINES rows of CH chunks, the chunks of a row exchanged by the row's number so that both
// ways of reading spread over the banks.
// ---------------------------------------------------------------------------
template <typename T, int CH>
struct WeightTile {
    static __device__ __forceinline__ int swap(int row)
    {
        const int s = sizeof(T) == 2 ? ((row & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 4) & 1) : row & 15;
        return s & (CH - 1);
    }
    static __device__ __forceinline__ char* at(char* lds, int row, int c) { return lds + ((row * CH + (c ^ swap(row))) << 4); }
    static __device__ __forceinline__ const char* at(const char* lds, int row, int c) { return lds + ((row * CH + (c ^ swap(row))) << 4); }

    static __device__ __forceinline__ void fill(char* lds, const T* __restrict__ w, long long ldw, int n, int k, int lines,
                                                int tid, int threads)
    {
        for (int i = tid; i < lines * CH; i += threads) {
            const int row = i / CH, c = i % CH;
            *(u32x4*)at(lds, row, c) = load16_head(w + row * ldw + c * Chunk<T>::N, row < n ? k - c * Chunk<T>::N : 0);
        }
    }
    // the order in which fragment f takes 16 result columns: lane group g's four are neighbours, and for 16-bit types
    // continue those of fragment f - 1 (f odd) to a chunk
    static __device__ __forceinline__ int column(int f, int i)
    {
        return sizeof(T) == 2 ? (f >> 1) * 32 + (i >> 2) * 8 + (f & 1) * 4 + (i & 3) : f * 16 + i;
    }
    // Results of two fragments of `across` (packed: two words of four columns each) as whole chunks: lane groups trade
    // halves with their neighbours, after which group g holds the pair's chunk number chunk_of(g).  (Taking the columns in
    // `column` order instead would make every read meet half its banks twice.)
    static __device__ __forceinline__ int chunk_of(int g) { return sizeof(T) == 2 ? ((g & 1) << 1) | (g >> 1) : g; }
    static __device__ __forceinline__ u32x4 join(u32x4 v)
    {
        if (sizeof(T) != 2) return v;
        const auto lo = __builtin_amdgcn_permlane16_swap(v.x, v.z, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(v.y, v.w, false, false);
        return (u32x4){lo[0], hi[0], lo[1], hi[1]};
    }
    // fragment f of z's columns (the weight's rows), reduced along the weight's rows; chunks 4 s + g
    static __device__ __forceinline__ u32x4 along(const char* lds, int f, int s, int lane)
    {
        return *(const u32x4*)at(lds, column(f, lane & 15), s * 4 + (lane >> 4));
    }
    // fragment f of dx's columns (the weight's columns 16 f ...), reduced across the weight's rows: those of chunks
    // 4 s + g of dz
    static __device__ __forceinline__ u32x4 across(const char* lds, int f, int s, int lane)
    {
        const int g = lane >> 4, i = lane & 15;
        if (sizeof(T) == 2) {
            const int row = s * 32 + g * 8 + (i >> 2), c = f * 2 + ((i & 3) >> 1);
            typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at(lds, row, c) + (i & 1) * 8));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at(lds, row + 4, c) + (i & 1) * 8));
            const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
            return (u32x4){l.x, l.y, h.x, h.y};
        }
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[j] = *(const uint32_t*)(at(lds, s * 16 + g * 4 + j, f * 4 + (i >> 2)) + (i & 3) * 4);
        return v;
    }
};

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <typename T>
struct StreamForward {
    long long rows;
    int k, n;
    const T *x, *w, *bias, *residual;
    long long ldx, ldw, ldr;
    int act;
    T* y;
    float* slope;  // or NULL
};

// KS: steps of four chunks that a row of x takes.  NB: groups of four chunks of the result that a workgroup computes
// (blockIdx.y counts these).  SHORT: rows of x are shorter than a chunk.  A wave takes 16 rows at a time.  Loads and stores retire in order, so a row's results are
// kept until the next rows have arrived: the wait for those then covers nothing younger, and both the stores and the
// loads behind them have the whole computation of the next rows to get done.
template <typename T, int KS, int NB, bool SHORT, bool RESIDUAL, int THREADS>
__global__ __launch_bounds__(THREADS) void stream_forward_kernel(StreamForward<T> a)
{
    constexpr int N = Chunk<T>::N, CH = KS * 4, PARTS = N / 4, COLS = NB * 4 * N;  // PARTS: fragments that make a chunk
    typedef WeightTile<T, CH> W;
    __shared__ __attribute__((aligned(16))) char weight[COLS * CH * 16];
    __shared__ __attribute__((aligned(16))) float bias[COLS];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
    const int n0 = blockIdx.y * COLS, n = a.n - n0 < COLS ? a.n - n0 : COLS;  // this workgroup's columns
    const int blocks = (n + 4 * N - 1) / (4 * N);
    W::fill(weight, a.w + n0 * a.ldw, a.ldw, n, a.k, COLS, tid, THREADS);
    for (int c = tid; c < COLS; c += THREADS) bias[c] = a.bias && c < n ? (float)a.bias[n0 + c] : 0.0f;
    __syncthreads();

    const RowChunks<T, SHORT> xc(a.k);
    const long long groups = (a.rows + 15) / 16, waves = (long long)gridDim.x * (THREADS / 64);
    long long group = (long long)blockIdx.x * (THREADS / 64) + (tid >> 6), done = -1;
    u32x4 nx[KS], nr[RESIDUAL ? NB : 1], y[NB];
    auto fetch = [&](long long at) {
        const long long r = at * 16 + i, row = r < a.rows ? r : a.rows - 1;
        const T* const px = a.x + row * a.ldx;
#pragma unroll
        for (int s = 0; s < KS; s++) nx[s] = xc.fetch(px, s * 4 + g);
        if constexpr (RESIDUAL) {
            const T* const pr = a.residual + row * a.ldr + n0;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int col = (b * 4 + g) * N;
                if ((b + 1) * 4 * N <= n) nr[b] = load16(pr + col);       // uniform
                else if (b < blocks) nr[b] = load16_head(pr + col, n - col);
            }
        }
    };
    auto store = [&](long long at) {
        const long long r = at * 16 + i;
        if (r >= a.rows) return;
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (b < blocks) RowChunks<T>::store(a.y + r * a.n + n0, y[b], b * 4 + g, b * 4, n);
    };
    if (group < groups) fetch(group);
    for (; group < groups; group += waves) {
        u32x4 x[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) x[s] = xc.settle(nx[s], s * 4 + g, s * 4, true);
        if (done >= 0) store(done);
        done = group;
        if constexpr (RESIDUAL) {
#pragma unroll
            for (int b = 0; b < NB; b++) y[b] = nr[b];
        }
        if (group + waves < groups) fetch(group + waves);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (b < blocks) {  // uniform
                f32x4 acc[PARTS];
#pragma unroll
                for (int h = 0; h < PARTS; h++) acc[h] = *(const f32x4*)&bias[(b * 4 + g) * N + h * 4];
#pragma unroll
                for (int s = 0; s < KS; s++) {
#pragma unroll
                    for (int h = 0; h < PARTS; h++)
                        acc[h] = mma(W::along(weight, b * PARTS + h, s, lane), x[s], acc[h], (const T*)nullptr);
                }
                float z[N], v[N], slope[N];
#pragma unroll
                for (int e = 0; e < N; e++) z[e] = acc[e / 4][e % 4];
                if (a.slope) {
                    activate<N>(a.act, z, v, slope);
                    const long long r = group * 16 + i;
                    const int col = (b * 4 + g) * N;
#pragma unroll
                    for (int e = 0; e < N; e += 4) {
                        const float four[4] = {slope[e], slope[e + 1], slope[e + 2], slope[e + 3]};
                        if (r < a.rows && col + e < n) store4(a.slope + r * a.n + n0 + col + e, four, n - col - e);
                    }
                } else {
                    activate<N>(a.act, z, v, nullptr);
                }
                if constexpr (RESIDUAL) {
                    float f[N];
                    unpack<T>(y[b], f);
#pragma unroll
                    for (int e = 0; e < N; e++) v[e] += f[e];
                }
                y[b] = pack<T>(v);
            }
        }
    }
    if (done >= 0) store(done);
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// Backward: the product of x's and dz's steps that one workgroup's shared memory holds (the weight, and the tiles of 16
// rows per wave).
constexpr int stream_most(int size) { return size == 4 ? 64 : 32; }
// Waves of a workgroup: eight share a large weight; four where a wave holds more than 256 registers' worth, and where
// little enough is held that several workgroups fit a compute unit and need not wait together (640000 rows 39 -> 3
// float32 there and back: 153 us by eights, 134 us by fours, with a grid of four to a unit).
constexpr int stream_waves(int ks, int ns, int size)
{
    return ks * ns <= 8 || ks * ns > 32 || ks > 8 || ns > 8 || (size == 2 && (ks > 4 || ns > 4)) ? 4 : 8;
}
// Workgroups of a compute unit: at most what its registers hold, so that the launch is one round and no unit works on a
// second while others wait.  A table, kept by hand with the compiler's report: it is the kernel's launch bound, so the
// compiler makes the registers fit, and the smallest (one or two steps in all), of which five to seven would fit, stay at
// four (640000 rows 39 (of 64) -> 3 float32 there and back: 116 us, 133 us
// with four workgroups where three were held; 200 -> 3 bfloat16 190 us, 278 us).
constexpr int stream_per_cu(int ks, int ns, int size)
{
    if (stream_waves(ks, ns, size) == 8) return 1;
    if (size == 4) return ks * ns <= 4 ? 4 : ks * ns <= 8 ? (ks <= 4 && ns <= 4 ? 3 : 2) : 1;
    return ks * ns <= 2 ? 4 : ks * ns <= 4 && ns <= 2 ? 3 : ks * ns <= 8 && ns <= 4 ? 2 : 1;
}

template <typename T>
struct StreamBackward {
    long long rows, tiles;
    int k, n;
    const T *x, *w, *bias, *dy;
    long long ldx, ldw, lddy;
    int act;
    T* dx;           // or NULL
    bool dw, db;
    float* partial;  // [workgroup][n k + n]: sums for dW, then for db
};

// KS, NS: steps of four chunks that a row of x and of dz take; SHORT_X, SHORT_Z: they are shorter than
// a chunk.  As in the forward pass, dx is kept until the next rows have arrived, where there are registers for it.
template <typename T, int KS, int NS, bool SHORT_X, bool SHORT_Z, int WAVES>
__global__ __launch_bounds__(64 * WAVES, stream_per_cu(KS, NS, sizeof(T)) * (WAVES / 4))
void stream_backward_kernel(StreamBackward<T> a)
{
    constexpr int N = Chunk<T>::N, CK = KS * 4, CN = NS * 4, PARTS = N / 4;
    constexpr int TK = CK * N, TN = CN * N, TM = WAVES * 16;          // columns of x, columns of dz, rows of a tile
    constexpr int FK = TK / 16, FN = TN / 16, EACH = (FK * FN + WAVES - 1) / WAVES;  // dW's fragments, and a wave's share:
    constexpr int EK0 = EACH >= 8 ? 4 : EACH >= 2 ? 2 : 1, EK1 = EK0 < FK ? EK0 : FK;
    constexpr int EN = EACH / EK1 < FN ? EACH / EK1 : FN, EK = EACH / EN;   // EK by EN of them
    static_assert(FK % EK == 0 && FN % EN == 0, "shares fill dW");
    constexpr int STEPS = TM / (16 * PARTS);                          // reduction steps over a tile's rows
    typedef WeightTile<T, CK> W;
    typedef Tile<T, true, TK> TileX;
    typedef Tile<T, true, TN> TileZ;
    __shared__ __attribute__((aligned(16))) char weight[TN * CK * 16];
    __shared__ __attribute__((aligned(16))) char tile_x[TM * CK * 16];
    __shared__ __attribute__((aligned(16))) char tile_z[TM * CN * 16];
    __shared__ __attribute__((aligned(16))) float bias[TN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15;
    // Of KS and NS steps, and of FK and FN fragments, those that the widths fill; the rest is left out where there is much
    // of it to leave out.  (The branches are uniform, but they keep the compiler from interleaving what they part: at up
    // to four steps each, 640000 x 128 -> 128 bfloat16 there and back took 323 us with them and takes 259 us without.)
    constexpr bool TRIM = KS * NS > (sizeof(T) == 4 ? 32 : 16);
    const int ks = TRIM ? (a.k + 4 * N - 1) / (4 * N) : KS, ns = TRIM ? (a.n + 4 * N - 1) / (4 * N) : NS;
    const int fk = TRIM ? (a.k + 15) / 16 : FK, fn = TRIM ? (a.n + 15) / 16 : FN;
    // what only the wanted gradients read may be NULL: dx alone needs no x, dW alone no weight, unless z is formed again
    const bool uses_x = a.dw || a.act != NGS_ACT_NONE, uses_w = a.dx || a.act != NGS_ACT_NONE;
    if (uses_w) W::fill(weight, a.w, a.ldw, a.n, a.k, TN, tid, 64 * WAVES);
    for (int c = tid; c < TN; c += 64 * WAVES) bias[c] = a.bias && c < a.n ? (float)a.bias[c] : 0.0f;
    __syncthreads();

    const RowChunks<T, SHORT_X> xc(a.k);
    const RowChunks<T, SHORT_Z> zc(a.n);
    // db of 16-bit types gathers beside dz, unrounded; of floats it comes from the matrix units, as the product of ones
    // with the tile's dz, which costs a register per 16 columns and wave instead of N per step
    constexpr bool DB_MMA = sizeof(T) == 4;
    constexpr int DB_EACH = (FN + WAVES - 1) / WAVES;
    const bool tiles_wanted = a.dw || (DB_MMA && a.db);
    // this wave's share, in strides so that a width that does not fill the steps is shared evenly
    constexpr int WK = FK / EK, WN = FN / EN;
    const int kf0 = wave % WK, nf0 = wave / WK < WN ? wave / WK : FN;
    f32x4 acc[EACH], dbm[DB_EACH];
    float db[DB_MMA ? 1 : NS][N];
#pragma unroll
    for (int e = 0; e < EACH; e++) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < DB_EACH; e++) dbm[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < (DB_MMA ? 1 : NS); s++)
#pragma unroll
        for (int e = 0; e < N; e++) db[s][e] = 0.0f;

    constexpr bool HOLD = KS + NS < 8;  // (where the registers allow it)
    u32x4 nx[KS], ng[NS], dx[KS];
    auto store = [&](long long t) {
        const long long r = t * TM + wave * 16 + i;
        if (r >= a.rows) return;
#pragma unroll
        for (int b = 0; b < KS; b++) RowChunks<T>::store(a.dx + r * a.k, dx[b], b * 4 + W::chunk_of(g), b * 4, a.k);
    };
    auto fetch = [&](long long t) {
        const long long r = t * TM + wave * 16 + i, row = r < a.rows ? r : a.rows - 1;
        const T *const px = a.x + row * a.ldx, *const pg = a.dy + row * a.lddy;
#pragma unroll
        for (int s = 0; s < KS; s++)
            if (uses_x && s < ks) nx[s] = xc.fetch(px, s * 4 + g);
#pragma unroll
        for (int s = 0; s < NS; s++)
            if (s < ns) ng[s] = zc.fetch(pg, s * 4 + g);
    };
#pragma unroll
    for (int s = 0; s < KS; s++) nx[s] = (u32x4){0, 0, 0, 0};
    fetch(blockIdx.x);
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        const bool there = t * TM + wave * 16 + i < a.rows;
        u32x4 x[KS], dz[NS];
#pragma unroll
        for (int s = 0; s < KS; s++)
            if (s < ks) x[s] = xc.settle(nx[s], s * 4 + g, s * 4, there);
#pragma unroll
        for (int s = 0; s < NS; s++)
            if (s < ns) dz[s] = zc.settle(ng[s], s * 4 + g, s * 4, there);
        if (HOLD && a.dx && t != blockIdx.x) store(t - gridDim.x);
        if (t + gridDim.x < a.tiles) fetch(t + gridDim.x);

        if (a.act != NGS_ACT_NONE || (!DB_MMA && a.db)) {
#pragma unroll
            for (int s = 0; s < NS; s++) {
                if (s < ns) {
                    float d[N];
                    unpack<T>(dz[s], d);
                    if (a.act != NGS_ACT_NONE) {
                        float z[N], y[N], slope[N];
#pragma unroll
                        for (int h = 0; h < PARTS; h++) {
                            f32x4 c = *(const f32x4*)&bias[(s * 4 + g) * N + h * 4];
#pragma unroll
                            for (int q = 0; q < KS; q++)
                                if (q < ks) c = mma(W::along(weight, s * PARTS + h, q, lane), x[q], c, (const T*)nullptr);
#pragma unroll
                            for (int e = 0; e < 4; e++) z[h * 4 + e] = c[e];
                        }
                        activate<N>(a.act, z, y, slope);
                        // (behind the last column z may be NaN where x is not finite, and must not reach dx)
                        const int left = a.n - (s * 4 + g) * N;
                        const bool whole = (s * 4 + 4) * N <= a.n;  // uniform
#pragma unroll
                        for (int e = 0; e < N; e++) d[e] = whole || e < left ? d[e] * slope[e] : 0.0f;
                        dz[s] = pack<T>(d);  // (rounded for the matrix units: see linear_dz_kernel)
                    }
                    if constexpr (!DB_MMA) {
#pragma unroll
                        for (int e = 0; e < N; e++) db[s][e] += d[e];
                    }
                }
            }
        }
        if (tiles_wanted) {
            const int line = wave * 16 + i;
#pragma unroll
            for (int s = 0; s < KS; s++)
                if (s < ks) TileX::put(tile_x, line * CK + s * 4 + g, x[s]);
#pragma unroll
            for (int s = 0; s < NS; s++)
                if (s < ns) TileZ::put(tile_z, line * CN + s * 4 + g, dz[s]);
        }
        if (a.dx) {
#pragma unroll
            for (int b = 0; b < KS; b++) {
                if (b < ks) {
                    f32x4 c[PARTS];
#pragma unroll
                    for (int h = 0; h < PARTS; h++) c[h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < NS; s++) {
#pragma unroll
                        for (int h = 0; h < PARTS; h++)
                            if (s < ns) c[h] = mma(W::across(weight, b * PARTS + h, s, lane), dz[s], c[h], (const T*)nullptr);
                    }
                    float d[N];
#pragma unroll
                    for (int e = 0; e < N; e++) d[e] = c[e / 4][e % 4];
                    dx[b] = W::join(pack<T>(d));
                    if (!HOLD && there) RowChunks<T>::store(a.dx + (t * TM + wave * 16 + i) * a.k, dx[b], b * 4 + W::chunk_of(g), b * 4, a.k);
                }
            }
        }
        if (tiles_wanted) {
            __syncthreads();
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                if constexpr (DB_MMA) {
                    const u32x4 ones = (u32x4){0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u};
#pragma unroll
                    for (int e = 0; e < DB_EACH; e++) {
                        const int f = wave + e * WAVES;
                        if (f < fn) dbm[e] = mma(ones, TileZ::fragment(tile_z, f, s, lane), dbm[e], (const T*)nullptr);
                    }
                }
                u32x4 f[EK];
#pragma unroll
                for (int e = 0; e < EK; e++)
                    if (kf0 + e * WK < fk) f[e] = TileX::fragment(tile_x, kf0 + e * WK, s, lane);
#pragma unroll
                for (int o = 0; o < EN; o++) {
                    if (nf0 + o * WN < fn) {
                        const u32x4 h = TileZ::fragment(tile_z, nf0 + o * WN, s, lane);
#pragma unroll
                        for (int e = 0; e < EK; e++)
                            if (kf0 + e * WK < fk) acc[o * EK + e] = mma(f[e], h, acc[o * EK + e], (const T*)nullptr);
                    }
                }
            }
            __syncthreads();
        }
    }

    if (HOLD && a.dx) store(blockIdx.x + (a.tiles - 1 - blockIdx.x) / gridDim.x * gridDim.x);
    float* const out = a.partial + (long long)blockIdx.x * ((long long)a.n * a.k + a.n);
    if (a.dw) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int col = (kf0 + e % EK * WK) * 16 + g * 4, row = (nf0 + e / EK * WN) * 16 + i;
            if (row < a.n && col < a.k) {
                const float v[4] = {acc[e][0], acc[e][1], acc[e][2], acc[e][3]};
                store4(out + (long long)row * a.k + col, v, a.k - col);
            }
        }
    }
    if (DB_MMA && a.db) {
#pragma unroll
        for (int e = 0; e < DB_EACH; e++) {
            const int f = wave + e * WAVES, col = f * 16 + i;
            if (f < FN && g == 0 && col < a.n) out[(long long)a.n * a.k + col] = dbm[e][0];
        }
    }
    if constexpr (!DB_MMA) {
        if (!a.db) return;
        // over the 16 rows of a wave, then over the waves
        __syncthreads();
        float* const sums = (float*)tile_z;  // [WAVES][TN]: TM lines of TN elements hold it
        static_assert(WAVES * TN * 4 <= TM * CN * 16, "the waves' sums fit the tile");
#pragma unroll
        for (int s = 0; s < NS; s++) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                float v = db[s][e];
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
                if (i == 0) sums[wave * TN + (s * 4 + g) * N + e] = v;
            }
        }
        __syncthreads();
        for (int c = tid; c < a.n; c += 64 * WAVES) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < WAVES; k++) v += sums[k * TN + c];
            out[(long long)a.n * a.k + c] = v;
        }
    }
}

// ---------------------------------------------------------------------------
// Launch shapes
// ---------------------------------------------------------------------------
inline int steps_of(long long width, int dtype)  // steps of four chunks, as a power of two
{
    const long long per = 64 / (long long)ngs_decoder_size(dtype);
    int s = 1;
    while (s * per < width) s *= 2;
    return s;
}

// groups of four chunks of the result per workgroup: 1, 4 or 8
inline int stream_blocks(int n, int dtype)
{
    const int per = 64 / (int)ngs_decoder_size(dtype), b = (n + per - 1) / per;
    return b <= 1 ? 1 : b <= 4 ? 4 : 8;
}

template <typename T, int KS, int NB, bool SHORT, bool RESIDUAL>
static int stream_forward_launch(hipStream_t st, const StreamForward<T>& a)
{
    constexpr int COLS = NB * 4 * Chunk<T>::N, LDS = COLS * (KS * 64 + 4);
    constexpr int THREADS = LDS > 32 * 1024 ? 512 : 256;
    // Two rounds of what a compute unit holds at a time: a part of a round would leave units idle at the end, and with one
    // round alone the slowest workgroup is waited for (2000000 rows 64 -> 3 bfloat16 with residual: 84 us; 97 us with eight
    // to a unit, of which six are held; 32 -> 32: 75 us, 83 us with eight, 89 us with one round).
    static const int held = [] {
        int n = 0;
        const void* const kernel = (const void*)stream_forward_kernel<T, KS, NB, SHORT, RESIDUAL, THREADS>;
        return hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, THREADS, 0) == hipSuccess && n > 0 ? n : 4;
    }();
    const long long need = ((a.rows + 15) / 16 + THREADS / 64 - 1) / (THREADS / 64), most = 2LL * NGS_CUS * held;
    const dim3 grid((unsigned)(need < most ? need : most), (unsigned)((a.n + COLS - 1) / COLS));
    hipLaunchKernelGGL((stream_forward_kernel<T, KS, NB, SHORT, RESIDUAL, THREADS>), grid, dim3(THREADS), 0, st, a);
    return ngs_decoder_launched("ngs_linear_forward");
}

template <typename T, int KS, bool SHORT = false>
static int stream_forward_of(hipStream_t st, const StreamForward<T>& a, int dtype)
{
    const int blocks = stream_blocks(a.n, dtype);
#define NGS_STREAM_FORWARD(NB) \
    (a.residual ? stream_forward_launch<T, KS, NB, SHORT, true>(st, a) : stream_forward_launch<T, KS, NB, SHORT, false>(st, a))
    if (blocks == 1) return NGS_STREAM_FORWARD(1);
    // (eight steps and eight groups do not fit a wave's registers: the rows pass twice)
    if constexpr (KS < 8)
        if (blocks == 8) return NGS_STREAM_FORWARD(8);
    return NGS_STREAM_FORWARD(4);
#undef NGS_STREAM_FORWARD
}

template <typename T>
int ngs_stream_forward(hipStream_t st, long long rows, int k, int n, int dtype, const T* x, long long ldx, const T* w,
                       long long ldw, const Epilogue<T>& e)
{
    const StreamForward<T> a = {rows, k, n, x, w, e.bias, e.residual, ldx, ldw, e.ldr, e.act, e.y, e.slope};
    if (k < Chunk<T>::N) return stream_forward_of<T, 1, true>(st, a, dtype);
    switch (steps_of(k, dtype)) {
    case 1: return stream_forward_of<T, 1>(st, a, dtype);
    case 2: return stream_forward_of<T, 2>(st, a, dtype);
    case 4: return stream_forward_of<T, 4>(st, a, dtype);
    default: return stream_forward_of<T, 8>(st, a, dtype);
    }
}

template <typename T, int KS, int NS, bool SHORT_X, bool SHORT_Z = false>
static int stream_backward_launch(hipStream_t st, StreamBackward<T> a, unsigned blocks)
{
    constexpr int WAVES = stream_waves(KS, NS, sizeof(T));
    a.tiles = (a.rows + WAVES * 16 - 1) / (WAVES * 16);
    hipLaunchKernelGGL((stream_backward_kernel<T, KS, NS, SHORT_X, SHORT_Z, WAVES>), dim3(blocks), dim3(64 * WAVES), 0, st, a);
    return ngs_decoder_launched("ngs_linear_backward");
}

template <typename T, int KS, bool SHORT_X = false>
static int stream_backward_of(hipStream_t st, const StreamBackward<T>& a, int ns, unsigned blocks)
{
    constexpr int MOST = stream_most(sizeof(T)) / KS;  // steps of dz beside KS of x
    if (a.n < Chunk<T>::N) return stream_backward_launch<T, KS, 1, SHORT_X, true>(st, a, blocks);
    if (ns == 1) return stream_backward_launch<T, KS, 1, SHORT_X>(st, a, blocks);
    if (ns == 2) return stream_backward_launch<T, KS, 2, SHORT_X>(st, a, blocks);
    if (ns == 4) return stream_backward_launch<T, KS, 4, SHORT_X>(st, a, blocks);
    if constexpr (MOST >= 8)
        if (ns == 8) return stream_backward_launch<T, KS, 8, SHORT_X>(st, a, blocks);
    if constexpr (MOST >= 16 && sizeof(T) == 4)
        if (ns == 16) return stream_backward_launch<T, KS, 16, SHORT_X>(st, a, blocks);
    return ngs_set_error("ngs_linear_backward", "no kernel for this width");
}

template <typename T>
int ngs_stream_backward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const T* x, long long ldx,
                        const T* w, long long ldw, const T* bias, const T* dy, long long lddy, T* dx, T* dw, T* db,
                        float* partial)
{
    const StreamBackward<T> a = {rows, 0, k, n, x, w, bias, dy, ldx, ldw, lddy, act, dx, dw != nullptr, db != nullptr, partial};
    const unsigned blocks = (unsigned)ngs_stream_backward_blocks(rows, k, n, dtype);
    const int ns = steps_of(n, dtype);
    const int ks = steps_of(k, dtype);
    int rc;
    if (k < Chunk<T>::N) {
        rc = stream_backward_of<T, 1, true>(st, a, ns, blocks);
    } else if (ks == 1) {
        rc = stream_backward_of<T, 1>(st, a, ns, blocks);
    } else if (ks == 2) {
        rc = stream_backward_of<T, 2>(st, a, ns, blocks);
    } else if (ks == 4) {
        rc = stream_backward_of<T, 4>(st, a, ns, blocks);
    } else if (ks == 8) {
        rc = stream_backward_of<T, 8>(st, a, ns, blocks);
    } else {
        if constexpr (sizeof(T) == 4) rc = stream_backward_of<T, 16>(st, a, ns, blocks);
        else rc = ngs_set_error("ngs_linear_backward", "no kernel for this width");
    }
    if (rc) return rc;
    if (dw || db) ngs_launch_column_finish(st, partial, blocks, (long long)n * k, n, dw, db, dtype);
    return ngs_decoder_launched("ngs_linear_backward");
}

#define NGS_STREAM_INSTANCE(T)                                                                                             \
    template int ngs_stream_forward<T>(hipStream_t, long long, int, int, int, const T*, long long, const T*, long long,    \
                                       const Epilogue<T>&);                                                                \
    template int ngs_stream_backward<T>(hipStream_t, long long, int, int, int, int, const T*, long long, const T*,         \
                                        long long, const T*, const T*, long long, T*, T*, T*, float*);
