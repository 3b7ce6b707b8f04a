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
    // how far rows may be read (zeros behind their end where they are padded): of an operand that lies across, its np or
    // nq columns; of one that lies along, the reduction's nr
    long long width_p, width_q, along;
    long long tiles_p, tiles_q;
    // The first `full` tiles are computed whole, by `full_groups` workgroups (a multiple of the dies); each of the others
    // by `parts` workgroups, which take `run` elements of the reduction each (a multiple of a step's) and, if there is
    // more than one, leave their sums in partial[workgroup][q in tile][p in tile].
    long long full, full_groups, run;
    int parts;
    float* partial;
    Epilogue<T> epi;
};

// Which tile and which run of the reduction a workgroup computes.  Workgroups go to the dies in turn: each die takes a
// contiguous run of the whole tiles, whose operands meet in its cache.
struct Place {
    long long p0, q0, r_begin, r_end;
    float* partial;  // where the sums go, if the tile is shared
    bool there;
};
template <typename T, int TP, int TQ>
__device__ __forceinline__ Place place_of(const Product<T>& a)
{
    Place w;
    long long tile;
    w.r_begin = 0;
    w.r_end = a.nr;
    w.partial = nullptr;
    if (blockIdx.x < a.full_groups) {
        tile = (long long)(blockIdx.x % NGS_XCDS) * (a.full_groups / NGS_XCDS) + blockIdx.x / NGS_XCDS;
        w.there = tile < a.full;
    } else {
        const long long u = blockIdx.x - a.full_groups;
        tile = a.full + u / a.parts;
        w.there = true;
        if (a.parts > 1) {
            w.r_begin = u % a.parts * a.run;
            w.r_end = w.r_begin + a.run < a.nr ? w.r_begin + a.run : a.nr;
            w.partial = a.partial + u * (TP * TQ);
        }
    }
    w.p0 = (tile % a.tiles_p) * TP;
    w.q0 = (tile / a.tiles_p) * TQ;
    return w;
}

// A wave's share of a tile's sums, `first` elements into it
template <int MP, int MQ, int TP>
__device__ __forceinline__ void leave_partial(float* partial, const f32x4 (&acc)[MP][MQ], int p, int q, int lane)
{
#pragma unroll
    for (int i = 0; i < MP; i++)
#pragma unroll
        for (int j = 0; j < MQ; j++)
            *(f32x4*)&partial[(q + j * 16 + (lane & 15)) * TP + p + i * 16 + (lane >> 4) * 4] = acc[i][j];
}

// A wave's MP x MQ fragments from (p0, q0) on: a lane holds four neighbouring p of one q.
template <typename T, int MP, int MQ>
__device__ __forceinline__ void finish_tile(const Product<T>& a, const f32x4 (&acc)[MP][MQ], long long p0, long long q0, int lane)
{
#pragma unroll
    for (int i = 0; i < MP; i++) {
        const int p = (int)p0 + i * 16 + (lane >> 4) * 4;
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p < a.np && a.epi.bias) load4(a.epi.bias + p, bias, a.np - p);
#pragma unroll
        for (int j = 0; j < MQ; j++) {
            const long long q = q0 + j * 16 + (lane & 15);
            if (p < a.np && q < a.nq) finish4(a.epi, q, p, acc[i][j], bias);
        }
    }
}

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
    const Place at = place_of<T, TP, TQ>(a);
    if (!at.there) return;
    const long long p0 = at.p0, q0 = at.q0, r_begin = at.r_begin, r_end = at.r_end;

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

    if (at.partial) leave_partial<MP, MQ, TP>(at.partial, acc, wp * MP * 16, wq * MQ * 16, lane);
    else finish_tile<T, MP, MQ>(a, acc, p0 + wp * MP * 16, q0 + wq * MQ * 16, lane);
}

// The same with operands that lie on 16-byte boundaries: they go from memory into shared memory without passing
// through registers, the next step's while this one is multiplied.  With 256 x 256 tiles and eight waves (128 x 64 each)
// the matrix units have 2048 cycles of work per step of 64 16-bit elements and the fragments' reads take 1536 of the
// shared memory's: bound by the matrix units (8192 x 4096 -> 4096 bfloat16 233 to 240 us, 1150 TFLOP/s or more, of
// 1290 that a large library product reaches; float32 2012 us, 137 of 153 TFLOP/s).
//
// A wave's load fills 1 KiB of a tile in lane order; which chunk a lane fetches undoes the exchange of the tile's layout.
// What lies beyond the operand's end reads as zero (the resource's bound), and so does, along, what lies beyond the
// reduction's (an offset past the bound).
template <typename T, bool ACROSS, int ROWS, int WAVES>
struct TileLoader {
    static constexpr int N = Chunk<T>::N, STEP = ROW_BYTES / (int)sizeof(T), LINE = ROWS * (int)sizeof(T) / 16;
    static constexpr int LOADS = ROWS * ROW_BYTES / 1024 / WAVES;
    static_assert(LOADS * WAVES * 1024 == ROWS * ROW_BYTES, "loads divide over the waves");
    uint32_t offset[LOADS];
    const char* base;
    long long left, advance;  // bytes from base to the operand's end (of the reduction, across), and per step
    int first;                // along: this lane's first reduction element in a step

    __device__ __forceinline__ TileLoader(const T* p, long long ld, long long row0, long long rows, long long r0, long long r_end,
                                          int wave, int lane)
    {
        if (!ACROSS) {
            base = (const char*)(p + row0 * ld + r0);
            left = ((rows - 1 - row0) * ld + (r_end - r0)) * (long long)sizeof(T);
            advance = ROW_BYTES;
            const int c = (lane & 7) ^ (lane >> 3);
            first = c * N;
#pragma unroll
            for (int k = 0; k < LOADS; k++)
                offset[k] = (uint32_t)((k * WAVES + wave) * 8 + (lane >> 3)) * (uint32_t)(ld * sizeof(T)) + c * 16;
        } else {
            base = (const char*)(p + r0 * ld + row0);
            left = ((r_end - 1 - r0) * ld + (rows - row0)) * (long long)sizeof(T);
            advance = STEP * ld * (long long)sizeof(T);
            first = 0;
#pragma unroll
            for (int k = 0; k < LOADS; k++) {
                const int i = (k * WAVES + wave) * 64 + lane, line = i / LINE;
                const int c = (i % LINE) ^ (Tile<T, true, ROWS>::segment_swap(line) * Tile<T, true, ROWS>::SEG);
                offset[k] = (uint32_t)line * (uint32_t)(ld * sizeof(T)) + c * 16;
            }
        }
    }
    // the next step's tile into `lds` (an address in shared memory); `length`: reduction elements that are left
    __device__ __forceinline__ void load(uint32_t lds, long long length, int wave)
    {
        const uint64_t b = (uint64_t)base;
        const long long bytes = left < 0 ? 0 : left < 0x7ffffff0 ? left : 0x7ffffff0;
        u32x4 rsrc;
        rsrc.x = __builtin_amdgcn_readfirstlane((uint32_t)b);
        rsrc.y = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32) & 0xffffu);
        rsrc.z = __builtin_amdgcn_readfirstlane((uint32_t)bytes);
        rsrc.w = 0x00020000u;
        const bool beyond = !ACROSS && first >= length;
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
            const uint32_t o = beyond ? 0x7ffffff0u : offset[k];
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (k * WAVES + wave) * 1024);
            // (the compiler does not see the load in here: a scalar register of the resource that a vector instruction has
            // just written is only safe to read five wait states later)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved: nothing of the compiler's lives in it across the statement)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :: "s"(to), "v"(o), "s"(rsrc) : "memory", "m0");
#pragma clang diagnostic pop
        }
        base += advance;
        left -= advance;
    }
};

// A wave's results through its own piece of shared memory, 16 rows at a time, so that they leave as whole lines and the
// epilogue's code is there once per 16 rows rather than once per fragment.  BARE: no epilogue.
template <typename T, int MP>
constexpr int finish_wide_bytes() { return 16 * (MP * 16 + 4) * 4 + 16 * MP * 16 * (int)sizeof(T); }  // a wave's piece

template <typename T, int MP, int MQ, bool BARE>
__device__ __forceinline__ void finish_wide(const Product<T>& a, const f32x4 (&acc)[MP][MQ], float* lds, long long p0,
                                            long long q0, int lane)
{
    constexpr int N = Chunk<T>::N, PITCH = MP * 16 + 4, LANES = MP * 16 / N, ROWS = 64 / LANES, TRIPS = 16 / ROWS;
    const int g = lane >> 4, i = lane & 15;
    const int col = (lane % LANES) * N, p = (int)p0 + col, valid = a.np - p;
    float bias[N];
#pragma unroll
    for (int e = 0; e < N; e++) bias[e] = 0.0f;
    if (!BARE && a.epi.bias && valid > 0) unpack<T>(load16_head(a.epi.bias + p, valid), bias);
    // the residual's chunks of the next 16 rows are on their way while these are finished; they wait in shared memory, so
    // that the loop over the rows can stay a loop
    u32x4 res[TRIPS];
    u32x4* const parked = (u32x4*)(lds + 16 * PITCH) + lane;
    auto fetch = [&](int j) {
#pragma unroll
        for (int t = 0; t < TRIPS; t++) {
            const long long q = q0 + j * 16 + t * ROWS + lane / LANES;
            res[t] = load16_head(a.epi.residual + (q < a.nq ? q : 0) * a.epi.ldr + p, valid);
        }
    };
    if (!BARE && a.epi.residual) fetch(0);
#pragma unroll
    for (int j = 0; j < MQ; j++) {
#pragma unroll
        for (int f = 0; f < MP; f++) *(f32x4*)&lds[i * PITCH + f * 16 + g * 4] = acc[f][j];
        if (!BARE && a.epi.residual) {
#pragma unroll
            for (int t = 0; t < TRIPS; t++) parked[t * 64] = res[t];
            if (j + 1 < MQ) fetch(j + 1);
        }
        __builtin_amdgcn_wave_barrier();  // (one wave's accesses to shared memory are in order)
#pragma unroll 1
        for (int t = 0; t < TRIPS; t++) {
            const int r = t * ROWS + lane / LANES;
            const long long q = q0 + j * 16 + r;
            if (q >= a.nq || valid <= 0) continue;
            float z[N], y[N];
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const f32x4 v = *(const f32x4*)&lds[r * PITCH + col + e];
#pragma unroll
                for (int k = 0; k < 4; k++) z[e + k] = v[k] + bias[e + k];
            }
            if constexpr (BARE) {
                store16_head(a.epi.y + q * a.np + p, pack<T>(z), valid);
            } else {
                float slope[N];
                if (a.epi.slope) {
                    activate<N>(a.epi.act, z, y, slope);
                    // (into the place of z: its chunks are twice a result's of 16 bits, and leave below in whole lines)
#pragma unroll
                    for (int e = 0; e < N; e += 4)
                        *(f32x4*)&lds[r * PITCH + col + e] = (f32x4){slope[e], slope[e + 1], slope[e + 2], slope[e + 3]};
                } else {
                    activate<N>(a.epi.act, z, y, nullptr);
                }
                if (a.epi.residual) {
                    float f[N];
                    unpack<T>(parked[t * 64], f);
#pragma unroll
                    for (int e = 0; e < N; e++) y[e] += f[e];
                }
                store16_head(a.epi.y + q * a.np + p, pack<T>(y), valid);
            }
        }
        __builtin_amdgcn_wave_barrier();
        if (!BARE && a.epi.slope) {
            constexpr int QUADS = MP * 4;  // of a row
#pragma unroll 1
            for (int t = lane; t < 16 * QUADS; t += 64) {
                const int r = t / QUADS, c = t % QUADS * 4;
                const long long q = q0 + j * 16 + r;
                if (q >= a.nq || p0 + c >= a.np) continue;
                const f32x4 v = *(const f32x4*)&lds[r * PITCH + c];
                const float four[4] = {v[0], v[1], v[2], v[3]};
                store4(a.epi.slope + q * a.np + p0 + c, four, a.np - (int)p0 - c);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <typename T, bool P_ACROSS, bool Q_ACROSS, int TP, int TQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void product_direct_kernel(Product<T> a)
{
    typedef Tile<T, P_ACROSS, TP> TileP;
    typedef Tile<T, Q_ACROSS, TQ> TileQ;
    constexpr int WAVES = WP * WQ, STEP = TileP::STEP, MP = TP / WP / 16, MQ = TQ / WQ / 16;
    constexpr int P_BYTES = TP * ROW_BYTES, STAGE = (TP + TQ) * ROW_BYTES;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = wave % WP, wq = wave / WP;
    const Place at = place_of<T, TP, TQ>(a);
    if (!at.there) return;

    f32x4 acc[MP][MQ];
#pragma unroll
    for (int i = 0; i < MP; i++)
#pragma unroll
        for (int j = 0; j < MQ; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    const long long r_read = at.r_end == a.nr ? a.along : at.r_end;
    TileLoader<T, P_ACROSS, TP, WAVES> lp(a.p, a.ldp, at.p0, a.width_p, at.r_begin, P_ACROSS ? at.r_end : r_read, wave, lane);
    TileLoader<T, Q_ACROSS, TQ, WAVES> lq(a.q, a.ldq, at.q0, a.width_q, at.r_begin, Q_ACROSS ? at.r_end : r_read, wave, lane);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const long long length = at.r_end - at.r_begin;
    if (length > 0) {
        lp.load(lds0, length, wave);
        lq.load(lds0 + P_BYTES, length, wave);
    }
    int buf = 0;
    for (long long r = 0; r < length; r += STEP) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // this step's tiles are there, the other buffer is free
        if (r + STEP < length) {
            const uint32_t to = lds0 + (buf ^ 1) * STAGE;
            lp.load(to, length - r - STEP, wave);
            lq.load(to + P_BYTES, length - r - STEP, wave);
        }
        const char *const sp = lds + buf * STAGE, *const sq = sp + P_BYTES;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            u32x4 f[MP], h[MQ];
#pragma unroll
            for (int j = 0; j < MQ; j++) h[j] = TileQ::fragment(sq, wq * MQ + j, s, lane);
#pragma unroll
            for (int i = 0; i < MP; i++) f[i] = TileP::fragment(sp, wp * MP + i, s, lane);
#pragma unroll
            for (int i = 0; i < MP; i++)
#pragma unroll
                for (int j = 0; j < MQ; j++) acc[i][j] = mma(f[i], h[j], acc[i][j], (const T*)nullptr);
        }
        buf ^= 1;
    }
    if (at.partial) {
        leave_partial<MP, MQ, TP>(at.partial, acc, wp * MP * 16, wq * MQ * 16, lane);
        return;
    }
    __syncthreads();  // the tiles are done with
    static_assert(WAVES * finish_wide_bytes<T, MP>() <= 2 * STAGE, "a piece of the tiles' memory for each wave");
    finish_wide<T, MP, MQ, P_ACROSS>(a, acc, (float*)(lds + wave * finish_wide_bytes<T, MP>()), at.p0 + wp * MP * 16, at.q0 + wq * MQ * 16,
                                     lane);
}

// Adds up the parts of the tiles that several workgroups share, in their order, and finishes them (for
// 4099 x 1001 -> 2003 float16 4.5 us: a launch and a short pass).
template <typename T>
__global__ __launch_bounds__(256) void product_finish_kernel(const float* __restrict__ partial, int parts, long long full,
                                                             long long tiles_p, int tp, int tq, long long nq, Epilogue<T> e)
{
    const int quads = tp / 4 * tq, per = quads / 256;  // workgroups per tile
    const long long shared = blockIdx.x / per, tile = full + shared;
    const int i = (int)(blockIdx.x % per) * 256 + threadIdx.x, pt = i % (tp / 4) * 4, qt = i / (tp / 4);
    const long long q = tile / tiles_p * tq + qt, p0 = tile % tiles_p * tp + pt;
    if (p0 >= e.np || q >= nq) return;
    const int p = (int)p0;
    const float* at = partial + shared * parts * (tp * tq) + qt * tp + pt;
    f32x4 sum = *(const f32x4*)at;
#pragma unroll 4
    for (int k = 1; k < parts; k++) sum += *(const f32x4*)(at + (long long)k * (tp * tq));
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e.bias) load4(e.bias + p, bias, e.np - p);
    finish4(e, q, p, sum, bias);
}

// ---------------------------------------------------------------------------
// dz = dL_dy * slope and the column sums of dz
// ---------------------------------------------------------------------------
// 16-bit types: dz is rounded to the type, as the matrix units take it, and a float16 dz beyond 65504 is infinite, as any
// float16 gradient is.  With the gradients' own rounding that puts them 1.4 roundings from their values instead of one
// (8192 x 4096 -> 4096 bfloat16: 0.0023 in norm, 0.0017 with dz in 32 bits).  What the rounding takes away could follow as
// a second operand: the two products of the backward pass would take twice their 553 us there, in a pass of 760 us.
//
// A workgroup is `across` threads wide (each owns a chunk of neighbouring columns) and 256 / across rows high; it
// walks down its share of the rows.  slope == NULL: dz is dL_dy and only summed.  Bound by memory: 8192 x 4096 bfloat16,
// 268 MB in 58 us (4.6 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(long long rows, int n, int across, const T* __restrict__ dy,
                                                        long long lddy, const float* __restrict__ slope,
                                                        T* __restrict__ dz, long long lddz, float* __restrict__ partial)
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
                    float s[N];
                    __builtin_memcpy(s, slope + r * n + col, sizeof s);
#pragma unroll
                    for (int i = 0; i < N; i++) g[i] *= s[i];
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (i < valid) g[i] *= slope[r * n + col + i];
                }
            }
            if (dz) store16_head(dz + r * lddz + col, pack<T>(g), lddz - col);
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

// COLS columns by 1024 / COLS rows of threads: a thread adds every so many rows, the threads' sums are joined pairwise.
// Sixteen columns spread a few columns over many threads; 64 read whole lines, where there are enough of them to fill
// the chip (512 x 10002: 12 us by 16, DRAM lines read in quarters, 6.3 us by 64).
template <typename T, int COLS>
__global__ __launch_bounds__(1024) void column_finish_kernel(const float* __restrict__ partial, long long blocks,
                                                             long long width0, long long width1, T* __restrict__ out0,
                                                             T* __restrict__ out1)
{
    constexpr int ROWS = 1024 / COLS;
    __shared__ float sums[ROWS][COLS + 1];
    const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
    const long long c = (long long)blockIdx.x * COLS + tx, pitch = width0 + width1;
    float s = 0.0f;
    if (c < pitch) {
#pragma unroll 8
        for (long long b = ty; b < blocks; b += ROWS) s += partial[b * pitch + c];
    }
    sums[ty][tx] = s;
    __syncthreads();
    for (int half = ROWS / 2; half > 0; half >>= 1) {
        if (ty < half) sums[ty][tx] += sums[ty + half][tx];
        __syncthreads();
    }
    if (ty != 0 || c >= pitch) return;
    T* const out = c < width0 ? out0 : out1;
    if (out) out[c < width0 ? c : c - width0] = (T)sums[0][tx];
}

template <typename T>
static void column_finish(hipStream_t s, const float* partial, long long blocks, long long width0, long long width1, void* out0,
                          void* out1)
{
    const long long pitch = width0 + width1;
    if (pitch >= 32 * NGS_CUS)
        hipLaunchKernelGGL((column_finish_kernel<T, 64>), dim3((unsigned)((pitch + 63) / 64)), dim3(1024), 0, s, partial, blocks,
                           width0, width1, (T*)out0, (T*)out1);
    else
        hipLaunchKernelGGL((column_finish_kernel<T, 16>), dim3((unsigned)((pitch + 15) / 16)), dim3(1024), 0, s, partial, blocks,
                           width0, width1, (T*)out0, (T*)out1);
}

void ngs_launch_column_finish(hipStream_t s, const float* partial, long long blocks, long long width0, long long width1,
                              void* out0, void* out1, int dtype)
{
    if (dtype == NGS_FLOAT32) column_finish<float>(s, partial, blocks, width0, width1, out0, out1);
    else if (dtype == NGS_FLOAT16) column_finish<f16>(s, partial, blocks, width0, width1, out0, out1);
    else column_finish<bf16>(s, partial, blocks, width0, width1, out0, out1);
}

// ---------------------------------------------------------------------------
// Launch shapes
// ---------------------------------------------------------------------------
struct Shape {
    int tp, tq;
    long long tiles_p, tiles_q, full, shared, run;  // as in Product; shared: tiles that `parts` workgroups share
    int parts;
    double cost;
    long long full_groups() const { return (full + NGS_XCDS - 1) / NGS_XCDS * NGS_XCDS; }
    size_t partial_bytes() const { return parts > 1 ? (size_t)shared * parts * tp * tq * 4 : 0; }
};

static inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Microseconds that `count` workgroups take for a step of their reductions, side by side on the chip, as measured
// (8192 x 4096 -> 4096 bfloat16, 64 steps: 2 rounds of 256 x 256 tiles 233 us, 4 rounds of 512 tiles of 128 x 128 317 us;
// 2048 x 2048 -> 2048, 32 steps: 256 tiles of 128 x 128 30 us; float32, where the matrix units bound any tile:
// 8192 x 4096 -> 4096, 128 steps: 2048 tiles of 128 x 128 2020 us).  Through registers, where what is large comes from rows
// that start off a word's boundary, about four times as long (801 x 5556, 801 x 269 -> 5556 x 269 bfloat16: 62 us for 13 steps).
static double step_us(int tp, int tq, long long count, int dtype, bool direct)
{
    const double rounds = (double)((count + NGS_CUS - 1) / NGS_CUS), area = (double)tp * tq / (128.0 * 128.0);
    if (dtype == NGS_FLOAT32) {
        const double busy = rounds * area * (direct ? 1.9 : 2.5);
        return count > 0 && busy < 0.8 ? 0.8 : busy;
    }
    if (tp == 256) return rounds * 1.9;
    const double whole = (double)(count / (2 * NGS_CUS));
    const long long rest = count % (2 * NGS_CUS);
    return (direct ? 1.0 : 4.0) * (1.25 * whole + (rest == 0 ? 0.0 : rest <= NGS_CUS ? 0.8 : 1.25)) * (area < 0.3 ? 0.6 : 1.0);
}

// Tiles of tp x tq, `slots` of which the chip works on at a time.  Rounds that fill it are computed whole.  The tiles of
// the last round may share the chip: each is cut along the reduction into parts of at least four steps, and a second
// kernel adds the parts up, which takes a launch and a way to memory and back.  5114 x 2776 -> 3400 bfloat16: 1080
// tiles of 128 x 128 on 512 slots, 146 us in whole tiles, 114 us with the last 56 shared.
static Shape shape_of(int tp, int tq, long long slots, long long np, long long nq, long long nr, int dtype, bool direct)
{
    Shape s;
    s.tp = tp;
    s.tq = tq;
    s.tiles_p = (np + tp - 1) / tp;
    s.tiles_q = (nq + tq - 1) / tq;
    const long long step = ROW_BYTES / (long long)ngs_decoder_size(dtype), steps = (nr + step - 1) / step;
    const long long tiles = s.tiles_p * s.tiles_q, last = tiles % slots;
    s.parts = 1;
    s.run = steps * step;
    s.full = tiles;
    s.cost = (double)steps * step_us(tp, tq, tiles, dtype, direct);
    const long long most = last > 0 ? (slots / last < steps / 4 ? slots / last : steps / 4) : 1;
    const double whole = (double)steps * step_us(tp, tq, tiles - last, dtype, direct);
    for (long long p = 2; p <= most; p = p < most && p + (p + 1) / 2 > most ? most : p + (p + 1) / 2) {
        const long long run = (steps + p - 1) / p, parts = (steps + run - 1) / run;
        const double bytes = 2.0 * 4.0 * (double)(last * parts) * tp * tq;
        const double cost = whole + (double)run * step_us(tp, tq, last * parts, dtype, direct) + 4.0 + bytes / 5.0e6;
        if (cost < s.cost) {
            s.cost = cost;
            s.parts = (int)parts;
            s.run = run * step;
            s.full = tiles - last;
        }
    }
    s.shared = tiles - s.full;
    return s;
}

// Through registers, tiles are 128 wide unless the matrix is 32 or narrower; directly, 128 x 128 or, of 16-bit types,
// 256 x 256, or, of float32, 64 x 64, whichever should take less time.
static Shape product_shape(long long np, long long nq, long long nr, int dtype, bool direct)
{
    if (!direct) return shape_of(np <= 32 ? 32 : 128, nq <= 32 ? 32 : 128, 2 * NGS_CUS, np, nq, nr, dtype, false);
    const Shape a = shape_of(128, 128, 2 * NGS_CUS, np, nq, nr, dtype, true);
    const Shape b = dtype == NGS_FLOAT32 ? shape_of(64, 64, 2 * NGS_CUS, np, nq, nr, dtype, true)
                                         : shape_of(256, 256, NGS_CUS, np, nq, nr, dtype, true);
    return b.cost < a.cost ? b : a;
}

// Whether product_direct_kernel has a tile for these sizes
static bool direct_sizes(long long np, long long nq) { return np > 32 && nq > 32; }

// Whether it can read an operand: whole aligned chunks, and offsets within a tile's rows in 31 bits
template <typename T>
static bool direct_operand(const T* p, long long ld, long long width)
{
    return (uintptr_t)p % 16 == 0 && ld % Chunk<T>::N == 0 && width % Chunk<T>::N == 0 && ld >= width && ld < (1LL << 21);
}

// Rows of an odd width are copied into rows of whole chunks first, zeros behind them, when the product is large against
// the copies (two launches and two passes over the operands): 4099 x 1001 -> 2003 half precision 61 us through registers.
static long long whole_chunks(long long width, int dtype)
{
    const long long n = 16 / (long long)ngs_decoder_size(dtype);
    return (width + n - 1) / n * n;
}
static bool pads(long long width, long long np, long long nq, long long nr, int dtype)
{
    return width != whole_chunks(width, dtype) && direct_sizes(np, nq) &&
           (double)np * (double)nq * (double)nr >= (dtype == NGS_FLOAT32 ? 268435456.0 : 536870912.0);
}

// (rows2 rows of a second matrix of the same width follow the first's.  Both of 4099 x 1001 and 2003 x 1001 float16 in
// one launch: 24 MB in 7.0 us.)
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(const T* __restrict__ from, long long ld, long long rows, int width,
                                                       T* __restrict__ to, const T* __restrict__ from2, long long ld2,
                                                       long long rows2)
{
    constexpr int N = Chunk<T>::N;
    const int chunks = (width + N - 1) / N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (rows + rows2) * chunks; i += (long long)gridDim.x * 256) {
        const long long r = i / chunks;
        const int c = (int)(i - r * chunks) * N;
        const T* const row = r < rows ? from + r * ld : from2 + (r - rows) * ld2;
        *(u32x4*)(to + r * chunks * N + c) = load16_head(row + c, width - c);
    }
}

template <typename T>
static void pad_rows(hipStream_t st, const T* from, long long ld, long long rows, int width, T* to,
                     const T* from2 = nullptr, long long ld2 = 0, long long rows2 = 0)
{
    const long long blocks = ((rows + rows2) * ((width + Chunk<T>::N - 1) / Chunk<T>::N) + 255) / 256;
    hipLaunchKernelGGL(pad_rows_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, from, ld, rows,
                       width, to, from2, ld2, rows2);
}

static size_t partial_bytes(long long np, long long nq, long long nr, int dtype)
{
    const size_t a = product_shape(np, nq, nr, dtype, false).partial_bytes();
    if (!direct_sizes(np, nq)) return a;
    const size_t b = product_shape(np, nq, nr, dtype, true).partial_bytes();
    return a > b ? a : b;
}

template <typename T, bool PA, bool QA>
static int launch_product(hipStream_t st, int dtype, Product<T> a, float* partial)
{
    const bool direct = direct_sizes(a.np, a.nq) && direct_operand(a.p, a.ldp, PA ? a.width_p : a.along) &&
                 direct_operand(a.q, a.ldq, QA ? a.width_q : a.along);
    const Shape s = product_shape(a.np, a.nq, a.nr, dtype, direct);
    a.tiles_p = s.tiles_p;
    a.tiles_q = s.tiles_q;
    a.full = s.full;
    a.full_groups = s.full_groups();
    a.parts = s.parts;
    a.run = s.run;
    a.partial = partial;
    a.epi.np = a.np;
    const long long groups = a.full_groups + s.shared * s.parts;
    if (ngs_decoder_grid("ngs_linear", groups, direct && s.tp == 256 ? 512 : 256)) return 1;
    const dim3 grid((unsigned)groups);
    if (direct && s.tp == 128) {
        hipLaunchKernelGGL((product_direct_kernel<T, PA, QA, 128, 128, 2, 2>), grid, dim3(256), 0, st, a);
    } else if (direct) {
        if constexpr (sizeof(T) == 2)
            hipLaunchKernelGGL((product_direct_kernel<T, PA, QA, 256, 256, 2, 4>), grid, dim3(512), 0, st, a);
        else
            hipLaunchKernelGGL((product_direct_kernel<T, PA, QA, 64, 64, 2, 2>), grid, dim3(256), 0, st, a);
    } else if (s.tp == 128 && s.tq == 128) {
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 128, 128, 2, 2>), grid, dim3(256), 0, st, a);
    } else if (s.tp == 128) {
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 128, 32, 4, 1>), grid, dim3(256), 0, st, a);
    } else if (s.tq == 128) {
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 32, 128, 1, 4>), grid, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((product_kernel<T, PA, QA, 32, 32, 2, 2>), grid, dim3(256), 0, st, a);
    }
    if (s.parts > 1) {
        const long long finish = s.shared * (s.tp * s.tq / 1024);
        hipLaunchKernelGGL(product_finish_kernel<T>, dim3((unsigned)finish), dim3(256), 0, st, partial, s.parts, s.full,
                           s.tiles_p, s.tp, s.tq, a.nq, a.epi);
    }
    return ngs_decoder_launched("ngs_linear");
}


// Backward workspace: dz (when there is an activation), the column sums' partials, the cut products' partials (the
// two products run one after the other and share them).
struct BackwardPlan {
    int across;
    long long col_blocks, row_blocks;
    long long ldz;                       // elements between the rows of dz: n, or n in whole chunks
    bool copy_dz, pad_w, pad_x;          // dz is made although it is dL_dy; weight and x are padded
    size_t sums_at, partial_at, weight_at, x_at, total;
};

static BackwardPlan backward_plan(long long rows, int k, int n, int dtype, int act)
{
    BackwardPlan b;
    const long long size = (long long)ngs_decoder_size(dtype), chunk = 16 / size;
    const long long chunks = (n + chunk - 1) / chunk;
    b.across = 1;
    while (b.across < 64 && b.across < chunks) b.across *= 2;
    b.col_blocks = (chunks + b.across - 1) / b.across;
    const long long high = 256 / b.across;
    b.row_blocks = 2048 / (b.col_blocks > 0 ? b.col_blocks : 1);
    if (b.row_blocks > (rows + 4 * high - 1) / (4 * high)) b.row_blocks = (rows + 4 * high - 1) / (4 * high);
    if (b.row_blocks < 1) b.row_blocks = 1;
    const bool pad_z = pads(n, k, rows, n, dtype) || pads(n, k, n, rows, dtype);
    b.ldz = pad_z ? whole_chunks(n, dtype) : n;
    b.copy_dz = pad_z;
    b.pad_w = pads(k, k, rows, n, dtype);
    b.pad_x = pads(k, k, n, rows, dtype);
    b.sums_at = act == NGS_ACT_NONE && !pad_z ? 0 : align256((size_t)rows * b.ldz * size);
    b.partial_at = b.sums_at + align256((size_t)b.row_blocks * n * 4);
    const size_t p1 = partial_bytes(k, rows, n, dtype), p2 = partial_bytes(k, n, rows, dtype);
    b.weight_at = b.partial_at + align256(p1 > p2 ? p1 : p2);
    b.x_at = b.weight_at + (b.pad_w ? align256((size_t)n * whole_chunks(k, dtype) * size) : 0);
    b.total = b.x_at + (b.pad_x ? align256((size_t)rows * whole_chunks(k, dtype) * size) : 0) + 256;
    return b;
}

template <typename T>
static int linear_forward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const void* x, long long ldx,
                          const void* w, long long ldw, const void* bias, const void* res, long long ldr, void* y,
                          float* slope, char* workspace)
{
    Product<T> a = {};
    a.p = (const T*)w;
    a.q = (const T*)x;
    a.ldp = ldw;
    a.ldq = ldx;
    a.np = n;
    a.nq = rows;
    a.nr = a.along = k;
    a.epi.act = act;
    a.epi.bias = (const T*)bias;
    a.epi.residual = (const T*)res;
    a.epi.ldr = ldr;
    a.epi.y = (T*)y;
    a.epi.slope = act == NGS_ACT_NONE ? nullptr : slope;
    a.epi.np = n;
    if (ngs_few_rows_takes(rows, k, n, dtype)) return ngs_few_rows<T>(st, rows, k, n, a.q, ldx, a.p, ldw, a.epi);
    if (ngs_stream_forward_takes(rows, k, n, dtype))
        return ngs_stream_forward<T>(st, rows, k, n, dtype, a.q, ldx, a.p, ldw, a.epi);
    a.width_p = n;
    a.width_q = rows;
    if (pads(k, n, rows, k, dtype)) {
        const long long wide = whole_chunks(k, dtype);
        T* const wp = (T*)(workspace + align256(partial_bytes(n, rows, k, dtype)));
        T* const xp = wp + (size_t)n * wide;
        pad_rows(st, a.p, ldw, n, k, wp, a.q, ldx, rows);
        a.p = wp;
        a.q = xp;
        a.ldp = a.ldq = a.along = wide;
    }
    return launch_product<T, false, false>(st, dtype, a, (float*)workspace);
}

template <typename T>
static int linear_backward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const void* x, long long ldx,
                           const void* w, long long ldw, const void* bias, const float* slope, const void* dy, long long lddy,
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
    const bool make_dz = (act != NGS_ACT_NONE || b.copy_dz) && (dx || dw) && rows > 0 && n > 0;
    if (make_dz || db) {
        const dim3 grid((unsigned)b.row_blocks, (unsigned)b.col_blocks);
        hipLaunchKernelGGL(linear_dz_kernel<T>, grid, dim3(256), 0, st, rows, n, b.across, (const T*)dy, lddy,
                           act == NGS_ACT_NONE ? nullptr : slope,
                           make_dz ? (T*)workspace : nullptr, b.ldz, db ? sums : nullptr);
        if (db) ngs_launch_column_finish(st, sums, b.row_blocks, n, 0, db, nullptr, dtype);
        if (ngs_decoder_launched("ngs_linear_backward")) return 1;
        if (make_dz) {
            dz = (const T*)workspace;
            lddz = b.ldz;
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
        a.along = make_dz ? b.ldz : n;
        a.width_p = k;
        a.width_q = rows;
        if (b.pad_w) {
            pad_rows(st, a.p, ldw, n, k, (T*)(workspace + b.weight_at));
            a.p = (const T*)(workspace + b.weight_at);
            a.ldp = a.width_p = whole_chunks(k, dtype);
        }
        a.epi.y = (T*)dx;
        if (launch_product<T, true, false>(st, dtype, a, partial)) return 1;
    }
    if (dw) {
        Product<T> a = {};
        a.p = (const T*)x;
        a.q = dz;
        a.ldp = ldx;
        a.ldq = lddz;
        a.np = k;
        a.nq = n;
        a.nr = a.along = rows;
        a.width_p = k;
        a.width_q = make_dz ? b.ldz : n;
        if (b.pad_x) {
            pad_rows(st, a.p, ldx, rows, k, (T*)(workspace + b.x_at));
            a.p = (const T*)(workspace + b.x_at);
            a.ldp = a.width_p = whole_chunks(k, dtype);
        }
        a.epi.y = (T*)dw;
        if (launch_product<T, true, true>(st, dtype, a, partial)) return 1;
    }
    return 0;
}

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
// (byte counts of operands and workspaces stay far from 64 bits)
static bool too_many(long long rows, int k, int n)
{
    return rows > (1LL << 40) || k > NGS_WIDEST || n > NGS_WIDEST || (double)rows * (k > n ? k : n) > 281474976710656.0;
}

static int check_linear(const char* what, long long rows, int k, int n, int dtype, int act)
{
    if (rows < 0 || k < 0 || n < 0) return ngs_set_error(what, "a size is negative");
    if (too_many(rows, k, n)) return ngs_set_error(what, "too many elements for one launch");
    if (!ngs_decoder_dtype(dtype)) return ngs_set_error(what, "unknown element type");
    if (act < NGS_ACT_NONE || act > NGS_ACT_SIGMOID) return ngs_set_error(what, "unknown activation");
    return 0;
}

extern "C" size_t ngs_linear_forward_workspace_bytes(long long rows, int in_features, int out_features, int dtype)
{
    if (rows <= 0 || out_features <= 0 || in_features < 0 || too_many(rows, in_features, out_features) ||
        !ngs_decoder_dtype(dtype))
        return 0;
    if (ngs_few_rows_takes(rows, in_features, out_features, dtype) ||
        ngs_stream_forward_takes(rows, in_features, out_features, dtype))
        return 0;
    const size_t partial = partial_bytes(out_features, rows, in_features, dtype);
    if (!pads(in_features, out_features, rows, in_features, dtype)) return partial;
    return align256(partial) + (size_t)whole_chunks(in_features, dtype) * (rows + out_features) * ngs_decoder_size(dtype);
}

extern "C" int ngs_linear_forward(long long rows, int in_features, int out_features, int dtype, int activation,
                                  const void* x, long long x_stride, const void* weight, long long weight_stride,
                                  const void* bias, const void* residual, long long residual_stride, void* y,
                                  float* slope, char* workspace, void* stream)
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

extern "C" size_t ngs_linear_slope_bytes(long long rows, int in_features, int out_features, int dtype, int activation)
{
    if (rows <= 0 || in_features < 0 || out_features <= 0 || too_many(rows, in_features, out_features) ||
        !ngs_decoder_dtype(dtype) || activation == NGS_ACT_NONE)
        return 0;
    if (ngs_stream_backward_takes(rows, in_features, out_features, dtype)) return 0;
    return (size_t)rows * (size_t)out_features * sizeof(float);
}

extern "C" size_t ngs_linear_backward_workspace_bytes(long long rows, int in_features, int out_features, int dtype,
                                                      int activation)
{
    if (rows < 0 || in_features < 0 || out_features < 0 || too_many(rows, in_features, out_features) ||
        !ngs_decoder_dtype(dtype))
        return 0;
    if (ngs_stream_backward_takes(rows, in_features, out_features, dtype))
        return (size_t)ngs_stream_backward_blocks(rows, in_features, out_features, dtype) *
               ((size_t)in_features * out_features + out_features) * sizeof(float);
    return backward_plan(rows, in_features, out_features, dtype, activation).total;
}

extern "C" int ngs_linear_backward(long long rows, int in_features, int out_features, int dtype, int activation,
                                   const void* x, long long x_stride, const void* weight, long long weight_stride,
                                   const void* bias, const float* slope, const void* dL_dy, long long dL_dy_stride,
                                   void* dL_dx, void* dL_dweight, void* dL_dbias, char* workspace, void* stream)
{
    const int k = in_features, n = out_features;
    if (check_linear("ngs_linear_backward", rows, k, n, dtype, activation)) return 1;
    if (rows == 0 || k == 0) dL_dx = nullptr;   // nothing to write
    if (n == 0 || k == 0) dL_dweight = nullptr;
    if (n == 0) dL_dbias = nullptr;
    if (!dL_dx && !dL_dweight && !dL_dbias) return 0;
    if (dL_dbias && ngs_decoder_columns("ngs_linear_backward", n)) return 1;
    const bool reads_slope = ngs_linear_slope_bytes(rows, k, n, dtype, activation) > 0;
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
