// Shared by the kernels of the matrix product (linear.hip, linear_stream.hip): activations and the rest of the epilogue,
// matrix instructions on 16-byte fragments, tiles in shared memory.
#pragma once
#include "decoder_common.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define ROW_BYTES 128  // bytes of the reduction index that one step stages per row: 64 16-bit elements or 32 floats

#define NGS_FEW_ROWS 64  // rows that linear_rows.hip takes at most

// ---------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float activate_one(float z, float& slope)
{
    if (ACT == NGS_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;  // NaN stays
    }
    if (ACT == NGS_ACT_GELU) {
        // Phi(-a) = Q(a) exp(-a^2 / 2) for a = |z|: the exponential is the density's, which the derivative needs as well.
        // Q falls from 1/2 as 1 / a does: t = 1 / (1 + a / 4) times a polynomial in t, least in relative error over all a
        // (3.4e-8 before rounding, 4e-7 in 32 bits), so that Phi keeps its size in the far tail, where a sum about 1 or an
        // approximation of erf to so many decimals has none left.  (640000 x 128 -> 128 bfloat16 with residual: forward 101 us,
        // there and back 287 us; 98 and 279 us with five coefficients, which are 5e-5 off at -3.)
        const float a = fabsf(z), e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.25f * a);
        float q = 0.0197819583f;
        q = q * t - 0.080877088f;
        q = q * t + 0.095596686f;
        q = q * t - 0.0317171291f;
        q = q * t + 0.0636988878f;
        q = q * t + 0.0589752235f;
        q = q * t + 0.0816030949f;
        q = q * t + 0.0934663564f;
        q = q * t + 0.0997364298f;
        q = q * t + 0.0997355655f;
        const float tail = q * t * e;
        const float phi = z < 0.0f ? tail : 1.0f - tail;
        slope = phi + z * (0.39894228040143268f * e);
        return z * phi;
    }
    if (ACT == NGS_ACT_SILU) {
        const float s = sigmoid(z);
        slope = s * (1.0f + z * (1.0f - s));
        return z * s;
    }
    if (ACT == NGS_ACT_SIGMOID) {
        // sigmoid' = sigmoid(z) sigmoid(-z): of the difference 1 - sigmoid(z) nothing would be left where z is large
        const float t = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + t), s = t * r;
        slope = s * r;
        return z < 0.0f ? s : r;
    }
    slope = 1.0f;
    return z;
}

// act(z) of N values and its derivative (slope NULL: not wanted): one uniform branch for all of them
template <int N>
__device__ __forceinline__ void activate(int act, const float (&z)[N], float (&y)[N], float* slope)
{
    switch (act) {
#define NGS_ACTIVATE(A)                                                \
    case A:                                                            \
        for (int i = 0; i < N; i++) {                                  \
            float s;                                                   \
            y[i] = activate_one<A>(z[i], s);                           \
            if (slope) slope[i] = s;                                   \
        }                                                              \
        break;
        NGS_ACTIVATE(NGS_ACT_RELU)
        NGS_ACTIVATE(NGS_ACT_GELU)
        NGS_ACTIVATE(NGS_ACT_SILU)
        NGS_ACTIVATE(NGS_ACT_SIGMOID)
#undef NGS_ACTIVATE
    default:
        for (int i = 0; i < N; i++) {
            y[i] = z[i];
            if (slope) slope[i] = 1.0f;
        }
    }
}

// ---------------------------------------------------------------------------
// What happens to four neighbouring sums of one result row
// ---------------------------------------------------------------------------
template <typename T>
struct Epilogue {
    int act;
    int np;               // width of a result row
    const T* bias;        // [np] or NULL
    const T* residual;    // rows ldr apart, or NULL
    long long ldr;
    T* y;                 // [nq][np]
    // The activation's derivative [nq][np], or NULL.  In 32 bits whatever T: a saturated unit's derivative is far below
    // what half precision holds (sigmoid' is 2e-9 at 20), and its gradient may not depend on the kernel that a width selects.
    float* slope;
};

template <typename U>
__device__ __forceinline__ void store4(U* p, const float (&v)[4], int valid)
{
    union { U e[4]; } u;
#pragma unroll
    for (int i = 0; i < 4; i++) u.e[i] = (U)v[i];
    if (valid >= 4) {
        __builtin_memcpy(p, u.e, 4 * sizeof(U));
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (i < valid) p[i] = u.e[i];
    }
}

template <typename U>
__device__ __forceinline__ void load4(const U* p, float (&v)[4], int valid)
{
    union { U e[4]; } u = {};
    if (valid >= 4) {
        __builtin_memcpy(u.e, p, 4 * sizeof(U));
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (i < valid) u.e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (float)u.e[i];
}

template <typename T>
__device__ __forceinline__ void finish4(const Epilogue<T>& e, long long q, int p, f32x4 z, const float (&bias)[4])
{
    const int valid = e.np - p;
    const long long at = q * e.np + p;
    float v[4], y[4], s[4], r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e.residual) load4(e.residual + q * e.ldr + p, r, valid);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = z[i] + bias[i];
    if (e.slope) activate<4>(e.act, v, y, s);
    else activate<4>(e.act, v, y, nullptr);
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] += r[i];
    store4(e.y + at, y, valid);
    if (e.slope) store4(e.slope + at, s, valid);
}

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, const bf16*)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, const f16*)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, const float*)
{
#pragma unroll
    for (int j = 0; j < 4; j++)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
}

// One operand's tile of ROWS rows in shared memory, ROWS * ROW_BYTES bytes either way.
//
// Along: row after row, the eight 16-byte chunks of a row exchanged by the row's low bits, so that the 16 rows a
// fragment is read from spread over the banks.  Lane (g, i) = (lane / 16, lane % 16) of a fragment holds row i,
// chunk g of a group of four: 8 16-bit elements or 4 floats of the reduction.
//
// Across: one line of ROWS elements per reduction index.  A fragment needs, per lane, one column and neighbouring
// reduction indices: 16-bit elements come through the transposing read (four lines of 16 columns per 16 lanes, two
// reads a fragment), floats one by one.  The 16 columns' segment within the line is exchanged by the line's number,
// so that the lines that are read together lie in different banks.
template <typename T, bool ACROSS, int ROWS>
struct Tile {
    static constexpr int N = Chunk<T>::N;
    static constexpr int STEP = ROW_BYTES / (int)sizeof(T);        // reduction elements of a step
    static constexpr int CHUNKS = ROWS * (ROW_BYTES / 16);
    static constexpr int LINE = ROWS * (int)sizeof(T) / 16;        // across: chunks of a line
    static constexpr int SEG = (int)sizeof(T);                     // across: chunks of 16 columns (2 or 4)

    static __device__ __forceinline__ int segment_swap(int line)
    {
        const int s = sizeof(T) == 2 ? (line & 3) | ((line >> 1) & 4) : (line >> 2) & 3;
        return s & (LINE / SEG - 1);
    }

    // the 16 bytes that chunk number i of the tile holds, from memory
    static __device__ __forceinline__ u32x4 fetch(const T* __restrict__ base, long long ld, long long row0,
                                                  long long rows, long long r0, long long r_end, int i)
    {
        if (!ACROSS) {
            const long long row = row0 + i / 8, r = r0 + (i % 8) * N;
            if (row >= rows) return (u32x4){0, 0, 0, 0};
            return load16_head(base + row * ld + r, r_end - r);
        } else {
            const long long r = r0 + i / LINE, col = row0 + (i % LINE) * N;
            if (r >= r_end) return (u32x4){0, 0, 0, 0};
            return load16_head(base + r * ld + col, rows - col);
        }
    }
    static __device__ __forceinline__ void put(char* lds, int i, u32x4 v)
    {
        int at;
        if (!ACROSS) {
            const int row = i / 8, c = i % 8;
            at = row * ROW_BYTES + ((c ^ (row & 7)) << 4);
        } else {
            const int line = i / LINE, c = i % LINE;
            at = line * (LINE << 4) + ((c ^ (segment_swap(line) * SEG)) << 4);
        }
        *(u32x4*)(lds + at) = v;
    }
    // fragment of rows [16 block, 16 block + 16), half `s` of the step's reduction elements
    static __device__ __forceinline__ u32x4 fragment(const char* lds, int block, int s, int lane)
    {
        const int g = lane >> 4, i = lane & 15;
        if (!ACROSS) {
            const int row = block * 16 + i, c = s * 4 + g;
            return *(const u32x4*)(lds + row * ROW_BYTES + ((c ^ (row & 7)) << 4));
        } else if (sizeof(T) == 2) {
            const int line = s * 32 + g * 8 + (i >> 2);
            const int seg = block ^ segment_swap(line);  // the same for line and line + 4
            const char* at = lds + line * (LINE << 4) + (seg << 5) + ((i & 3) << 3);
            typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * (LINE << 4)));
            const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
            return (u32x4){l.x, l.y, h.x, h.y};
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int line = s * 16 + g * 4 + j;
                const int seg = block ^ segment_swap(line);
                v[j] = *(const uint32_t*)(lds + line * (LINE << 4) + (seg << 6) + (i << 2));
            }
            return v;
        }
    }
};


// linear_stream.hip: the product over many narrow rows, and whether a size is its business
bool ngs_stream_forward_takes(long long rows, int k, int n, int dtype);
template <typename T>
int ngs_stream_forward(hipStream_t st, long long rows, int k, int n, int dtype, const T* x, long long ldx, const T* w,
                       long long ldw, const Epilogue<T>& e);
bool ngs_stream_backward_takes(long long rows, int k, int n, int dtype);
long long ngs_stream_backward_blocks(long long rows, int k, int n, int dtype);
template <typename T>
int ngs_stream_backward(hipStream_t st, long long rows, int k, int n, int dtype, int act, const T* x, long long ldx,
                        const T* w, long long ldw, const T* bias, const T* dy, long long lddy, T* dx, T* dw, T* db,
                        float* partial);

// linear_rows.hip: the product for a few rows
bool ngs_few_rows_takes(long long rows, int k, int n, int dtype);
template <typename T>
int ngs_few_rows(hipStream_t st, long long rows, int k, int n, const T* x, long long ldx, const T* w, long long ldw,
                 const Epilogue<T>& e);
