// Shared by the operators over feature rows (linear.hip, layer_norm.hip, dropout.hip): element types, 16-byte accesses
// that need no alignment, launch checks, and the reduction of per-workgroup partial sums of columns.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../../include/ngs_rasterizer.h"

// Nothing in these kernels has to match another evaluation bit for bit: products and sums may contract.
#pragma clang fp contract(fast)

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

int ngs_set_error(const char* what, const char* detail);  // capi.hip: keeps the message, returns 1

#define NGS_CUS 256     // compute units of the MI355X: what launch shapes are chosen for
#define NGS_XCDS 8      // its dies; workgroups go to them in turn

// Elements of T in 16 bytes.
template <typename T> struct Chunk { static constexpr int N = 16 / (int)sizeof(T); };

// 16 bytes as N elements, wide loads and stores at any alignment the type allows (the hardware takes unaligned
// global accesses; one that straddles a cache line costs a second line, elements one by one cost N requests).
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p)
{
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// The same for 16-bit elements that may start in the middle of a word: the words they lie in, shifted into place.  A
// 16-byte load that is not on a word's boundary takes the address unit several times as long (64 x 3711 -> 1000 bfloat16:
// 58 us, against 20 us with 3710 or 3712 columns).  Every word that is read holds an element that was asked for.
template <typename T>
__device__ __forceinline__ u32x4 load16_any(const T* p)
{
    if constexpr (sizeof(T) != 2) return load16(p);
    const uint32_t odd = ((uintptr_t)p >> 1) & 1;
    const uint32_t* const words = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
    u32x4 v;
    __builtin_memcpy(&v, words, 16);
    const uint32_t last = words[3 + odd], s = odd * 16;
    return (u32x4){__builtin_amdgcn_alignbit(v.y, v.x, s), __builtin_amdgcn_alignbit(v.z, v.y, s),
                   __builtin_amdgcn_alignbit(v.w, v.z, s), __builtin_amdgcn_alignbit(last, v.w, s)};
}

// The first `valid` of the N elements at p (all, if that many or more; none, if <= 0), zeros behind them.
template <typename T>
__device__ __forceinline__ u32x4 load16_head(const T* p, long long valid)
{
    constexpr int N = Chunk<T>::N;
    if (valid >= N) return load16(p);
    union { u32x4 v; T e[N]; } u;
    u.v = (u32x4){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N - 1; i++)
        if (i < valid) u.e[i] = p[i];
    return u.v;
}

template <typename T>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[Chunk<T>::N])
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) f[i] = (float)u.e[i];
}

// Values rounded to nearest, ties to even.
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&f)[Chunk<T>::N])
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) u.e[i] = (T)f[i];
    return u.v;
}

template <typename T>
__device__ __forceinline__ void store16_head(T* p, u32x4 v, long long valid)
{
    constexpr int N = Chunk<T>::N;
    if (valid >= N) {
        __builtin_memcpy(p, &v, 16);
        return;
    }
    union { u32x4 v; T e[N]; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < N - 1; i++)
        if (i < valid) p[i] = u.e[i];
}

inline int ngs_decoder_launched(const char* what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : ngs_set_error(what, hipGetErrorString(e));
}

#define NGS_WIDEST (1 << 30)  // columns of a row at most: kernels count them, a tile past the end, in 32 bits

// A launch has fewer than 2^32 threads along x.
inline int ngs_decoder_grid(const char* what, long long groups, int threads)
{
    return groups > 0xffffffffLL / threads ? ngs_set_error(what, "too many elements for one launch") : 0;
}

inline bool ngs_decoder_dtype(int t) { return t == NGS_FLOAT32 || t == NGS_FLOAT16 || t == NGS_BFLOAT16; }
inline size_t ngs_decoder_size(int t) { return t == NGS_FLOAT32 ? 4 : 2; }

// Whether a 2-D operand of `rows` rows of `width` elements, `stride` apart, is there and can be addressed.  Byte
// offsets inside a tile are formed in 64 bits; the bound keeps the whole extent in range as well.
inline int ngs_decoder_operand(const char* what, const void* p, long long rows, long long width, long long stride)
{
    if (rows <= 0 || width <= 0) return 0;
    if (!p) return ngs_set_error(what, "is NULL");
    if (stride < 0) return ngs_set_error(what, "has a negative row stride");
    if (stride > 0 && rows > (1LL << 58) / stride) return ngs_set_error(what, "spans too many elements");
    return 0;
}

// Joins workgroups' sums of columns, always in the same order: out[c] = sum over b of partial[b][c], rows width0 + width1
// long, the first width0 columns going to out0, the others to out1.  A NULL output is left out.  No rows: zeros.
void ngs_launch_column_finish(hipStream_t s, const float* partial, long long blocks, long long width0, long long width1,
                              void* out0, void* out1, int dtype);
// That launch takes 1024 threads for 64 columns: more than it holds are refused before anything else is launched.
inline int ngs_decoder_columns(const char* what, long long columns) { return ngs_decoder_grid(what, (columns + 63) / 64, 1024); }
