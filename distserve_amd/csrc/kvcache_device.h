// kvcache_device.h -- what the cache operators' kernels share: element types, e4m3 codes, division
// by a number the host knows, and the attention kernels' arguments.
#ifndef KVCACHE_DEVICE_H
#define KVCACHE_DEVICE_H

#include "kvcache_plan.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

namespace kvc {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- element types

template <typename T> struct Elem;
template <> struct Elem<_Float16> {
    typedef f16x4 V4;
    typedef f16x8 Frag;     // 16 bytes: an operand of a matrix instruction
    static constexpr uint32_t kExponent = 0x7c007c00u;
};
template <> struct Elem<__bf16> {
    typedef bf16x4 V4;
    typedef bf16x8 Frag;
    static constexpr uint32_t kExponent = 0x7f807f80u;
};
template <> struct Elem<float> {
    typedef f32x4 V4;
    typedef f32x4 Frag;
    static constexpr uint32_t kExponent = 0x7f800000u;
};

// Whether one of the word's elements is an infinity or a NaN (its exponent is all ones).
template <typename T> __device__ inline bool not_finite(uint32_t w)
{
    constexpr uint32_t m = Elem<T>::kExponent;
    if constexpr (sizeof(T) == 4) return (w & m) == m;
    // 16-bit types: one more in the exponent's lowest place carries into the sign's
    constexpr uint32_t one = std::is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u;
    return (((w & 0x7fff7fffu) + one) & 0x80008000u) != 0;
}

// ---- e4m3 codes with a power-of-two scale for each row

__device__ inline float power_of(uint32_t byte) { return __uint_as_float(byte << 23); }   // 2^(byte-127), byte >= 1

// Four codes as T, times the row's scale: exact (four significant bits), but for fp16's range, which `saturated` sees to.
template <typename T> __device__ inline void decode4(uint32_t codes, float scale, uint32_t out[])
{
    if constexpr (std::is_same<T, _Float16>::value) {
        union { f16x2 h; uint32_t w; } a, b;
        a.h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false);
        b.h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true);
        out[0] = a.w;
        out[1] = b.w;
    } else if constexpr (std::is_same<T, __bf16>::value) {
        union { bf16x2 h; uint32_t w; } a, b;
        a.h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false);
        b.h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true);
        out[0] = a.w;
        out[1] = b.w;
    } else {
        union { f32x2 f; uint32_t w[2]; } a, b;
        a.f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, false);
        b.f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, true);
        out[0] = a.w[0];
        out[1] = a.w[1];
        out[2] = b.w[0];
        out[3] = b.w[1];
    }
}

// Whether codes under this scale may be past the largest fp16 number (448 * 2^7 is not).
template <typename T> __device__ inline bool may_overflow(float scale) { return std::is_same<T, _Float16>::value && scale >= 256.0f; }

// A code may have rounded past the largest fp16 number, which it then becomes.
__device__ inline uint32_t saturated(uint32_t w)
{
    if ((w & 0x7fffu) == 0x7c00u) w -= 1;
    if ((w & 0x7fff0000u) == 0x7c000000u) w -= 0x10000u;
    return w;
}

// An output row's numbers in T's range.  A mean of fp16 numbers is in it, but weights that were rounded to fp16 for the product
// (2^-11 of each at most) may carry it past the largest one, and from 2^-12 past it on it would round to an infinity: it is
// the largest number then.  What V's infinities and NaN have made stays.
template <typename T> __device__ inline float in_range(float x)
{
    if constexpr (std::is_same<T, _Float16>::value) return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    return x;
}
template <typename T> __device__ inline typename Elem<T>::V4 output4(f32x4 x)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = in_range<T>(x[i]);
    return __builtin_convertvector(x, typename Elem<T>::V4);
}

// Two elements of T in a word (one of float) as floats.
template <typename T> __device__ inline float element(const uint32_t *w, int i)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const uint32_t half = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(half << 16);
    union { uint16_t u; _Float16 h; } c;
    c.u = (uint16_t)half;
    return (float)c.h;
}

// ---- division by a number the host knows: n / d for n < 2^31 (the multiplier has 32 bits)

struct Divider {
    uint32_t magic, shift;
};

__host__ inline Divider divider(uint32_t d)
{
    uint32_t bits = 0;
    while ((1ull << bits) < d) ++bits;
    return Divider{(uint32_t)(((1ull << (31 + bits)) + d - 1) / d), 31 + bits};
}

__device__ inline uint32_t div_by(uint32_t n, Divider d) { return (uint32_t)(((uint64_t)n * d.magic) >> d.shift); }

// ---- the attention kernels' arguments

struct AttnArgs {
    const KvTile *tiles;                      // few rows
    const KvStart *starts;
    const KvItem *items;                      // many rows
    const int32_t *table;
    const char *q;
    char *out;
    const char *k, *v;                        // the pools at the layer, or the packed rows
    uint64_t q_token, q_head, out_token, out_head;   // bytes
    uint64_t k_block, k_head, v_block, v_head;       // bytes: block (or token) and head strides
    uint32_t row_bytes, codes;                // of a token in the pool; B * D
    uint32_t block_size, heads, group, head_dim;   // heads: KV heads
    Divider by_block, by_heads, by_group;
    float scale_log2;                         // |scale| * log2(e): the softmax is taken in powers of two
    uint32_t q_sign;                          // sign bits of q to turn over (a negative scale)
    float *part_acc, *part_ml;                // partial rows: [row][head_dim], and {maximum, sum}
    uint32_t part_starts, part_pitch;         // few rows: workgroup w's partial rows for a pair it starts (begins anew) with are at
                                              // w * part_pitch, for one it leaves unfinished at part_starts + w * part_pitch
    uint32_t part_items, part_head;           // many rows: KV head h's partial rows start at part_items + h * part_head
};

// Rows row0 .. of a sequence for one KV head over keys [kv_begin, kv_end).
struct RowWork {
    int q_start, rows, first, table_at, row0;   // as in KvTile
    int head;
    int kv_begin, kv_end;
    int64_t part_row;                           // partial rows start here; -1: these are all of the rows' keys
};

enum { kPlain = 0, kE4m3 = 1, kPacked = 2 };

// A structure of words that is the same for the whole wave, in scalar registers.
template <typename S> __device__ inline S uniform(const S *p)
{
    union { S s; int w[sizeof(S) / 4]; } u;
    u.s = *p;
#pragma unroll
    for (unsigned i = 0; i < sizeof(S) / 4; ++i) u.w[i] = __builtin_amdgcn_readfirstlane(u.w[i]);
    return u.s;
}

template <typename V> __device__ inline V as(u32x4 w)
{
    union { u32x4 w; V v; } c;
    c.w = w;
    return c.v;
}

// 2^x
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace kvc

#endif  // KVCACHE_DEVICE_H
