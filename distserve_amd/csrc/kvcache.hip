// kvcache.hip -- the cache operators for MI355X (gfx950, wave64): new tokens' K and V into the
// paged pools (plain or as e4m3 codes), the pools read back, and attention over them.
//
// A step plan (kvcache_plan.cpp) says which cache slot each new token has and which pieces the
// attention is cut into; the kernels find everything else from it.  Reference call site of
// what these operators do: distserve/worker.py:211-227 (the model forward gets the pools and
// the block table).
#include "kv_internal.h"
#include "kvcache_plan.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

namespace {

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
    return (w & m & 0xffffu) == (m & 0xffffu) || (w & m & 0xffff0000u) == (m & 0xffff0000u);
}

// ---- e4m3 codes with a power-of-two scale for each row

__device__ inline float power_of(uint32_t byte) { return __uint_as_float(byte << 23); }   // 2^(byte-127), byte >= 1

// Four codes as T, times the row's scale: exact (four significant bits), except that a code may
// have rounded past the largest fp16 number, which it then becomes (byte >= 135 only: 448 * 2^7
// still fits).
template <typename T> __device__ inline void decode4(uint32_t codes, float scale, uint32_t out[])
{
    if constexpr (std::is_same<T, _Float16>::value) {
        union { f16x2 h; uint32_t w; } a, b;
        a.h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false);
        b.h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true);
        if (scale >= 256.0f) {
            for (uint32_t *w : {&a.w, &b.w}) {
                if ((*w & 0x7fffu) == 0x7c00u) *w -= 1;
                if ((*w & 0x7fff0000u) == 0x7c000000u) *w -= 0x10000u;
            }
        }
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

// ---- write and read back
//
// Pure data movement: a lane takes eight elements of a row, 8, 16 or 32 lanes a row (the power of two
// that covers head_dim; lanes past it idle).  Both are bound by HBM.

struct MoveArgs {
    const int32_t *slots;       // write: the new tokens' cache slots; read: {first output row, tokens} of each table entry
    const int32_t *table;       // read: the block table
    const char *src_k, *src_v;  // write: rows; read: the pools (at the layer)
    char *dst_k, *dst_v;
    uint64_t block_stride, head_stride;           // bytes, in the pool
    uint64_t k_token, k_head, v_token, v_head;    // bytes, of the rows
    uint32_t row_bytes;         // of a token in the pool
    uint32_t codes;             // B * D: where a quantised slab's scales start
    uint32_t tokens, heads, head_dim, block_size;
    Divider by_heads, by_block;
};

// T: the rows' type.  Q: quantised pool.  LANES: lanes of a row.
template <typename T, bool Q, int LANES>
__global__ __launch_bounds__(256) void kvm_write_kernel(const MoveArgs a)
{
    constexpr int W = sizeof(T) * 2;                                   // words of a lane's eight elements
    const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= a.tokens * a.heads) return;                             // a row's lanes leave together
    const uint32_t token = div_by(row, a.by_heads), head = row - token * a.heads;
    const bool is_v = blockIdx.y != 0;
    const uint32_t d = threadIdx.x % LANES * 8;
    const bool live = d < a.head_dim;
    const char *src = (is_v ? a.src_v + token * a.v_token + head * a.v_head : a.src_k + token * a.k_token + head * a.k_head)
                      + d * sizeof(T);
    uint32_t w[W] = {};
    if (live) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) *(u32x4 *)(w + 4 * i) = __builtin_nontemporal_load((const u32x4 *)src + i);
    }
    const uint32_t slot = (uint32_t)a.slots[token], block = div_by(slot, a.by_block), off = slot - block * a.block_size;
    char *slab = (is_v ? a.dst_v : a.dst_k) + block * a.block_stride + head * a.head_stride;
    if constexpr (!Q) {
        if (live) {
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
                *((u32x4 *)(slab + off * a.row_bytes + d * sizeof(T)) + i) = *(u32x4 *)(w + 4 * i);
        }
    } else {
        float x[8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = element<T>(w, i);
            top = fmaxf(top, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
        }
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
        // smallest e with top <= 448 * 2^e; 448 = 0.875 * 2^9
        int e = 0;
        if (top > 0.0f) {
            int x2;
            const float part = frexpf(top, &x2);
            e = max(part <= 0.875f ? x2 - 9 : x2 - 8, -126);
        }
        const float inverse = power_of((uint32_t)(127 - e));          // e <= 120, so this is a normal number
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x[i] * inverse;
            x[i] = y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f);
        }
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], p, true);
        }
        if (live) *(u32x2 *)(slab + off * a.row_bytes + d) = u32x2{c[0], c[1]};
        if (d == 0) *(uint8_t *)(slab + a.codes + off) = (uint8_t)(e + 127);
    }
}

// One workgroup for each (table entry, eight tokens or so, KV head): the block's tokens to their packed rows.
template <typename T, bool Q, int LANES>
__global__ __launch_bounds__(256) void kvm_read_kernel(const MoveArgs a)
{
    constexpr int W = sizeof(T) * 2;
    const uint32_t page = div_by(blockIdx.x, a.by_heads), head = blockIdx.x - page * a.heads;
    const int32_t first = a.slots[2 * page], count = a.slots[2 * page + 1], block = a.table[page];
    const bool is_v = blockIdx.y != 0;
    const uint32_t d = threadIdx.x % LANES * 8;
    if (d >= a.head_dim) return;
    const char *slab = (is_v ? a.src_v : a.src_k) + (uint64_t)block * a.block_stride + head * a.head_stride;
    char *out = (is_v ? a.dst_v : a.dst_k) + head * a.k_head + d * sizeof(T);
    for (int32_t t = threadIdx.x / LANES; t < count; t += 256 / LANES) {
        uint32_t w[W];
        if constexpr (Q) {
            const u32x2 c = *(const u32x2 *)(slab + (uint64_t)t * a.row_bytes + d);
            const float scale = power_of(*(const uint8_t *)(slab + a.codes + t));
            decode4<T>(c[0], scale, w);
            decode4<T>(c[1], scale, w + W / 2);
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
                *(u32x4 *)(w + 4 * i) = *((const u32x4 *)(slab + (uint64_t)t * a.row_bytes + d * sizeof(T)) + i);
        }
#pragma unroll
        for (int i = 0; i < W / 4; ++i)
            __builtin_nontemporal_store(*(u32x4 *)(w + 4 * i), (u32x4 *)(out + (uint64_t)(first + t) * a.k_token) + i);
    }
}

// ---- attention

struct AttnArgs {
    const KvItem *items;
    const int32_t *table;
    const char *q;
    char *out;
    const char *k, *v;                        // the pools at the layer, or the packed rows
    uint64_t q_token, q_head, out_token, out_head;   // bytes
    uint64_t k_block, k_head, v_block, v_head;       // bytes: block (or token) and head strides
    uint32_t row_bytes, codes;                // of a token in the pool; B * D
    uint32_t block_size, heads, group, head_dim;   // heads: KV heads
    Divider by_block, by_heads, by_group;
    float scale_log2;                         // scale * log2(e): the softmax is taken in powers of two
    float *part_acc, *part_ml;                // partial rows: [row][kv head][head_dim], and {maximum, sum}
};

enum { kPlain = 0, kE4m3 = 1, kPacked = 2 };

// Matrix product step of 16x16 tiles: C[m][n] += sum_k A[m][k] B[k][n].  Lane l holds A[l%16][..] and
// B[..][l%16] of the k slots of its quarter l/16 (8 consecutive ones of 32 for 16-bit types, 1 of 4 for
// float), and C[4*(l/16)+i][l%16], i = 0..3.
__device__ inline f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mma(f32x4 a, f32x4 b, f32x4 c)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

template <typename V> __device__ inline V as(u32x4 w)
{
    union { u32x4 w; V v; } c;
    c.w = w;
    return c.v;
}

// 2^x
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// maximum and sum over the four lanes of a query row (l%16)
__device__ inline float max_quarters(float x)
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float sum_quarters(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Row kernel: a workgroup takes RT*16 query rows (tokens x the group's heads) of one KV head over the
// keys of its item; its four waves take tiles of TK keys in turn, each on its own, and their
// maxima, sums and accumulators are joined at the end (all in 32 bits).
//
// S^T = K Q^T puts a query row in a lane column, so that the softmax over keys runs over a lane's own
// registers and three other lanes, and P^T comes out just as the second product O^T = V^T P^T wants
// it: the k slots of its B operand are the rows of C, and which key a slot stands for does not
// matter as long as V^T has the same order.  K goes from memory straight into A operands (16
// contiguous bytes a lane; Q is loaded in the same order of head_dim).  V^T has to be transposed:
// through a tile in LDS of the wave's own, with the transposing LDS read (16-bit types) or element
// reads (float).
//
// LDS pitch: 32 bytes more than a row, so that the four rows of a transposing read and the
// eight rows of a write fall into different banks.
template <typename T, int SRC, int DP, int RT> struct RowShape {
    static constexpr int kSub = sizeof(T) == 4 ? 1 : 2;           // 16-key subtiles of a tile: one k step of the second product
    static constexpr int TK = 16 * kSub;
    static constexpr int kPitch = DP * (int)sizeof(T) + (sizeof(T) == 4 ? 16 : 32);
    static constexpr int kTileBytes = TK * kPitch;
    static constexpr int kJoinPitch = DP + 4;                     // floats
    static constexpr int kJoinBytes = RT * 16 * kJoinPitch * 4 + 4 * RT * 16 * 8;
    static constexpr int kLds = 4 * kTileBytes > kJoinBytes ? 4 * kTileBytes : kJoinBytes;
};

template <typename T, int SRC, int DP, int RT>
__global__ __launch_bounds__(256) void kvm_rows_kernel(const AttnArgs a)
{
    typedef RowShape<T, SRC, DP, RT> S;
    typedef typename Elem<T>::Frag Frag;
    constexpr int EF = 16 / (int)sizeof(T);                       // elements of a fragment
    constexpr int U = SRC == kE4m3 ? 16 : EF;                     // elements of a 16-byte load
    constexpr int NL = DP / (4 * U);                              // loads of a row for a lane
    constexpr int FL = U / EF;                                    // fragments of a load
    constexpr int TK = S::TK, KS = S::kSub;
    constexpr int DT = DP / 16;                                   // 16-wide tiles of head_dim in the output
    __shared__ __attribute__((aligned(16))) char lds[S::kLds];

    const uint32_t item_id = div_by(blockIdx.x, a.by_heads), h = blockIdx.x - item_id * a.heads;
    const KvItem it = a.items[item_id];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quarter = lane >> 4;
    const int D = (int)a.head_dim;
    char *tile = lds + wave * S::kTileBytes;

    // the query rows, and the last key each may see
    Frag q[RT][NL * FL];
    int limit[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = it.row0 + rt * 16 + col;
        const int clamped = min(r, it.rows - 1);
        const uint32_t token = div_by((uint32_t)clamped, a.by_group), g = (uint32_t)clamped - token * a.group;
        limit[rt] = min(it.first + (int)token, it.kv_end - 1);
        const char *src = a.q + (uint64_t)(it.q_start + token) * a.q_token + (uint64_t)(h * a.group + g) * a.q_head;
#pragma unroll
        for (int j = 0; j < NL; ++j)
#pragma unroll
            for (int f = 0; f < FL; ++f) {
                const int d = (4 * j + quarter) * U + f * EF;
                u32x4 w = {0, 0, 0, 0};
                if (r < it.rows && d < D) w = *(const u32x4 *)(src + d * sizeof(T));
                q[rt][j * FL + f] = as<Frag>(w);
            }
    }
    // the rows see different last keys from this one on
    const int diagonal = it.first + (int)div_by((uint32_t)it.row0, a.by_group);

    f32x4 acc[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4{0, 0, 0, 0};
    }

    u32x4 kw[KS][NL], vw[KS][NL];
    float kscale[KS], vscale[KS];
    auto load = [&](int base) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int key = base + s * 16 + col, safe = min(key, it.kv_end - 1);
            const char *kp, *vp;
            if constexpr (SRC == kPacked) {
                kp = a.k + (uint64_t)(it.q_start + safe) * a.k_block + h * a.k_head;
                vp = a.v + (uint64_t)(it.q_start + safe) * a.v_block + h * a.v_head;
            } else {
                const uint32_t page = div_by((uint32_t)safe, a.by_block), off = (uint32_t)safe - page * a.block_size;
                const uint64_t slab = (uint64_t)(uint32_t)a.table[it.table_at + page] * a.k_block + h * a.k_head;
                kp = a.k + slab + off * a.row_bytes;
                vp = a.v + slab + off * a.row_bytes;
                if constexpr (SRC == kE4m3) {
                    kscale[s] = power_of(*(const uint8_t *)(a.k + slab + a.codes + off));
                    vscale[s] = power_of(*(const uint8_t *)(a.v + slab + a.codes + off));
                }
            }
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int d = (4 * j + quarter) * U;
                kw[s][j] = vw[s][j] = u32x4{0, 0, 0, 0};
                if (d < D) {
                    kw[s][j] = *(const u32x4 *)(kp + d * (16 / U));
                    if (key < it.kv_end) vw[s][j] = *(const u32x4 *)(vp + d * (16 / U));   // a weight of zero must not meet a NaN
                }
            }
        }
    };
    // fragment f of a loaded 16 bytes
    auto fragment = [&](u32x4 w, int f, float scale) {
        if constexpr (SRC != kE4m3) return w;
        u32x4 o;
        if constexpr (sizeof(T) == 2) {
            uint32_t t[4];
            decode4<T>(w[2 * f], scale, t);
            decode4<T>(w[2 * f + 1], scale, t + 2);
            o = u32x4{t[0], t[1], t[2], t[3]};
        } else {
            uint32_t t[4];
            decode4<T>(w[f], scale, t);
            o = u32x4{t[0], t[1], t[2], t[3]};
        }
        return o;
    };

    int base = it.kv_begin + wave * TK;
    if (base < it.kv_end) load(base);
    for (; base < it.kv_end; base += 4 * TK) {
        // V into the wave's tile
        bool odd = false;
        const bool masked = base + TK > diagonal + 1;   // some row may not see all of the tile
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma unroll
                for (int f = 0; f < FL; ++f) {
                    const u32x4 w = fragment(vw[s][j], f, vscale[s]);
                    if (masked)
                        odd |= not_finite<T>(w[0]) || not_finite<T>(w[1]) || not_finite<T>(w[2]) || not_finite<T>(w[3]);
                    *(u32x4 *)(tile + (s * 16 + col) * S::kPitch + ((4 * j + quarter) * U + f * EF) * (int)sizeof(T)) = w;
                }
        const bool careful = __any(odd);   // only ever true where a later token holds an infinity or a NaN

        // S^T = K Q^T
        f32x4 sc[RT][KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][s] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma unroll
                for (int f = 0; f < FL; ++f) {
                    const Frag kf = as<Frag>(fragment(kw[s][j], f, kscale[s]));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) sc[rt][s] = mma(kf, q[rt][j * FL + f], sc[rt][s]);
                }
        }
        if (base + 4 * TK < it.kv_end) load(base + 4 * TK);

        // softmax: running maximum and sum of each query row
        typename Elem<T>::V4 p4[RT][KS];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float top = -INFINITY;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = sc[rt][s][i] * a.scale_log2;
                    if (masked && base + s * 16 + 4 * quarter + i > limit[rt]) x = -INFINITY;
                    sc[rt][s][i] = x;
                    top = fmaxf(top, x);
                }
            const float m_new = fmaxf(m[rt], max_quarters(top));
            const float m_safe = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: weights of zero, not NaN
            const float alpha = exp2_of(m[rt] - m_safe);
            m[rt] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_of(sc[rt][s][i] - m_safe);
                    sc[rt][s][i] = p;
                    sum += p;
                }
                // weights are rounded to T for the product: half a step of T each, against 32-bit sums
                p4[rt][s] = __builtin_convertvector(sc[rt][s], typename Elem<T>::V4);
            }
            l[rt] = l[rt] * alpha + sum;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= alpha;
        }

        // the tile's writes are visible to the wave's own reads in order; keep the compiler to it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

        // O^T += V^T P^T.  Where a later token holds an infinity or a NaN (careful), a zero weight does not
        // keep it from the rows that may not see it: then once for each last key, with the keys behind it
        // taken out of V, for the rows whose last key it is.
        for (int last = careful ? base : base + TK - 1; last < base + TK; ++last) {
            bool mine[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mine[rt] = !careful || min(limit[rt], base + TK - 1) == last;
            const int gone = last - base - 4 * quarter;      // of the lane's keys, the i-th of subtile s is visible if s*16 + i <= gone
            if constexpr (sizeof(T) == 2) {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4 *Lds4;
                Frag p[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) p[rt] = __builtin_shufflevector(p4[rt][0], p4[rt][1], 0, 1, 2, 3, 4, 5, 6, 7);
                // lane's share of a 4 x 16 block: row col/4, columns 4*(col%4) ..; comes back as column col
                const char *at = tile + (4 * quarter + (col >> 2)) * S::kPitch + (col & 3) * 8;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    union { s16x4 h[2]; u32x4 w; } vf;
                    vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + dt * 32));
                    vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + 16 * S::kPitch + dt * 32));
                    if (careful) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if ((i >> 2) * 16 + (i & 3) > gone) vf.h[i >> 2][i & 3] = 0;
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const f32x4 sum = mma(as<Frag>(vf.w), p[rt], acc[rt][dt]);
                        if (mine[rt]) acc[rt][dt] = sum;
                    }
                }
            } else {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    f32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = *(const float *)(tile + (4 * quarter + i) * S::kPitch + (dt * 16 + col) * 4);
                        if (careful && i > gone) v[i] = 0.0f;
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const f32x4 sum = mma(v, p4[rt][0], acc[rt][dt]);
                        if (mine[rt]) acc[rt][dt] = sum;
                    }
                }
            }
        }
    }

    // ---- join the waves
    float *joined = (float *)lds;
    f32x2 *ml = (f32x2 *)(lds + RT * 16 * S::kJoinPitch * 4);
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = sum_quarters(l[rt]);
        if (quarter == 0) ml[wave * RT * 16 + rt * 16 + col] = f32x2{m[rt], sum};
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float top = -INFINITY;
        for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * RT * 16 + rt * 16 + col][0]);
        const float f = exp2_of(m[rt] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= f;
    }
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    f32x4 *at = (f32x4 *)(joined + (rt * 16 + col) * S::kJoinPitch + dt * 16 + 4 * quarter);
                    *at = w == 0 ? acc[rt][dt] : *at + acc[rt][dt];
                }
        }
        __syncthreads();
    }

    // ---- rows out: eight elements a lane
    constexpr int LANES = DP / 8;
    for (int r = threadIdx.x / LANES; r < RT * 16; r += 256 / LANES) {
        const int row = it.row0 + r, d = threadIdx.x % LANES * 8;
        if (row >= it.rows || d >= D) continue;
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * RT * 16 + r][0]);
        for (int w = 0; w < 4; ++w)
            sum += ml[w * RT * 16 + r][1] * exp2_of(ml[w * RT * 16 + r][0] - (top == -INFINITY ? 0.0f : top));
        f32x4 x = *(f32x4 *)(joined + r * S::kJoinPitch + d), y = *(f32x4 *)(joined + r * S::kJoinPitch + d + 4);
        if (it.part_row >= 0) {
            const uint64_t at = (uint64_t)(it.part_row + r) * a.heads + h;
            *(f32x4 *)(a.part_acc + at * D + d) = x;
            *(f32x4 *)(a.part_acc + at * D + d + 4) = y;
            if (d == 0) *(f32x2 *)(a.part_ml + at * 2) = f32x2{top, sum};
            continue;
        }
        const uint32_t token = div_by((uint32_t)row, a.by_group), g = (uint32_t)row - token * a.group;
        char *dst = a.out + (uint64_t)(it.q_start + token) * a.out_token + (uint64_t)(h * a.group + g) * a.out_head + d * sizeof(T);
        const float inverse = 1.0f / sum;
        typedef typename Elem<T>::V4 V4;
        V4 *o = (V4 *)dst;
        o[0] = __builtin_convertvector(x * inverse, V4);
        o[1] = __builtin_convertvector(y * inverse, V4);
    }
}

// Partial rows into output rows: one row of one KV head for each LANES lanes.
struct JoinArgs {
    const KvJoin *joins;
    const float *part_acc, *part_ml;
    char *out;
    uint64_t out_token, out_head;
    uint32_t heads, group, head_dim, num_joins;
    Divider by_heads, by_group;
};

template <typename T, int LANES>
__global__ __launch_bounds__(256) void kvm_join_kernel(const JoinArgs a)
{
    const uint32_t join_id = div_by(blockIdx.x, a.by_heads), h = blockIdx.x - join_id * a.heads;
    const KvJoin j = a.joins[join_id];
    const int d = threadIdx.x % LANES * 8;
    const int r = blockIdx.y * (256 / LANES) + threadIdx.x / LANES;
    if (r >= j.rows || d >= (int)a.head_dim) return;
    float top = -INFINITY;
    for (int p = 0; p < j.pieces; ++p)
        top = fmaxf(top, a.part_ml[((uint64_t)(j.part_row + p * j.pitch + r) * a.heads + h) * 2]);
    const float safe = top == -INFINITY ? 0.0f : top;
    f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    float sum = 0.0f;
    for (int p = 0; p < j.pieces; ++p) {
        const uint64_t at = (uint64_t)(j.part_row + p * j.pitch + r) * a.heads + h;
        const f32x2 ml = *(const f32x2 *)(a.part_ml + at * 2);
        const float f = exp2_of(ml[0] - safe);
        sum += f * ml[1];
        x += f * *(const f32x4 *)(a.part_acc + at * a.head_dim + d);
        y += f * *(const f32x4 *)(a.part_acc + at * a.head_dim + d + 4);
    }
    const uint32_t row = (uint32_t)(j.row0 + r), token = div_by(row, a.by_group), g = row - token * a.group;
    typedef typename Elem<T>::V4 V4;
    V4 *o = (V4 *)(a.out + (uint64_t)(j.q_start + token) * a.out_token + (uint64_t)(h * a.group + g) * a.out_head + d * sizeof(T));
    const float inverse = 1.0f / sum;
    o[0] = __builtin_convertvector(x * inverse, V4);
    o[1] = __builtin_convertvector(y * inverse, V4);
}

// --------------------------------------------------------------------------- host

int refuse(int code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return kvm_internal_error(code, buf);
}

#define KV_TRY(expr)                  \
    do {                              \
        if (int rc_ = (expr)) return rc_; \
    } while (0)

int check_launch(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return refuse(KVM_EHIP, "%s failed: %s", what, hipGetErrorString(e));
    return KVM_OK;
}

int type_bytes(int64_t dtype) { return dtype == KVM_F32 ? 4 : 2; }

int check_step(const KvmStep *step, const int32_t *words, int *device)
{
    if (!step || step->seal != kvm_step_seal(*step)) return refuse(KVM_EINVAL, "the step is not one kvm_plan_step made");
    if (step->num_tokens == 0) return KVM_OK;
    return kvm_internal_pool(words, (uint64_t)step->words * 4, "the plan's words", device);
}

struct Layer {
    char *k, *v;
    uint64_t block_stride, head_stride;
    uint32_t row_bytes, codes;
};

int check_cache(const KvmStep *step, const KvmCache *c, int device, Layer *out)
{
    if (!c || !c->k || !c->v) return refuse(KVM_EINVAL, "null pool");
    if (step->num_blocks == 0) return refuse(KVM_EINVAL, "the plan was made without a cache");
    if (c->format != KVM_CACHE_PLAIN && c->format != KVM_CACHE_E4M3) return refuse(KVM_EINVAL, "unknown pool format %d", c->format);
    if (c->dtype != step->dtype)
        return refuse(KVM_EMISMATCH, "the pools' rows are of type %d, the plan is for type %d", c->dtype, (int)step->dtype);
    if (c->num_blocks != step->num_blocks || c->block_size != step->block_size || c->num_kv_heads != step->num_kv_heads ||
        c->head_dim != step->head_dim)
        return refuse(KVM_EMISMATCH,
                      "the pools are %lld blocks x %lld heads x %lld tokens x %lld, the plan is for %lld x %lld x %lld x %lld",
                      (long long)c->num_blocks, (long long)c->num_kv_heads, (long long)c->block_size, (long long)c->head_dim,
                      (long long)step->num_blocks, (long long)step->num_kv_heads, (long long)step->block_size,
                      (long long)step->head_dim);
    if (c->num_layers < 1 || c->layer < 0 || c->layer >= c->num_layers)
        return refuse(KVM_ERANGE, "layer %lld is outside [0, %lld)", (long long)c->layer, (long long)c->num_layers);
    const bool coded = c->format == KVM_CACHE_E4M3;
    if (coded && c->block_size % 16 != 0)
        return refuse(KVM_EINVAL, "a quantised pool wants a block_size that is a multiple of 16, not %lld", (long long)c->block_size);
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 != 0) return refuse(KVM_EINVAL, "pools must be 16-byte aligned");
    out->row_bytes = (uint32_t)(coded ? c->head_dim : c->head_dim * type_bytes(c->dtype));
    out->codes = (uint32_t)(c->block_size * c->head_dim);
    out->head_stride = (uint64_t)c->block_size * (out->row_bytes + (coded ? 1 : 0));
    out->block_stride = out->head_stride * (uint64_t)(c->num_kv_heads * c->num_layers);
    const uint64_t bytes = out->block_stride * (uint64_t)c->num_blocks;
    int dev = device;
    KV_TRY(kvm_internal_pool(c->k, bytes, "K pool", &dev));
    if (dev != device) return refuse(KVM_EINVAL, "the K pool is on device %d, the plan on device %d", dev, device);
    KV_TRY(kvm_internal_pool(c->v, bytes, "V pool", &dev));
    if (dev != device) return refuse(KVM_EINVAL, "the V pool is on device %d, the plan on device %d", dev, device);
    const uint64_t layer = out->head_stride * (uint64_t)(c->num_kv_heads * c->layer);
    out->k = (char *)c->k + layer;
    out->v = (char *)c->v + layer;
    return KVM_OK;
}

int check_rows(const KvmRows *r, const char *what, int64_t tokens, int64_t heads, const KvmStep *step, int device)
{
    const int64_t size = type_bytes(step->dtype);
    if (!r || !r->ptr) return refuse(KVM_EINVAL, "%s is null", what);
    if (r->token_stride < 0 || r->head_stride < 0) return refuse(KVM_EINVAL, "%s has a negative stride", what);
    if ((uintptr_t)r->ptr % 16 != 0 || r->token_stride * size % 16 != 0 || r->head_stride * size % 16 != 0)
        return refuse(KVM_EINVAL, "%s: rows must start at multiples of 16 bytes (strides %lld and %lld elements)", what,
                      (long long)r->token_stride, (long long)r->head_stride);
    const uint64_t need = (uint64_t)((tokens - 1) * r->token_stride + (heads - 1) * r->head_stride + step->head_dim) * (uint64_t)size;
    int dev = device;
    KV_TRY(kvm_internal_pool(r->ptr, need, what, &dev));
    if (dev != device) return refuse(KVM_EINVAL, "%s is on device %d, the plan on device %d", what, dev, device);
    return KVM_OK;
}

// Output rows of different (token, head) must not share memory.
int check_apart(const KvmRows *r, const char *what, int64_t tokens, int64_t heads, int64_t head_dim)
{
    const bool heads_inside = heads == 1 || (r->head_stride >= head_dim && (tokens == 1 || r->token_stride >= (heads - 1) * r->head_stride + head_dim));
    const bool tokens_inside = tokens == 1 || (r->token_stride >= head_dim && (heads == 1 || r->head_stride >= (tokens - 1) * r->token_stride + head_dim));
    if (heads == 1 ? !(tokens == 1 || r->token_stride >= head_dim) : !(heads_inside || tokens_inside))
        return refuse(KVM_EINVAL, "%s: rows overlap (strides %lld and %lld elements)", what, (long long)r->token_stride,
                      (long long)r->head_stride);
    return KVM_OK;
}

// The device the operands are on is the current one while a call launches.
struct OnDevice {
    int before = -1;
    int status = KVM_OK;
    explicit OnDevice(int device)
    {
        int now = 0;
        if (hipGetDevice(&now) != hipSuccess) {
            status = refuse(KVM_EHIP, "hipGetDevice failed");
            return;
        }
        if (now != device) {
            if (hipSetDevice(device) != hipSuccess) status = refuse(KVM_EHIP, "hipSetDevice(%d) failed", device);
            else before = now;
        }
    }
    ~OnDevice()
    {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

constexpr uint64_t kMaxGroups = 0xffffffffull / 256;   // workgroups of 256 in a launch: below 2^32 work-items

template <typename T, bool Q, int LANES> int launch_write(const MoveArgs &a, hipStream_t stream)
{
    const uint64_t groups = ((uint64_t)a.tokens * a.heads + 256 / LANES - 1) / (256 / LANES);
    if (2 * groups > kMaxGroups) return refuse(KVM_EINVAL, "too many rows for one launch");
    kvm_write_kernel<T, Q, LANES><<<dim3((uint32_t)groups, 2), 256, 0, stream>>>(a);
    return check_launch("kvm_write_kv");
}

template <typename T, bool Q> int launch_write_q(const MoveArgs &a, hipStream_t stream)
{
    if (a.head_dim <= 64) return launch_write<T, Q, 8>(a, stream);
    if (a.head_dim <= 128) return launch_write<T, Q, 16>(a, stream);
    return launch_write<T, Q, 32>(a, stream);
}

template <typename T, bool Q, int LANES> int launch_read(const MoveArgs &a, uint64_t pages, hipStream_t stream)
{
    const uint64_t groups = pages * a.heads;
    if (2 * groups > kMaxGroups) return refuse(KVM_EINVAL, "too many blocks for one launch");
    kvm_read_kernel<T, Q, LANES><<<dim3((uint32_t)groups, 2), 256, 0, stream>>>(a);
    return check_launch("kvm_read_kv");
}

template <typename T, bool Q> int launch_read_q(const MoveArgs &a, uint64_t pages, hipStream_t stream)
{
    if (a.head_dim <= 64) return launch_read<T, Q, 8>(a, pages, stream);
    if (a.head_dim <= 128) return launch_read<T, Q, 16>(a, pages, stream);
    return launch_read<T, Q, 32>(a, pages, stream);
}

template <typename T, int SRC, int DP> int launch_rows_d(const AttnArgs &a, const KvmStep *step, hipStream_t stream)
{
    const dim3 grid((uint32_t)(step->num_row_items * step->num_kv_heads));
    if constexpr (DP <= 128) {
        if (step->row_tiles == 2) kvm_rows_kernel<T, SRC, DP, 2><<<grid, 256, 0, stream>>>(a);
    }
    if (step->row_tiles == 1) kvm_rows_kernel<T, SRC, DP, 1><<<grid, 256, 0, stream>>>(a);
    return check_launch("attention");
}

template <typename T, int SRC> int launch_rows(const AttnArgs &a, const KvmStep *step, hipStream_t stream)
{
    if (step->head_dim <= 64) return launch_rows_d<T, SRC, 64>(a, step, stream);
    if (step->head_dim <= 128) return launch_rows_d<T, SRC, 128>(a, step, stream);
    return launch_rows_d<T, SRC, 256>(a, step, stream);
}

template <int SRC> int launch_rows_t(const AttnArgs &a, const KvmStep *step, hipStream_t stream)
{
    if (step->dtype == KVM_F16) return launch_rows<_Float16, SRC>(a, step, stream);
    if (step->dtype == KVM_BF16) return launch_rows<__bf16, SRC>(a, step, stream);
    return launch_rows<float, SRC>(a, step, stream);
}

template <typename T> int launch_join(const JoinArgs &a, int64_t join_rows, hipStream_t stream)
{
    const uint32_t lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32, rows = 256 / lanes;
    const dim3 grid(a.num_joins * a.heads, (uint32_t)((join_rows + rows - 1) / rows));
    if (lanes == 8) kvm_join_kernel<T, 8><<<grid, 256, 0, stream>>>(a);
    else if (lanes == 16) kvm_join_kernel<T, 16><<<grid, 256, 0, stream>>>(a);
    else kvm_join_kernel<T, 32><<<grid, 256, 0, stream>>>(a);
    return check_launch("attention");
}

// What both attention entry points share.  `source` has filled the pool fields of the arguments.
int attend(const KvmStep *step, const int32_t *words, AttnArgs a, int format, const KvmRows *q, const KvmRows *out,
           float scale, void *workspace, int64_t workspace_bytes, int device, hipStream_t stream)
{
    if (!std::isfinite(scale)) return refuse(KVM_EINVAL, "scale is not a finite number");
    KV_TRY(check_rows(q, "q", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_rows(out, "out", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_apart(out, "out", step->num_tokens, step->num_heads, step->head_dim));
    const int64_t need = kvm_attention_workspace(step);
    if (need > 0) {
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)
            return refuse(KVM_EINVAL, "the workspace has %lld bytes, %lld (16-byte aligned) are needed",
                          (long long)(workspace ? workspace_bytes : 0), (long long)need);
        int dev = device;
        KV_TRY(kvm_internal_pool(workspace, (uint64_t)need, "the workspace", &dev));
        if (dev != device) return refuse(KVM_EINVAL, "the workspace is on device %d, the plan on device %d", dev, device);
    }
    if ((uint64_t)(step->num_row_items * step->num_kv_heads) > kMaxGroups ||
        (uint64_t)(step->num_joins * step->num_kv_heads) * 8 > kMaxGroups)
        return refuse(KVM_EINVAL, "too many rows for one launch");
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    a.items = (const KvItem *)(words + step->row_items_at);
    a.table = words + step->table_at;
    a.q = (const char *)q->ptr;
    a.out = (char *)out->ptr;
    a.q_token = (uint64_t)q->token_stride * size;
    a.q_head = (uint64_t)q->head_stride * size;
    a.out_token = (uint64_t)out->token_stride * size;
    a.out_head = (uint64_t)out->head_stride * size;
    a.block_size = (uint32_t)step->block_size;
    a.heads = (uint32_t)step->num_kv_heads;
    a.group = (uint32_t)(step->num_heads / step->num_kv_heads);
    a.head_dim = (uint32_t)step->head_dim;
    a.by_block = divider(a.block_size ? a.block_size : 1);
    a.by_heads = divider(a.heads);
    a.by_group = divider(a.group);
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.part_acc = (float *)workspace;
    a.part_ml = a.part_acc + step->part_rows * step->num_kv_heads * step->head_dim;
    OnDevice on(device);
    KV_TRY(on.status);
    if (format == kPacked) KV_TRY(launch_rows_t<kPacked>(a, step, stream));
    else if (format == kE4m3) KV_TRY(launch_rows_t<kE4m3>(a, step, stream));
    else KV_TRY(launch_rows_t<kPlain>(a, step, stream));
    if (step->num_joins == 0) return KVM_OK;
    JoinArgs j;
    j.joins = (const KvJoin *)(words + step->joins_at);
    j.part_acc = a.part_acc;
    j.part_ml = a.part_ml;
    j.out = a.out;
    j.out_token = a.out_token;
    j.out_head = a.out_head;
    j.heads = a.heads;
    j.group = a.group;
    j.head_dim = a.head_dim;
    j.num_joins = (uint32_t)step->num_joins;
    j.by_heads = a.by_heads;
    j.by_group = a.by_group;
    if (step->dtype == KVM_F16) return launch_join<_Float16>(j, step->join_rows, stream);
    if (step->dtype == KVM_BF16) return launch_join<__bf16>(j, step->join_rows, stream);
    return launch_join<float>(j, step->join_rows, stream);
}

}  // namespace

extern "C" {

int kvm_write_kv(const KvmStep *step, const int32_t *words, const KvmCache *cache, const KvmRows *k, const KvmRows *v,
                 void *stream)
{
    int device = 0;
    KV_TRY(check_step(step, words, &device));
    if (step->num_tokens == 0) return KVM_OK;
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    KV_TRY(check_rows(k, "k", step->num_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(v, "v", step->num_tokens, step->num_kv_heads, step, device));
    if (step->num_tokens * step->num_kv_heads > INT32_MAX) return refuse(KVM_EINVAL, "too many rows for one launch");
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    MoveArgs a = {};
    a.slots = words + step->slots_at;
    a.src_k = (const char *)k->ptr;
    a.src_v = (const char *)v->ptr;
    a.k_token = (uint64_t)k->token_stride * size;
    a.k_head = (uint64_t)k->head_stride * size;
    a.v_token = (uint64_t)v->token_stride * size;
    a.v_head = (uint64_t)v->head_stride * size;
    a.dst_k = layer.k;
    a.dst_v = layer.v;
    a.block_stride = layer.block_stride;
    a.head_stride = layer.head_stride;
    a.row_bytes = layer.row_bytes;
    a.codes = layer.codes;
    a.tokens = (uint32_t)step->num_tokens;
    a.heads = (uint32_t)step->num_kv_heads;
    a.head_dim = (uint32_t)step->head_dim;
    a.block_size = (uint32_t)step->block_size;
    a.by_heads = divider(a.heads);
    a.by_block = divider(a.block_size);
    OnDevice on(device);
    KV_TRY(on.status);
    const hipStream_t s = (hipStream_t)stream;
    const bool coded = cache->format == KVM_CACHE_E4M3;
    if (step->dtype == KVM_F16) return coded ? launch_write_q<_Float16, true>(a, s) : launch_write_q<_Float16, false>(a, s);
    if (step->dtype == KVM_BF16) return coded ? launch_write_q<__bf16, true>(a, s) : launch_write_q<__bf16, false>(a, s);
    return coded ? launch_write_q<float, true>(a, s) : launch_write_q<float, false>(a, s);
}

int kvm_read_kv(const KvmStep *step, const int32_t *words, const KvmCache *cache, void *k_out, void *v_out, void *stream)
{
    int device = 0;
    if (!step || step->seal != kvm_step_seal(*step)) return refuse(KVM_EINVAL, "the step is not one kvm_plan_step made");
    if (step->num_kv_tokens == 0) return KVM_OK;
    KV_TRY(kvm_internal_pool(words, (uint64_t)step->words * 4, "the plan's words", &device));
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    const KvmRows ko = {k_out, step->num_kv_heads * step->head_dim, step->head_dim}, vo = {v_out, ko.token_stride, ko.head_stride};
    KV_TRY(check_rows(&ko, "k_out", step->num_kv_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(&vo, "v_out", step->num_kv_tokens, step->num_kv_heads, step, device));
    if (step->num_pages * step->num_kv_heads > INT32_MAX) return refuse(KVM_EINVAL, "too many blocks for one launch");
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    MoveArgs a = {};
    a.slots = words + step->pages_at;
    a.table = words + step->table_at;
    a.src_k = layer.k;
    a.src_v = layer.v;
    a.dst_k = (char *)k_out;
    a.dst_v = (char *)v_out;
    a.block_stride = layer.block_stride;
    a.head_stride = layer.head_stride;
    a.k_token = (uint64_t)ko.token_stride * size;
    a.k_head = (uint64_t)ko.head_stride * size;
    a.row_bytes = layer.row_bytes;
    a.codes = layer.codes;
    a.heads = (uint32_t)step->num_kv_heads;
    a.head_dim = (uint32_t)step->head_dim;
    a.block_size = (uint32_t)step->block_size;
    a.by_heads = divider(a.heads);
    OnDevice on(device);
    KV_TRY(on.status);
    const hipStream_t s = (hipStream_t)stream;
    const uint64_t pages = (uint64_t)step->num_pages;
    const bool coded = cache->format == KVM_CACHE_E4M3;
    if (step->dtype == KVM_F16) return coded ? launch_read_q<_Float16, true>(a, pages, s) : launch_read_q<_Float16, false>(a, pages, s);
    if (step->dtype == KVM_BF16) return coded ? launch_read_q<__bf16, true>(a, pages, s) : launch_read_q<__bf16, false>(a, pages, s);
    return coded ? launch_read_q<float, true>(a, pages, s) : launch_read_q<float, false>(a, pages, s);
}

int kvm_paged_attention(const KvmStep *step, const int32_t *words, const KvmCache *cache, const KvmRows *q,
                        const KvmRows *out, float scale, void *workspace, int64_t workspace_bytes, void *stream)
{
    int device = 0;
    KV_TRY(check_step(step, words, &device));
    if (step->num_tokens == 0) return KVM_OK;
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    AttnArgs a = {};
    a.k = layer.k;
    a.v = layer.v;
    a.k_block = a.v_block = layer.block_stride;
    a.k_head = a.v_head = layer.head_stride;
    a.row_bytes = layer.row_bytes;
    a.codes = layer.codes;
    return attend(step, words, a, cache->format == KVM_CACHE_E4M3 ? kE4m3 : kPlain, q, out, scale, workspace,
                  workspace_bytes, device, (hipStream_t)stream);
}

int kvm_prompt_attention(const KvmStep *step, const int32_t *words, const KvmRows *q, const KvmRows *k, const KvmRows *v,
                         const KvmRows *out, float scale, void *workspace, int64_t workspace_bytes, void *stream)
{
    int device = 0;
    KV_TRY(check_step(step, words, &device));
    if (!step->all_new) return refuse(KVM_EINVAL, "prompt attention is for sequences without earlier tokens");
    if (step->num_tokens == 0) return KVM_OK;
    KV_TRY(check_rows(k, "k", step->num_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(v, "v", step->num_tokens, step->num_kv_heads, step, device));
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    AttnArgs a = {};
    a.k = (const char *)k->ptr;
    a.v = (const char *)v->ptr;
    a.k_block = (uint64_t)k->token_stride * size;
    a.k_head = (uint64_t)k->head_stride * size;
    a.v_block = (uint64_t)v->token_stride * size;
    a.v_head = (uint64_t)v->head_stride * size;
    return attend(step, words, a, kPacked, q, out, scale, workspace, workspace_bytes, device, (hipStream_t)stream);
}

}  // extern "C"
