// kvcache_rows.h -- attention of few query rows: decoding steps, short chunks, and everything in 32 bits.
#ifndef KVCACHE_ROWS_H
#define KVCACHE_ROWS_H

#include "kvcache_device.h"

#include <cmath>

namespace kvc {

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

// Few rows: a workgroup of four waves takes RT*16 query rows (tokens x the group's heads) of one KV head over a
// range of their keys; the waves take tiles of TK keys in turn, each on its own, and their maxima, sums and
// accumulators are joined at the end (all in 32 bits).
//
// S^T = K Q^T puts a query row in a lane column, so that the softmax over keys runs over a lane's own
// registers and three other lanes, and P^T comes out just as the second product O^T = V^T P^T wants
// it: the k slots of its B operand are the rows of C, and which key a slot stands for does not
// matter as long as V^T has the same order.  K goes from memory straight into A operands (16
// contiguous bytes a lane; Q is loaded in the same order of head_dim).  V^T has to be transposed:
// through a tile in LDS of the wave's own, with the transposing LDS read (16-bit types) or element
// reads (float).  The next tile's K and V are on their way while a tile is worked on.
//
// LDS pitch: 32 bytes more than a row, so that the four rows of a transposing read and the
// eight rows of a write fall into different banks.
// Waits for the wave's own LDS traffic only, not for its loads from memory, and then for the other waves.
__device__ inline void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, int SRC, int DP, int RT> struct Rows {
    typedef typename Elem<T>::Frag Frag;
    static constexpr int EF = 16 / (int)sizeof(T);                // elements of a fragment
    static constexpr int U = SRC == kE4m3 ? 16 : EF;              // elements of a 16-byte load
    static constexpr int NL = DP / (4 * U);                       // loads of a row for a lane
    static constexpr int FL = U / EF;                             // fragments of a load
    static constexpr int KS = sizeof(T) == 4 ? 1 : 2;             // 16-key subtiles of a tile: one k step of the second product
    static constexpr int TK = 16 * KS;
    static constexpr int DT = DP / 16;                            // 16-wide tiles of head_dim in the output
    static constexpr int kPitch = DP * (int)sizeof(T) + (sizeof(T) == 4 ? 16 : 32);
    static constexpr int kTileBytes = TK * kPitch;
    static constexpr int kJoinPitch = DP + 4;                     // floats
    static constexpr int kLds = 4 * kTileBytes + 4 * 16 * 8;
    static_assert(16 * kJoinPitch * 4 <= kTileBytes, "a wave's accumulators fit its V tile");

    const AttnArgs &a;
    char *lds, *tile;
    const int wave, lane, col, quarter;

    Frag q[RT][NL * FL];
    int limit[RT];           // last key that the lane's row may see
    int diagonal;            // the rows see different last keys from this one on
    u32x4 kw[KS][NL], vw[KS][NL];
    float kscale[KS], vscale[KS];
    f32x4 acc[RT][DT];
    float m[RT], l[RT];
    bool odd = false;        // a V row that not all rows may see held an infinity or a NaN: the caller sees to it

    __device__ Rows(const AttnArgs &args, char *shared)
        : a(args), lds(shared), tile(shared + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kTileBytes),
          wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), lane(threadIdx.x & 63), col(threadIdx.x & 15),
          quarter((threadIdx.x & 63) >> 4)
    {
    }

    __device__ __forceinline__ void load(const RowWork &w, int base)
    {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int safe = min(base + s * 16 + col, w.kv_end - 1);   // keys past the last one repeat it
            const char *kp, *vp;
            if constexpr (SRC == kPacked) {
                kp = a.k + (uint64_t)(w.q_start + safe) * a.k_block + w.head * a.k_head;
                vp = a.v + (uint64_t)(w.q_start + safe) * a.v_block + w.head * a.v_head;
            } else {
                const uint32_t page = div_by((uint32_t)safe, a.by_block), off = (uint32_t)safe - page * a.block_size;
                const uint64_t slab = (uint64_t)(uint32_t)a.table[w.table_at + page] * a.k_block + w.head * a.k_head;
                kp = a.k + slab + off * a.row_bytes;
                vp = a.v + slab + off * a.row_bytes;
                if constexpr (SRC == kE4m3) {
                    kscale[s] = power_of(*(const uint8_t *)(a.k + slab + a.codes + off));
                    vscale[s] = power_of(*(const uint8_t *)(a.v + slab + a.codes + off));
                }
            }
            const char *kq = kp + quarter * 16, *vq = vp + quarter * 16;
            if ((int)a.head_dim == DP) {
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    kw[s][j] = *(const u32x4 *)(kq + j * 64);
                    vw[s][j] = *(const u32x4 *)(vq + j * 64);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    kw[s][j] = vw[s][j] = u32x4{0, 0, 0, 0};
                    if ((4 * j + quarter) * U < (int)a.head_dim) {
                        kw[s][j] = *(const u32x4 *)(kq + j * 64);
                        vw[s][j] = *(const u32x4 *)(vq + j * 64);
                    }
                }
            }
        }
    }

    // Fragment f of a loaded 16 bytes.
    static __device__ __forceinline__ u32x4 fragment(u32x4 w, int f, float scale)
    {
        if constexpr (SRC != kE4m3) return w;
        uint32_t t[4];
        if constexpr (sizeof(T) == 2) {
            decode4<T>(w[2 * f], scale, t);
            decode4<T>(w[2 * f + 1], scale, t + 2);
        } else {
            decode4<T>(w[f], scale, t);
        }
        return u32x4{t[0], t[1], t[2], t[3]};
    }

    // The rows and the first tile start on their way.
    __device__ __forceinline__ void begin(const RowWork &w)
    {
        const int base = w.kv_begin + wave * TK;
        if (base < w.kv_end) load(w, base);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = w.row0 + rt * 16 + col;
            const int clamped = min(r, w.rows - 1);
            const uint32_t token = div_by((uint32_t)clamped, a.by_group), g = (uint32_t)clamped - token * a.group;
            limit[rt] = min(w.first + (int)token, w.kv_end - 1);
            const char *src = a.q + (uint64_t)(w.q_start + token) * a.q_token + (uint64_t)(w.head * a.group + g) * a.q_head;
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma unroll
                for (int f = 0; f < FL; ++f) {
                    const int d = (4 * j + quarter) * U + f * EF;
                    u32x4 x = {0, 0, 0, 0};
                    if (r < w.rows && d < (int)a.head_dim) x = *(const u32x4 *)(src + d * sizeof(T));
                    q[rt][j * FL + f] = as<Frag>(x ^ a.q_sign);
                }
        }
        diagonal = w.first + (int)div_by((uint32_t)w.row0, a.by_group);
    }

    __device__ __forceinline__ void run(const RowWork &w)
    {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4{0, 0, 0, 0};
        }
        for (int base = w.kv_begin + wave * TK; base < w.kv_end; base += 4 * TK) step(w, base);
    }

    __device__ __forceinline__ void step(const RowWork &w, int base)
    {
        // V into the wave's tile
        const bool masked = base + TK > diagonal + 1;   // some row may not see all of the tile
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma unroll
                for (int f = 0; f < FL; ++f) {
                    const u32x4 x = fragment(vw[s][j], f, vscale[s]);
                    if (masked)
                        odd |= not_finite<T>(x[0]) || not_finite<T>(x[1]) || not_finite<T>(x[2]) || not_finite<T>(x[3]);
                    *(u32x4 *)(tile + (s * 16 + col) * kPitch + ((4 * j + quarter) * U + f * EF) * (int)sizeof(T)) = x;
                }

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
        if (base + 4 * TK < w.kv_end) load(w, base + 4 * TK);

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

        // O^T += V^T P^T
        Frag p[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (sizeof(T) == 2) p[rt] = __builtin_shufflevector(p4[rt][0], p4[rt][1], 0, 1, 2, 3, 4, 5, 6, 7);
            else p[rt] = p4[rt][0];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const Frag v = v_operand(dt);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = mma(v, p[rt], acc[rt][dt]);
        }
    }

    // V^T for tile dt of head_dim: the lane's row of it is column dt*16 + col of V, its elements are keys
    // 16*(e/4) + 4*quarter + e%4.
    __device__ __forceinline__ Frag v_operand(int dt)
    {
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *Lds4;
            // the lane's share of a 4 x 16 block: row col/4, columns 4*(col%4) ..; comes back as column col
            const char *at = tile + (4 * quarter + (col >> 2)) * kPitch + (col & 3) * 8 + dt * 32;
            union { s16x4 h[2]; Frag f; } v;
            v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)at);
            v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + 16 * kPitch));
            return v.f;
        } else {
            Frag v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *(const float *)(tile + (4 * quarter + i) * kPitch + (dt * 16 + col) * 4);
            return v;
        }
    }

    // Joins the four waves and writes the rows, as the result or as partial rows.  Loads that are on their way stay so.
    __device__ __forceinline__ void finish(const RowWork &w)
    {
        const int D = (int)a.head_dim;
        f32x2 *ml = (f32x2 *)(lds + 4 * kTileBytes);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            // a wave's accumulators take the place of its V tile
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *(f32x4 *)(tile + (col * kJoinPitch + dt * 16 + 4 * quarter) * 4) = acc[rt][dt];
            const float sum_all = sum_quarters(l[rt]);
            if (quarter == 0) ml[wave * 16 + col] = f32x2{m[rt], sum_all};
            lds_barrier();
            constexpr int LANES = DP / 8;   // eight elements a lane
            for (int r = threadIdx.x / LANES; r < 16; r += 256 / LANES) {
                const int row = w.row0 + rt * 16 + r, d = threadIdx.x % LANES * 8;
                if (row >= w.rows || d >= D) continue;
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int v = 0; v < 4; ++v) top = fmaxf(top, ml[v * 16 + r][0]);
                f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const f32x2 part = ml[v * 16 + r];
                    const float f = exp2_of(part[0] - (top == -INFINITY ? 0.0f : top));
                    const f32x4 *from = (const f32x4 *)(lds + v * kTileBytes + (r * kJoinPitch + d) * 4);
                    sum += f * part[1];
                    x += f * from[0];
                    y += f * from[1];
                }
                if (w.part_row >= 0) {
                    const uint64_t at = (uint64_t)w.part_row + rt * 16 + r;
                    *(f32x4 *)(a.part_acc + at * D + d) = x;
                    *(f32x4 *)(a.part_acc + at * D + d + 4) = y;
                    if (d == 0) *(f32x2 *)(a.part_ml + at * 2) = f32x2{top, sum};
                    continue;
                }
                const uint32_t token = div_by((uint32_t)row, a.by_group), g = (uint32_t)row - token * a.group;
                typedef typename Elem<T>::V4 V4;
                V4 *o = (V4 *)(a.out + (uint64_t)(w.q_start + token) * a.out_token + (uint64_t)(w.head * a.group + g) * a.out_head +
                               d * sizeof(T));
                const float inverse = 1.0f / sum;
                o[0] = __builtin_convertvector(x * inverse, V4);
                o[1] = __builtin_convertvector(y * inverse, V4);
            }
            lds_barrier();   // before the tiles and the sums are written again
        }
    }
};

}  // namespace kvc

#endif  // KVCACHE_ROWS_H
