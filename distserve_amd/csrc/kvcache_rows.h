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

// Rows of an item: a workgroup of four waves takes RT*16 query rows (tokens x the group's heads) of one KV head over the
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
template <typename T, int DP, int RT> struct RowShape {
    static constexpr int kSub = sizeof(T) == 4 ? 1 : 2;           // 16-key subtiles of a tile: one k step of the second product
    static constexpr int TK = 16 * kSub;
    static constexpr int kPitch = DP * (int)sizeof(T) + (sizeof(T) == 4 ? 16 : 32);
    static constexpr int kTileBytes = TK * kPitch;
    static constexpr int kJoinPitch = DP + 4;                     // floats
    static constexpr int kJoinBytes = RT * 16 * kJoinPitch * 4 + 4 * RT * 16 * 8;
    static constexpr int kLds = 4 * kTileBytes > kJoinBytes ? 4 * kTileBytes : kJoinBytes;
};

template <typename T, int SRC, int DP, int RT>
__device__ __forceinline__ void attend_rows(const AttnArgs &a, const KvItem it, const uint32_t h, char *lds)
{
    typedef RowShape<T, DP, RT> S;
    typedef typename Elem<T>::Frag Frag;
    constexpr int EF = 16 / (int)sizeof(T);                       // elements of a fragment
    constexpr int U = SRC == kE4m3 ? 16 : EF;                     // elements of a 16-byte load
    constexpr int NL = DP / (4 * U);                              // loads of a row for a lane
    constexpr int FL = U / EF;                                    // fragments of a load
    constexpr int TK = S::TK, KS = S::kSub;
    constexpr int DT = DP / 16;                                   // 16-wide tiles of head_dim in the output
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
                q[rt][j * FL + f] = as<Frag>(w ^ a.q_sign);
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

}  // namespace kvc

#endif  // KVCACHE_ROWS_H
