// kvcache_slow.h -- attention row by row, for workgroups that met an infinity or a NaN.
//
// The matrix instructions multiply every key's V with every row's weight, and a weight of zero times
// an infinity is a NaN: where a V row that only some of the workgroup's query rows may see holds
// such a value, the workgroup's piece is computed here instead, a wave a row, over the
// keys that the row may see and no others.  Some ten times slower, and in use only where a model
// has left the finite numbers.
#ifndef KVCACHE_SLOW_H
#define KVCACHE_SLOW_H

#include "kvcache_device.h"

#include <cmath>

namespace kvc {

// A decoded value as a T holds it: past the largest fp16 number it is that number.
template <typename T> __device__ __forceinline__ float held(uint32_t w)
{
    const float x = __uint_as_float(w);
    if constexpr (std::is_same<T, _Float16>::value) return fabsf(x) > 65504.0f ? copysignf(65504.0f, x) : x;
    return x;
}

// Rows row0 .. row0 + count - 1 of the piece, dealt out over the workgroup's waves.
template <typename T, int SRC, int DP>
__device__ __forceinline__ void attend_slow(const AttnArgs &a, const RowWork w, const int count)
{
    constexpr int EL = DP / 64;                                   // columns of a lane: lane, lane + 64, ..
    constexpr int U = SRC == kE4m3 ? 16 : 16 / (int)sizeof(T);    // elements of a 16-byte load
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int D = (int)a.head_dim;
    for (int r = wave; r < count && w.row0 + r < w.rows; r += (int)blockDim.x / 64) {
        const uint32_t row = (uint32_t)(w.row0 + r), token = div_by(row, a.by_group), g = row - token * a.group;
        const int end = min(w.first + (int)token + 1, w.kv_end);
        const char *src = a.q + (uint64_t)(w.q_start + token) * a.q_token + (uint64_t)(w.head * a.group + g) * a.q_head;
        float q[EL], acc[EL], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
            const int d = lane + 64 * i;
            acc[i] = 0.0f;
            q[i] = d < D ? (float)*(const T *)(src + d * sizeof(T)) : 0.0f;
            if (a.q_sign) q[i] = -q[i];
        }
        for (int base = w.kv_begin; base < end; base += 64) {
            const int key = min(base + lane, end - 1), n = min(64, end - base);
            uint64_t k_off, v_off;
            float ks = 1.0f, vs = 1.0f;
            if constexpr (SRC == kPacked) {
                k_off = (uint64_t)(w.q_start + key) * a.k_block + w.head * a.k_head;
                v_off = (uint64_t)(w.q_start + key) * a.v_block + w.head * a.v_head;
            } else {
                const uint32_t page = div_by((uint32_t)key, a.by_block), off = (uint32_t)key - page * a.block_size;
                const uint64_t slab = (uint64_t)(uint32_t)a.table[w.table_at + page] * a.k_block + w.head * a.k_head;
                k_off = v_off = slab + off * a.row_bytes;
                if constexpr (SRC == kE4m3) {
                    ks = power_of(*(const uint8_t *)(a.k + slab + a.codes + off));
                    vs = power_of(*(const uint8_t *)(a.v + slab + a.codes + off));
                }
            }
            // a key a lane
            float s = 0.0f;
            for (int d = 0; d < D; d += U) {
                const u32x4 x = *(const u32x4 *)(a.k + k_off + d * (16 / U));
                uint32_t e[U];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (SRC == kE4m3) decode4<float>(x[i], ks, e + 4 * i);
                    else e[i] = x[i];
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float qd = 0.0f;
#pragma unroll
                    for (int j = 0; j < EL; ++j)
                        if ((d + i) / 64 == j) qd = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q[j]), (d + i) % 64));
                    float k;
                    if constexpr (SRC == kE4m3) k = held<T>(e[i]);
                    else k = element<T>(e, i);
                    s = fmaf(k, qd, s);
                }
            }
            s = lane < n ? s * a.scale_log2 : -INFINITY;
            float top = s;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
            const float m_new = fmaxf(m, top), safe = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = exp2_of(m - safe), p = exp2_of(s - safe);
            float sum = p;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
            m = m_new;
            l = l * alpha + sum;
#pragma unroll
            for (int i = 0; i < EL; ++i) acc[i] *= alpha;
            // a column a lane
            for (int j = 0; j < n; ++j) {
                const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j));
                const uint64_t off = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v_off >> 32), j) << 32) |
                                     (uint32_t)__builtin_amdgcn_readlane((uint32_t)v_off, j);
                const float scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), j));
#pragma unroll
                for (int i = 0; i < EL; ++i) {
                    const int d = lane + 64 * i;
                    if (d >= D) continue;
                    float v;
                    if constexpr (SRC == kE4m3) {
                        uint32_t four[4];
                        decode4<float>(*(const uint8_t *)(a.v + off + d), scale, four);
                        v = held<T>(four[0]);
                    } else {
                        v = (float)*(const T *)(a.v + off + d * sizeof(T));
                    }
                    acc[i] = fmaf(pj, v, acc[i]);
                }
            }
        }
        char *dst = a.out + (uint64_t)(w.q_start + token) * a.out_token + (uint64_t)(w.head * a.group + g) * a.out_head;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) continue;
            if (w.part_row >= 0) a.part_acc[(uint64_t)(w.part_row + r) * D + d] = acc[i];
            else *(T *)(dst + d * sizeof(T)) = (T)in_range<T>(acc[i] / l);
        }
        if (w.part_row >= 0 && lane == 0) *(f32x2 *)(a.part_ml + (uint64_t)(w.part_row + r) * 2) = f32x2{m, l};
    }
}

}  // namespace kvc

#endif  // KVCACHE_SLOW_H
