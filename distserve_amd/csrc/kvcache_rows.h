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

// Few rows: a workgroup takes RT*16 query rows (tokens x the group's heads) of one KV head over a range of
// their keys; its waves take tiles of TK keys in turn, each on its own, and their maxima, sums and
// accumulators are joined at the end (all in 32 bits).
//
// S^T = K Q^T puts a query row in a lane column, so that the softmax over keys runs over a lane's own
// registers and three other lanes, and P^T comes out just as the second product O^T = V^T P^T wants
// it: the k slots of its B operand are the rows of C, and which key a slot stands for does not
// matter as long as V^T has the same order.
//
// This is bound by reading K and V once.  Memory gives most when a load of the wave covers whole
// lines and says that they will not be used again: 6.9 TB/s against 5.9 TB/s for plain loads and 5.7 TB/s
// for the 64-byte pieces that loads straight into operands would be (512 MiB pools, scattered 4 KiB slabs).  So
// tiles go through LDS, 1 KiB of consecutive rows a load: plain pools straight into a tile of the wave's
// own, the next K as soon as the first product has read K, the next V after the second; codes through
// registers, where they become values.  A row's 16-byte chunks are swapped around by the row's number, so
// that the rows of an operand read, and those of a transposing read, fall into different banks.  One tile a
// wave and two workgroups a CU keep more loads in flight than two tiles a wave and one workgroup.

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
    typedef __attribute__((address_space(3))) char *LdsPtr;
    typedef const __attribute__((address_space(1))) void *GlobalPtr;
    static constexpr bool kCodes = SRC == kE4m3;
    static constexpr int EF = 16 / (int)sizeof(T);                // elements of a 16-byte chunk
    static constexpr int NF = DP / (4 * EF);                      // chunks of a row for a lane's operand
    static constexpr int KS = sizeof(T) == 4 ? 1 : 2;             // 16-key subtiles of a tile: one k step of the second product
    static constexpr int TK = 16 * KS;
    static constexpr int DT = DP / 16;                            // 16-wide tiles of head_dim in the output
    static constexpr int kRow = DP * (int)sizeof(T);              // bytes of a row in LDS
    static constexpr int kChunks = kRow / 16;
    static constexpr int kHalf = TK * kRow;                       // K's half of a tile, then V's
    static constexpr int kTile = 2 * kHalf;
    static constexpr int kWaves = DP == 256 ? 2 : 4;              // what fits a CU's LDS
    static constexpr int kLoads = kHalf / 1024;                   // 1 KiB loads of a tile's K
    static constexpr int kRowsPerLoad = TK / kLoads;
    static constexpr int kCodeLoads = TK * DP / 1024;             // the same for codes
    static constexpr int kCodeRows = 1024 / DP;
    static constexpr int kMl = kWaves * kTile;                    // where maxima and sums start
    static constexpr int kLds = kMl + kWaves * 16 * 8;
    static_assert(16 * DP * 4 == kHalf, "16 rows of a wave's accumulators fit V's half of its tile");

    static __device__ __forceinline__ int swizzle_k(int row) { return kChunks == 8 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int swizzle_v(int row)
    {
        if constexpr (sizeof(T) == 4) return ((row >> 2) & 3) << 2;
        return kChunks == 8 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
    }

    const AttnArgs &a;
    char *lds;
    const int wave, lane, col, quarter;

    Frag q[RT][NF];
    int limit[RT];           // last key that the lane's row may see
    int diagonal;            // the rows see different last keys from this one on
    int page;                // block of the lane's key (base + lane) in the tile after the one of k_off
    uint64_t k_off, v_off;   // where that key's K and V are, from the layer's start
    u32x4 kw[kCodes ? kCodeLoads : 1], vw[kCodes ? kCodeLoads : 1];   // codes on their way
    float kscale, vscale;    // of the lane's key
    f32x4 acc[RT][DT];
    float m[RT], l[RT];
    bool odd = false;        // a V row that not all rows may see held an infinity or a NaN: the caller sees to it

    __device__ Rows(const AttnArgs &args, char *shared)
        : a(args), lds(shared), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), lane(threadIdx.x & 63),
          col(threadIdx.x & 15), quarter((threadIdx.x & 63) >> 4)
    {
        // chunks of K past head_dim are never loaded: they stay as they are here
        if ((int)a.head_dim < DP) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) *(u32x4 *)(tile() + j * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        }
    }

    __device__ __forceinline__ char *tile() { return lds + wave * kTile; }

    // Keys past the last one repeat it: their weights are zero.
    __device__ __forceinline__ int key_of(const RowWork &w, int base) const { return min(base + (lane & (TK - 1)), w.kv_end - 1); }

    __device__ __forceinline__ void look_up(const RowWork &w, int base)
    {
        if constexpr (SRC != kPacked) page = a.table[w.table_at + (int)div_by((uint32_t)key_of(w, base), a.by_block)];
    }

    // Where the keys of the tile at `base` are; `page` is theirs.  The page of the wave's next tile is asked for now, before
    // this tile's loads, so that waiting for it will not mean waiting for them.
    __device__ __forceinline__ void locate(const RowWork &w, int base)
    {
        const int key = key_of(w, base);
        if constexpr (SRC == kPacked) {
            k_off = (uint64_t)(w.q_start + key) * a.k_block + w.head * a.k_head;
            v_off = (uint64_t)(w.q_start + key) * a.v_block + w.head * a.v_head;
        } else {
            const uint32_t off = (uint32_t)key - div_by((uint32_t)key, a.by_block) * a.block_size;
            const uint64_t slab = (uint64_t)(uint32_t)page * a.k_block + w.head * a.k_head;
            k_off = v_off = slab + off * a.row_bytes;
            if (base + kWaves * TK < w.kv_end) look_up(w, base + kWaves * TK);
            if constexpr (kCodes) {
                kscale = power_of(*(const uint8_t *)(a.k + slab + a.codes + off));
                vscale = power_of(*(const uint8_t *)(a.v + slab + a.codes + off));
            }
        }
    }

    // The offset that lane `row` has worked out.
    static __device__ __forceinline__ uint64_t of_row(uint64_t off, int row)
    {
        return ((uint64_t)(uint32_t)__shfl((int)(off >> 32), row) << 32) | (uint32_t)__shfl((int)off, row);
    }
    static __device__ __forceinline__ uint64_t of_first_row(uint64_t off, int row)
    {
        return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), row) << 32) |
               (uint32_t)__builtin_amdgcn_readlane((int)off, row);
    }

    // Whether all rows of a load lie one behind the other: then one address is enough.
    template <int ROWS> __device__ __forceinline__ bool in_a_row(const RowWork &w, int base) const
    {
        return base + TK <= w.kv_end && (SRC == kPacked || a.block_size % ROWS == 0);
    }

    // K's (V's) half of the tile starts on its way into LDS.
    template <bool IS_V> __device__ __forceinline__ void load(const RowWork &w, int base)
    {
        constexpr int kPolicy = sizeof(T) == 4 ? 0 : 2;      // not used again (in 32 bits, many rows share K and V)
        const char *from = IS_V ? a.v : a.k;
        const uint64_t off = IS_V ? v_off : k_off;
        const uint32_t pitch = SRC == kPacked ? (uint32_t)(IS_V ? a.v_block : a.k_block) : a.row_bytes;
        char *at = tile() + (IS_V ? kHalf : 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was there has been read
        if (in_a_row<kRowsPerLoad>(w, base)) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = j * kRowsPerLoad + lane / kChunks;
                const int chunk = lane % kChunks ^ (IS_V ? swizzle_v(row) : swizzle_k(row));
                const char *first = from + of_first_row(off, j * kRowsPerLoad);
                if (chunk * EF < (int)a.head_dim)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(first + (lane / kChunks * pitch + chunk * 16)), (LdsPtr)(at + j * 1024),
                                                     16, 0, kPolicy);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = j * kRowsPerLoad + lane / kChunks;
                const int chunk = lane % kChunks ^ (IS_V ? swizzle_v(row) : swizzle_k(row));
                const char *there = from + of_row(off, row);
                if (chunk * EF < (int)a.head_dim)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(there + chunk * 16), (LdsPtr)(at + j * 1024), 16, 0, kPolicy);
            }
        }
    }

    // Codes of the tile start on their way into registers.
    __device__ __forceinline__ void load_codes(const RowWork &w, int base)
    {
        const int row = lane / (DP / 16), d = lane % (DP / 16) * 16;
        uint64_t at[kCodeLoads];
        if (in_a_row<kCodeRows>(w, base)) {
#pragma unroll
            for (int j = 0; j < kCodeLoads; ++j) at[j] = of_first_row(k_off, j * kCodeRows) + (row * a.row_bytes + d);
        } else {
#pragma unroll
            for (int j = 0; j < kCodeLoads; ++j) at[j] = of_row(k_off, j * kCodeRows + row) + d;
        }
#pragma unroll
        for (int j = 0; j < kCodeLoads; ++j) kw[j] = vw[j] = u32x4{0, 0, 0, 0};
        if (d < (int)a.head_dim) {
#pragma unroll
            for (int j = 0; j < kCodeLoads; ++j) {
                kw[j] = __builtin_nontemporal_load((const u32x4 *)(a.k + at[j]));
                vw[j] = __builtin_nontemporal_load((const u32x4 *)(a.v + at[j]));
            }
        }
    }

    // Codes that have arrived, as values into the wave's tile.
    __device__ __forceinline__ void decode()
    {
        if (__builtin_expect(__any(may_overflow<T>(fmaxf(kscale, vscale))), 0)) decode_as<true>();
        else decode_as<false>();
    }
    template <bool LARGE> __device__ __forceinline__ void decode_as()
    {
#pragma unroll
        for (int j = 0; j < kCodeLoads; ++j) {
            const int row = j * kCodeRows + lane / (DP / 16), first = lane % (DP / 16) * (16 / EF);
            const float ks = __shfl(kscale, row), vs = __shfl(vscale, row);
            char *at = tile() + row * kRow;
#pragma unroll
            for (int f = 0; f < 16 / EF; ++f) {
                *(u32x4 *)(at + ((first + f) ^ swizzle_k(row)) * 16) = values<LARGE>(kw[j], f, ks);
                *(u32x4 *)(at + kHalf + ((first + f) ^ swizzle_v(row)) * 16) = values<LARGE>(vw[j], f, vs);
            }
        }
    }

    // Chunk f of 16 codes.
    template <bool LARGE> static __device__ __forceinline__ u32x4 values(u32x4 w, int f, float scale)
    {
        uint32_t t[4];
        if constexpr (sizeof(T) == 2) {
            decode4<T>(w[2 * f], scale, t);
            decode4<T>(w[2 * f + 1], scale, t + 2);
        } else {
            decode4<T>(w[f], scale, t);
        }
        if constexpr (LARGE) return u32x4{saturated(t[0]), saturated(t[1]), saturated(t[2]), saturated(t[3])};
        return u32x4{t[0], t[1], t[2], t[3]};
    }

    // The piece's first K and its query rows start on their way; V's half of the tile is left alone.
    __device__ __forceinline__ void begin(const RowWork &w)
    {
        const int base = w.kv_begin + wave * TK;
        look_up(w, base);
        locate(w, base);
        if constexpr (kCodes) load_codes(w, base);
        else if (base < w.kv_end) load<false>(w, base);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = w.row0 + rt * 16 + col;
            const int clamped = min(r, w.rows - 1);
            const uint32_t token = div_by((uint32_t)clamped, a.by_group), g = (uint32_t)clamped - token * a.group;
            limit[rt] = min(w.first + (int)token, w.kv_end - 1);
            const char *src = a.q + (uint64_t)(w.q_start + token) * a.q_token + (uint64_t)(w.head * a.group + g) * a.q_head;
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const int d = (4 * j + quarter) * EF;
                u32x4 x = {0, 0, 0, 0};
                if ((r < w.rows) & (d < (int)a.head_dim)) x = *(const u32x4 *)(src + d * sizeof(T));
                q[rt][j] = as<Frag>(x ^ a.q_sign);
            }
        }
        diagonal = w.first + (int)div_by((uint32_t)w.row0, a.by_group);
    }

    // After begin(), when V's half of the tile is free.
    __device__ __forceinline__ void begin_v(const RowWork &w)
    {
        const int base = w.kv_begin + wave * TK;
        if constexpr (!kCodes)
            if (base < w.kv_end) load<true>(w, base);
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
        for (int base = w.kv_begin + wave * TK; base < w.kv_end; base += kWaves * TK) {
            const int after = base + kWaves * TK;
            const bool more = after < w.kv_end;
            f32x4 sc[RT][KS];
            if constexpr (kCodes) {
                decode();
                if (more) {
                    locate(w, after);
                    load_codes(w, after);
                }
                scores(sc);
                weigh(base, sc);
            } else {
                // all loads but the last kLoads, which are V's: K has arrived
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
                scores(sc);
                if (more) {
                    locate(w, after);
                    load<false>(w, after);
                    // all but the next K's
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
                    weigh(base, sc);
                    load<true>(w, after);
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    weigh(base, sc);
                }
            }
        }
    }

    // Whether V's half of the tile holds an infinity or a NaN (in columns that exist).
    __device__ __forceinline__ bool odd_values()
    {
        bool seen = false;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int row = j * kRowsPerLoad + lane / kChunks, pos = lane % kChunks;
            const u32x4 x = *(const u32x4 *)(tile() + kHalf + j * 1024 + lane * 16);
            const bool there = (pos ^ swizzle_v(row)) * EF < (int)a.head_dim;
#pragma unroll
            for (int i = 0; i < 4; ++i) seen = seen || not_finite<T>(there ? x[i] : 0);
        }
        return seen;
    }

    // S^T = K Q^T for the tile's K.
    __device__ __forceinline__ void scores(f32x4 (&sc)[RT][KS])
    {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][s] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const int row = s * 16 + col, chunk = 4 * j + quarter;
                const u32x4 x = *(const u32x4 *)(tile() + row * kRow + (chunk ^ swizzle_k(row)) * 16);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][s] = mma(as<Frag>(x), q[rt][j], sc[rt][s]);
            }
        }
    }

    // Softmax of the scores of keys base .., and the tile's V.
    __device__ __forceinline__ void weigh(int base, f32x4 (&sc)[RT][KS])
    {
        const bool masked = base + TK > diagonal + 1;   // some row may not see all of the tile
        if (masked) odd |= odd_values();

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
            if (sizeof(T) == 4 || __any(alpha != 1.0f)) {   // most tiles move no maximum; bound by the product in 32 bits
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= alpha;
            }
        }

        // O^T += V^T P^T
        Frag p[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (sizeof(T) == 2) p[rt] = __builtin_shufflevector(p4[rt][0], p4[rt][1], 0, 1, 2, 3, 4, 5, 6, 7);
            else p[rt] = p4[rt][0];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const Frag v = v_operand(tile() + kHalf, dt);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = mma(v, p[rt], acc[rt][dt]);
        }
    }

    // V^T for tile dt of head_dim: the lane's row of it is column dt*16 + col of V, its elements are keys
    // 16*(e/4) + 4*quarter + e%4.
    __device__ __forceinline__ Frag v_operand(const char *vt, int dt)
    {
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *Lds4;
            // the lane's share of a 4 x 16 block: row col/4, columns 4*(col%4) ..; comes back as column col
            const int row = 4 * quarter + (col >> 2);
            const char *at = vt + row * kRow + ((2 * dt + ((col & 3) >> 1)) ^ swizzle_v(row)) * 16 + (col & 1) * 8;
            union { s16x4 h[2]; Frag f; } v;
            v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)at);
            v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + 16 * kRow));
            return v.f;
        } else {
            Frag v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 4 * quarter + i;
                v[i] = *(const float *)(vt + row * kRow + ((4 * dt + (col >> 2)) ^ swizzle_v(row)) * 16 + (col & 3) * 4);
            }
            return v;
        }
    }

    // Chunk c of row r of a wave's accumulators, in V's half of its tile.
    __device__ __forceinline__ f32x4 *part(int of_wave, int r, int c) const
    {
        return (f32x4 *)(lds + of_wave * kTile + kHalf + r * (DP * 4) + (c ^ r) * 16);
    }

    // Joins the waves and writes the rows, as the result or as partial rows.  K and rows that are on their way stay so.
    __device__ __forceinline__ void finish(const RowWork &w)
    {
        const int D = (int)a.head_dim;
        f32x2 *ml = (f32x2 *)(lds + kMl);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *part(wave, col, dt * 4 + quarter) = acc[rt][dt];
            const float sum_all = sum_quarters(l[rt]);
            if (quarter == 0) ml[wave * 16 + col] = f32x2{m[rt], sum_all};
            lds_barrier();
            // Eight elements a lane.  The conditions below are kept side by side, not one inside the other: where an inner
            // one ended right before an outer one, the compiler (ROCm 7.2) has been seen to copy registers back with
            // only the inner one's lanes enabled.
            constexpr int LANES = DP / 8, kPass = 64 * kWaves / LANES;   // rows at a time
#pragma unroll
            for (int pass = 0; pass < (16 + kPass - 1) / kPass; ++pass) {
                const int r = pass * kPass + threadIdx.x / LANES, row = w.row0 + rt * 16 + r, d = threadIdx.x % LANES * 8;
                const bool live = (r < 16) & (row < w.rows) & (d < D);
                const int rr = min(r, 15);
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int v = 0; v < kWaves; ++v) top = fmaxf(top, ml[v * 16 + rr][0]);
                f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
                for (int v = 0; v < kWaves; ++v) {
                    const f32x2 of_wave = ml[v * 16 + rr];
                    const float f = exp2_of(of_wave[0] - (top == -INFINITY ? 0.0f : top));
                    sum += f * of_wave[1];
                    x += f * *part(v, rr, d / 4);
                    y += f * *part(v, rr, d / 4 + 1);
                }
                if (w.part_row >= 0) {
                    const uint64_t at = (uint64_t)w.part_row + rt * 16 + rr;
                    if (live) {
                        *(f32x4 *)(a.part_acc + at * D + d) = x;
                        *(f32x4 *)(a.part_acc + at * D + d + 4) = y;
                    }
                    if (live & (d == 0)) *(f32x2 *)(a.part_ml + at * 2) = f32x2{top, sum};
                } else {
                    const uint32_t safe = (uint32_t)min(row, w.rows - 1), token = div_by(safe, a.by_group), g = safe - token * a.group;
                    typedef typename Elem<T>::V4 V4;
                    V4 *o = (V4 *)(a.out + (uint64_t)(w.q_start + token) * a.out_token + (uint64_t)(w.head * a.group + g) * a.out_head +
                                   d * sizeof(T));
                    const float inverse = 1.0f / sum;
                    if (live) {
                        o[0] = output4<T>(x * inverse);
                        o[1] = output4<T>(y * inverse);
                    }
                }
            }
            lds_barrier();   // before the tiles and the sums are written again
        }
    }
};

}  // namespace kvc

#endif  // KVCACHE_ROWS_H
