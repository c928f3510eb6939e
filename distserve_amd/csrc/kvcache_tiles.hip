// kvcache_tiles.hip -- attention of many query rows (chunks of prompts, whole prompts), 16-bit types.
//
// A workgroup of four waves takes 128 query rows (tokens x the group's heads) of one KV head over
// the keys of its item, 64 keys at a time; a wave has 32 of the rows.  As in the row kernel,
// S^T = K Q^T and O^T = V^T P^T, so that a query row is a lane column of both products (32x32x16
// matrix instructions; lanes l and l+32 share the row) and P^T needs no shuffle between them.
//
// K and V tiles lie in LDS, two of each: while a tile is used the next one is on its way from memory,
// straight into LDS (plain pools and packed rows) or through registers, where codes become values
// (quantised pools).  A row's 16-byte chunks are swapped around by the row's number, so that the 16
// rows of an operand read, and the four rows of a transposing read, fall into different banks.
//
// Bound by the matrix cores and the softmax's VALU work, which take turns: on a prompt of 8192 tokens, 64 query and 8
// KV heads of 128 in bf16, the matrix cores are busy 51 % of the time and the VALU 50 %, LDS 27 %, without bank
// conflicts; 1.08 ms, 1.02 PFLOP/s (a large library product reaches 1.14 on this card).  Two workgroups a CU cover for
// each other; 64 rows a wave, one workgroup a CU, is 2.7 times slower, and raising a wave's priority around the products or
// summing weights by dot products changes nothing.  Lengths 64 .. 2048 packed, 32 heads: 0.37 ms, 0.66 PFLOP/s,
// of an item 13 tiles on average: masked and empty parts of tiles are 6 % of the work by waves and 18 % by workgroups, matrix cores are
// busy 35 % and VALU 44 %; the rest is what an item does before its first product and after its last.
#include "kv_internal.h"
#include "kvcache_slow.h"
#include "kvcache_tiles.h"

#include <cstdio>

namespace {

using namespace kvc;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char *LdsPtr;
typedef __attribute__((address_space(3))) s16x4 *Lds4;
typedef const __attribute__((address_space(1))) void *GlobalPtr;

constexpr int kKeys = 64;   // of a tile

// C[m][n] += sum_k A[m][k] B[k][n]: lane l holds A[l%32][8*(l/32) ..] and B[8*(l/32) ..][l%32], and of C
// column l%32, rows 8*(i/4) + 4*(l/32) + i%4, i = 0..15.
__device__ inline f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ inline float max_halves(float x) { return fmaxf(x, __shfl_xor(x, 32)); }

template <typename T, int SRC, int DP> struct TileKernel {
    typedef typename Elem<T>::Frag Frag;
    static constexpr int kRow = DP * 2;                 // bytes of a row in LDS
    static constexpr int kChunks = DP / 8;
    static constexpr int kTile = kKeys * kRow;
    static constexpr int kFlags = 4 * kTile;            // K, K, V, V, then whether a wave saw an infinity or a NaN, twice
    static constexpr int kLds = kFlags + 32;
    static constexpr int kSteps = DP / 16;              // k steps of the first product
    static constexpr int kDt = DP / 32;                 // 32-wide tiles of head_dim in the output
    static constexpr int kRowsPerLoad = 1024 / kRow;    // rows of a wave's 16-byte-a-lane load
    static constexpr int kLoads = 16 / kRowsPerLoad;    // a wave brings 16 of the 64 rows
    static constexpr int kCoded = DP / 64;              // quantised: 16-code loads of a lane for a row

    static __device__ int swizzle_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ int swizzle_out(int row) { return DP == 64 ? row & 7 : row & 15; }
    static __device__ int swizzle_v(int row) { return DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

    const AttnArgs &a;
    const KvItem it;
    const int h, wave, lane, col, half;
    char *lds;

    // the wave's 16 rows of a tile
    u32x4 kw[kCoded], vw[kCoded];       // quantised: on their way to LDS
    float kscale, vscale;
    int pages;                          // lane i: the block of the wave's rows in tile page_tile + i
    int page_tile;

    __device__ void fetch_pages(int tile)
    {
        page_tile = tile;
        const int key = min(it.kv_begin + (tile + lane) * kKeys + 16 * wave, (it.kv_end - 1) & ~15);
        pages = a.table[it.table_at + (int)div_by((uint32_t)key, a.by_block)];
    }

    // Starts tile t's way into buffer `buffer`: rows past the last key repeat it (their weights are zero).
    __device__ void load(int t, int buffer)
    {
        const int last = it.kv_end - 1;
        int r0 = it.kv_begin + t * kKeys + 16 * wave;
        if (r0 > last) r0 = last & ~15;
        const int room = last - r0;             // rows of the 16 that exist, less one
        const char *kp, *vp;
        uint32_t k_pitch, v_pitch;
        if constexpr (SRC == kPacked) {
            kp = a.k + (uint64_t)(it.q_start + r0) * a.k_block + h * a.k_head;
            vp = a.v + (uint64_t)(it.q_start + r0) * a.v_block + h * a.v_head;
            k_pitch = (uint32_t)a.k_block;
            v_pitch = (uint32_t)a.v_block;
        } else {
            if (t >= page_tile + 64) fetch_pages(t);
            const uint32_t block = (uint32_t)__builtin_amdgcn_readlane(pages, t - page_tile);
            const uint32_t off = (uint32_t)r0 - div_by((uint32_t)r0, a.by_block) * a.block_size;   // of 16 rows in one block
            const uint64_t slab = (uint64_t)block * a.k_block + h * a.k_head;
            kp = a.k + slab + off * a.row_bytes;
            vp = a.v + slab + off * a.row_bytes;
            k_pitch = v_pitch = a.row_bytes;
            if constexpr (SRC == kE4m3) {
                const int row = min(lane >> 2, room);
                kscale = power_of(*(const uint8_t *)(a.k + slab + a.codes + off + row));
                vscale = power_of(*(const uint8_t *)(a.v + slab + a.codes + off + row));
#pragma unroll
                for (int j = 0; j < kCoded; ++j) {
                    const int d = (4 * j + (lane & 3)) * 16;
                    kw[j] = vw[j] = u32x4{0, 0, 0, 0};
                    if (d < (int)a.head_dim) {
                        kw[j] = *(const u32x4 *)(kp + (uint32_t)row * k_pitch + d);
                        vw[j] = *(const u32x4 *)(vp + (uint32_t)row * v_pitch + d);
                    }
                }
            }
        }
        if constexpr (SRC != kE4m3) {
            char *at = lds + buffer * kTile + 16 * wave * kRow;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = j * kRowsPerLoad + lane / kChunks, pos = lane % kChunks;
                const int kc = pos ^ swizzle_k(row), vc = pos ^ swizzle_v(row);
                const int there = min(row, room);
                // chunks past head_dim are zero since the start
                if (kc * 8 < (int)a.head_dim)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(kp + ((uint32_t)there * k_pitch + kc * 16)),
                                                     (LdsPtr)(at + j * 1024), 16, 0, 0);
                if (vc * 8 < (int)a.head_dim)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(vp + ((uint32_t)there * v_pitch + vc * 16)),
                                                     (LdsPtr)(at + 2 * kTile + j * 1024), 16, 0, 0);
            }
        }
    }

    // Quantised: the loaded codes as values into the buffer.
    __device__ void store(int buffer)
    {
        if constexpr (SRC == kE4m3) {
            if (__builtin_expect(__any(may_overflow<T>(fmaxf(kscale, vscale))), 0)) store_as<true>(buffer);
            else store_as<false>(buffer);
        }
    }
    template <bool LARGE> __device__ __forceinline__ void store_as(int buffer)
    {
        const int row = 16 * wave + (lane >> 2);
        char *at = lds + buffer * kTile + row * kRow;
#pragma unroll
        for (int j = 0; j < kCoded; ++j)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int chunk = (4 * j + (lane & 3)) * 2 + f;
                *(u32x4 *)(at + (chunk ^ swizzle_k(row)) * 16) = values<LARGE>(kw[j], f, kscale);
                *(u32x4 *)(at + 2 * kTile + (chunk ^ swizzle_v(row)) * 16) = values<LARGE>(vw[j], f, vscale);
            }
    }
    // Chunk f of 16 codes.
    template <bool LARGE> static __device__ __forceinline__ u32x4 values(u32x4 w, int f, float scale)
    {
        uint32_t t[4];
        decode4<T>(w[2 * f], scale, t);
        decode4<T>(w[2 * f + 1], scale, t + 2);
        if constexpr (LARGE) return u32x4{saturated(t[0]), saturated(t[1]), saturated(t[2]), saturated(t[3])};
        return u32x4{t[0], t[1], t[2], t[3]};
    }

    Frag q[kSteps];
    f32x16 acc[kDt];
    float m, l;    // maximum (scaled, in powers of two) that the weights refer to; the lane's share of their sum
    int limit;

    // Whether the wave's 16 rows of the V tile hold an infinity or a NaN: exponents of all ones carry into the
    // sign's place.
    __device__ bool odd_values(int buffer)
    {
        constexpr uint32_t one = std::is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u;
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const u32x4 w = *(const u32x4 *)(lds + (2 + buffer) * kTile + 16 * wave * kRow + j * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) seen |= (w[i] & 0x7fff7fffu) + one;
        }
        return (seen & 0x80008000u) != 0;
    }

    // One tile.  masked: some row may not see all of its keys.
    __device__ void compute(int base, int buffer, bool masked)
    {
        const char *kt = lds + buffer * kTile, *vt = kt + 2 * kTile;
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                const int row = 32 * u + col;
                const Frag kf = *(const Frag *)(kt + row * kRow + (((2 * step + half) ^ swizzle_k(row)) << 4));
                s[u] = mma(kf, q[step], s[u]);
            }
        Frag p[4];
        if (masked) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (base + 32 * u + 8 * (i / 4) + 4 * half + i % 4 > limit) s[u][i] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        top = max_halves(top) * a.scale_log2;
        // The weights may refer to an older maximum as long as they stay below 2^8 (fp16 holds 2^15): rescaling
        // the accumulators is then rare.
        if (__any(top > m + 8.0f)) {
            const float m_new = fmaxf(m, top);
            const float alpha = m == -INFINITY ? 0.0f : exp2_of(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
        }
        const float safe = m == -INFINITY ? 0.0f : m;   // nothing seen yet: weights of zero, not NaN
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = exp2_of(fmaf(s[u][i], a.scale_log2, -safe));
                s[u][i] = w;
                sum += w;
            }
        l += sum;
        // weights are rounded to T for the product: half a step of T each, against 32-bit sums
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            typedef float f32x8 __attribute__((ext_vector_type(8)));
            f32x8 w;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = s[k / 2][8 * (k % 2) + i];
            p[k] = __builtin_convertvector(w, Frag);
        }
        // O^T += V^T P^T; slot (half, e) of a k step stands for key 16*k + 8*(e/4) + 4*half + e%4
        const int rr = (lane & 15) >> 2, part = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) {
                const char *at = vt + (16 * k + 4 * half + rr) * kRow + (((dt * 4 + part) ^ swizzle_v(rr)) << 4) + (lane & 1) * 8;
                union { s16x4 h[2]; u32x4 w; } vf;
                vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)at);
                vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + 8 * kRow));
                acc[dt] = mma(as<Frag>(vf.w), p[k], acc[dt]);
            }
    }

    // All tiles, the first of which is on its way; false as soon as one that is masked holds an infinity or a NaN in V, which a weight of zero does
    // not keep from the rows that may not see it.
    __device__ bool pass(int first_row)
    {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;
        const int tiles = (it.kv_end - it.kv_begin + kKeys - 1) / kKeys;
        // the first row sees keys up to `least`; the wave's first row up to `wave_least`, its last one up to `most`
        const int last_row = min(first_row + 32, it.rows) - 1;
        const bool idle = first_row >= it.rows;
        const int least = it.first + (int)div_by((uint32_t)it.row0, a.by_group);
        const int wave_least = it.first + (int)div_by((uint32_t)min(first_row, it.rows - 1), a.by_group);
        const int most = it.first + (int)div_by((uint32_t)max(last_row, 0), a.by_group);
        store(0);
        for (int t = 0; t < tiles; ++t) {
            const int base = it.kv_begin + t * kKeys, end = base + kKeys - 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's share of the tile has arrived
            int *flags = (int *)(lds + kFlags) + (t & 1) * 4;
            if (end > least) {
                const bool odd = __any(odd_values(t & 1));
                if (lane == 0) flags[wave] = odd;
            }
            __syncthreads();                      // everybody's has; nobody reads the other buffer any more
            if (t + 1 < tiles) load(t + 1, (t + 1) & 1);
            if (end > least) {
                if (__builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3])) return false;
            }
            if (!idle && base <= most) compute(base, t & 1, end > wave_least);
            if (t + 1 < tiles) store((t + 1) & 1);
        }
        return true;
    }

    __device__ TileKernel(const AttnArgs &args, char *shared, const KvItem &item, uint32_t head)
        : a(args), it(item), h(item.head0 + (int)head), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          lane(threadIdx.x & 63), col(threadIdx.x & 31), half((threadIdx.x & 63) >> 5), lds(shared)
    {
    }

    // the item's first partial row
    __device__ int64_t part_at() const { return (int64_t)a.part_items + (int64_t)h * a.part_head + it.part_row; }

    __device__ void run()
    {
        const int D = (int)a.head_dim, first_row = it.row0 + wave * 32;
        if (D < DP) {
            for (int i = threadIdx.x; i < kFlags / 16; i += 256) *(u32x4 *)(lds + i * 16) = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        // the first tile, and the rows meanwhile
        if constexpr (SRC != kPacked) fetch_pages(0);
        load(0, 0);
        const int r = first_row + col, clamped = min(r, it.rows - 1);
        const uint32_t token = div_by((uint32_t)clamped, a.by_group), g = (uint32_t)clamped - token * a.group;
        limit = min(it.first + (int)token, it.kv_end - 1);
        const char *src = a.q + (uint64_t)(it.q_start + token) * a.q_token + (uint64_t)(h * a.group + g) * a.q_head;
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            const int d = step * 16 + half * 8;
            u32x4 w = {0, 0, 0, 0};
            if ((r < it.rows) & (d < D)) w = *(const u32x4 *)(src + d * 2);
            q[step] = as<Frag>(w ^ a.q_sign);
        }
        if (!pass(first_row)) {
            const RowWork all = {it.q_start, it.rows, it.first, it.table_at, it.row0, h, it.kv_begin, it.kv_end,
                                 it.part_row < 0 ? -1 : part_at()};
            attend_slow<T, SRC, DP>(a, all, 128);
            __builtin_amdgcn_s_waitcnt(0x0f70);   // the next tile may still be on its way into LDS
            return;
        }
        __syncthreads();   // the tiles have been read
        const float sum = l + __shfl_xor(l, 32);
        const bool live = r < it.rows;
        if (it.part_row >= 0) {
            const uint64_t at = (uint64_t)part_at() + (r - it.row0);
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 32 * dt + 8 * i + 4 * half;
                    if (live & (d < D))
                        *(f32x4 *)(a.part_acc + at * D + d) = f32x4{acc[dt][4 * i], acc[dt][4 * i + 1],
                                                                    acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
                }
            if (live & (half == 0)) *(f32x2 *)(a.part_ml + at * 2) = f32x2{m, sum};
            return;
        }
        // the wave's rows through its share of the tiles, so that whole rows are written at a time
        char *mine = lds + wave * kTile;
        const float inverse = 1.0f / sum;
        typedef typename Elem<T>::V4 V4;
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 x = {acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
                *(V4 *)(mine + col * kRow + ((4 * dt + i) ^ swizzle_out(col)) * 16 + half * 8) = output4<T>(x * inverse);
            }
#pragma unroll
        for (int j = 0; j < 2 * kLoads; ++j) {
            const int row = j * kRowsPerLoad + lane / kChunks, chunk = lane % kChunks, to = first_row + row;
            const u32x4 x = *(const u32x4 *)(mine + row * kRow + (chunk ^ swizzle_out(row)) * 16);
            const uint32_t safe = (uint32_t)min(to, it.rows - 1), token = div_by(safe, a.by_group), g = safe - token * a.group;
            char *dst = a.out + (uint64_t)(it.q_start + token) * a.out_token + (uint64_t)(h * a.group + g) * a.out_head;
            if ((to < it.rows) & (chunk * 8 < D)) *(u32x4 *)(dst + chunk * 16) = x;
        }
    }
};

template <typename T, int SRC, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void kvm_tiles_kernel(const AttnArgs a)
{
    typedef TileKernel<T, SRC, DP> K;
    __shared__ __attribute__((aligned(1024))) char lds[K::kLds];
    const uint32_t width = min(a.heads, (uint32_t)kHeadBlock);
    const uint32_t item_id = a.heads < kHeadBlock ? div_by(blockIdx.x, a.by_heads) : blockIdx.x / (uint32_t)kHeadBlock;
    K kernel(a, lds, uniform(a.items + item_id), blockIdx.x - item_id * width);
    if (kernel.h < (int)a.heads) kernel.run();
}

template <typename T, int SRC> void launch(const AttnArgs &a, uint32_t groups, hipStream_t stream)
{
    if (a.head_dim <= 64) kvm_tiles_kernel<T, SRC, 64><<<groups, 256, 0, stream>>>(a);
    else if (a.head_dim <= 128) kvm_tiles_kernel<T, SRC, 128><<<groups, 256, 0, stream>>>(a);
    else kvm_tiles_kernel<T, SRC, 256><<<groups, 256, 0, stream>>>(a);
}

template <typename T> void launch_source(const AttnArgs &a, int source, uint32_t groups, hipStream_t stream)
{
    if (source == kPacked) launch<T, kPacked>(a, groups, stream);
    else if (source == kE4m3) launch<T, kE4m3>(a, groups, stream);
    else launch<T, kPlain>(a, groups, stream);
}

}  // namespace

int kvm_launch_tiles(const kvc::AttnArgs &a, int dtype, int source, uint32_t groups, hipStream_t stream)
{
    if (dtype == KVM_F16) launch_source<_Float16>(a, source, groups, stream);
    else launch_source<__bf16>(a, source, groups, stream);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return KVM_OK;
    char text[128];
    snprintf(text, sizeof text, "attention failed: %s", hipGetErrorString(e));
    return kvm_internal_error(KVM_EHIP, text);
}
