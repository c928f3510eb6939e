// kvcache.hip -- the cache operators for MI355X (gfx950, wave64): new tokens' K and V into the
// paged pools (plain or as e4m3 codes), the pools read back, and attention over them.
//
// A step plan (kvcache_plan.cpp) says which cache slot each new token has and which pieces the
// attention is cut into; the kernels find everything else from it.  Reference call site of
// what these operators do: distserve/worker.py:211-227 (the model forward gets the pools and
// the block table).
#include "kv_internal.h"
#include "kvcache_rows.h"
#include "kvcache_slow.h"
#include "kvcache_tiles.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <limits>

namespace {

using namespace kvc;

// ---- write and read back
//
// Pure data movement: a lane takes eight elements of a row, 8, 16 or 32 lanes a row (the power of two
// that covers head_dim; lanes past it idle).  Consecutive rows of a workgroup are consecutive tokens of one
// head, which lie side by side in the pool (codes and, more so, their scale bytes).
//
// Both are bound by HBM, and by the launch where there is little to move.  Measured: 16 prompts, 20 heads of 128 in
// bf16 (392 MB read and written) 70.5 us, 5.6 TB/s; 12 prompts, 8 heads of 128 in bf16 written as codes 24.4 us and
// read back 17.5 us (179 MB together); one token of 96 sequences, 32 heads of 128, 2.7 us.  Two or four rows a lane, several
// heads a workgroup, or workgroups of one wave were slower by 2 to 10 %.
//
// Quantising: e is the smallest exponent with max|x| <= 448 * 2^e, code = e4m3(x / 2^e), rounded to nearest even (half a step,
// 2^-4 of the value); the division is by a power of two and exact.

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

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// Maximum over the LANES lanes of a row (8, 16 or 32): neighbours, pairs, mirrored eights and sixteens.
template <int LANES> __device__ inline uint32_t row_max(uint32_t x)
{
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));    // quad_perm 1 0 3 2
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));    // quad_perm 2 3 0 1
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));   // row_half_mirror
    if constexpr (LANES >= 16) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true));   // row_mirror
    if constexpr (LANES >= 32) x = max(x, (uint32_t)__shfl_xor((int)x, 16));
    return x;
}

// The finite number whose magnitude has these bits.
template <typename T> __device__ inline float magnitude(uint32_t bits)
{
    return element<T>(&bits, 0);
}

// Smallest e with top <= 448 * 2^e, -126 at least, 0 for 0; 448 = 0.875 * 2^9.
__device__ inline int scale_exponent(float top)
{
    int x;
    const float part = frexpf(top, &x);
    return top > 0.0f ? max(part <= 0.875f ? x - 9 : x - 8, -126) : 0;
}

// Four elements divided by the scale (a power of two), as codes: rounded to nearest, ties to even.
template <typename T> __device__ inline uint32_t encode4(const uint32_t *w, float scale)
{
    union { s16x2 h; uint32_t w; } c;
    c.w = 0;
    if constexpr (std::is_same<T, _Float16>::value) {
        union { uint32_t w; f16x2 h; } a, b;
        a.w = w[0];
        b.w = w[1];
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c.h, a.h, scale, false);
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c.h, b.h, scale, true);
    } else if constexpr (std::is_same<T, __bf16>::value) {
        union { uint32_t w; bf16x2 h; } a, b;
        a.w = w[0];
        b.w = w[1];
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c.h, a.h, scale, false);
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c.h, b.h, scale, true);
    } else {
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c.h, __uint_as_float(w[0]), __uint_as_float(w[1]), scale, false);
        c.h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c.h, __uint_as_float(w[2]), __uint_as_float(w[3]), scale, true);
    }
    return c.w;
}

// T: the rows' type.  Q: quantised pool.  LANES: lanes of a row.
template <typename T, bool Q, int LANES>
__global__ __launch_bounds__(256) void kvm_write_kernel(const MoveArgs a)
{
    constexpr int W = sizeof(T) * 2;                                   // words of a lane's eight elements
    const uint32_t group = div_by(blockIdx.x, a.by_heads), head = blockIdx.x - group * a.heads;
    const uint32_t token = group * (256 / LANES) + threadIdx.x / LANES;
    if (token >= a.tokens) return;                                     // a row's lanes leave together
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
                __builtin_nontemporal_store(*(u32x4 *)(w + 4 * i), (u32x4 *)(slab + off * a.row_bytes + d * sizeof(T)) + i);
        }
    } else {
        // Largest magnitude of the row, by bit patterns: those of finite numbers are in the numbers' order, and those of
        // infinities and NaN above them all.
        constexpr uint32_t kInf = sizeof(T) == 4 ? 0x7f800000u : Elem<T>::kExponent & 0xffffu;
        uint32_t top = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < W; ++i) top = max(top, w[i] & 0x7fffffffu);
        } else {
            u16x2 pair = {0, 0};
#pragma unroll
            for (int i = 0; i < W; ++i) {
                union { uint32_t w; u16x2 h; } x;
                x.w = w[i] & 0x7fff7fffu;
                pair = __builtin_elementwise_max(pair, x.h);
            }
            top = max((uint32_t)pair[0], (uint32_t)pair[1]);
        }
        top = row_max<LANES>(top);
        uint32_t c[2];
        int e;
        if (__builtin_expect(!__any(top >= kInf), 1)) {
            e = scale_exponent(magnitude<T>(top));
            const float scale = power_of((uint32_t)(127 + e));
#pragma unroll
            for (int i = 0; i < 2; ++i) c[i] = encode4<T>(w + i * W / 2, scale);
        } else {
            // infinities do not count for the scale and saturate; NaN stays NaN
            float x[8], most = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = element<T>(w, i);
                most = fmaxf(most, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
            }
            e = scale_exponent(__uint_as_float(row_max<LANES>(__float_as_uint(most))));
            const float inverse = power_of((uint32_t)(127 - e));          // e <= 120, so this is a normal number
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[i] * inverse;
                x[i] = y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
                c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], p, true);
            }
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
    const uint64_t token_stride = is_v ? a.v_token : a.k_token;
    char *out = (is_v ? a.dst_v + head * a.v_head : a.dst_k + head * a.k_head) + d * sizeof(T);
    for (int32_t t = threadIdx.x / LANES; t < count; t += 256 / LANES) {
        uint32_t w[W];
        if constexpr (Q) {
            const u32x2 c = *(const u32x2 *)(slab + (uint64_t)t * a.row_bytes + d);
            const float scale = power_of(*(const uint8_t *)(slab + a.codes + t));
            decode4<T>(c[0], scale, w);
            decode4<T>(c[1], scale, w + W / 2);
            if (may_overflow<T>(scale)) {
#pragma unroll
                for (int i = 0; i < W; ++i) w[i] = saturated(w[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
                *(u32x4 *)(w + 4 * i) = *((const u32x4 *)(slab + (uint64_t)t * a.row_bytes + d * sizeof(T)) + i);
        }
#pragma unroll
        for (int i = 0; i < W / 4; ++i)
            __builtin_nontemporal_store(*(u32x4 *)(w + 4 * i), (u32x4 *)(out + (uint64_t)(first + t) * token_stride) + i);
    }
}

// ---- attention

// Bound by reading K and V (the launch and the plan's first words where there are few).  Measured, kernel alone:
// single tokens of 32 sequences of 64 .. 2048, 32 heads of 128 in fp16, 80 us, 5.6 TB/s; of 8 sequences of 8000 .. 48000, 8 KV
// heads in bf16, 104 us, 6.5 TB/s; of 64 sequences over e4m3 codes, 58 us, 5.1 TB/s, where LDS is busy 47 % of the time (39 % of
// that with bank conflicts), VALU 37 %, and nothing is full.  In 32 bits, 32 sequences of 64 .. 2048, 32 heads, 173 us, 5.2 TB/s;
// 64 sequences over codes 144 us; chunks of 512 behind thousands 69 TFLOP/s and packed prompts 58 (a library product: 154).
//
// A workgroup for few rows walks its share of the units of all (row tile, KV head) pairs: perhaps the end of
// a pair, then whole ones, then the beginning of one.  The next piece's first K is under way while a piece's
// rows are joined and written.
template <typename T, int SRC, int DP, int RT>
__global__ __launch_bounds__(DP == 256 ? 128 : 256, DP == 128 && RT == 1 ? 2 : 1) void kvm_rows_kernel(const AttnArgs a)
{
    typedef Rows<T, SRC, DP, RT> R;
    static_assert(64 * R::kWaves == (DP == 256 ? 128 : 256), "the launch bounds are the workgroup's size");
    __shared__ __attribute__((aligned(1024))) char lds[R::kLds];
    R rows(a, lds);
    KvStart at;
    KvTile t;
    auto first = [&]() {
        at = uniform(a.starts + blockIdx.x);
        t = at.first;
    };
    auto piece = [&]() {
        RowWork w;
        const int n = min(at.units, t.units - at.unit);
        w.q_start = t.q_start;
        w.rows = t.rows;
        w.first = t.first;
        w.table_at = t.table_at;
        w.row0 = t.row0;
        w.head = at.head;
        w.kv_begin = at.unit * (int)kUnit;
        w.kv_end = min(t.kv_end, (at.unit + n) * (int)kUnit);
        w.part_row = n == t.units ? -1 : (int64_t)(at.unit == 0 ? a.part_starts : 0) + (int64_t)blockIdx.x * a.part_pitch;
        at.units -= n;
        at.unit = 0;
        if (++at.head == (int)a.heads) {
            at.head = 0;
            ++at.tile;
            if (at.units > 0) t = uniform(a.tiles + at.tile);
        }
        return w;
    };
    first();
    RowWork now = piece();
    rows.begin(now);
    rows.begin_v(now);
    for (;;) {
        rows.run(now);
        if (at.units == 0) break;
        const RowWork next = piece();
        rows.begin(next);
        rows.finish(now);
        rows.begin_v(next);
        now = next;
    }
    rows.finish(now);
    // some piece met an infinity or a NaN that not all of its rows may see: all pieces once more, row by row
    if (__builtin_expect(__syncthreads_or(rows.odd), 0)) {
        __builtin_amdgcn_s_waitcnt(0x0f70);   // the rows written above are to be written over
        __syncthreads();
        first();
        while (at.units > 0) attend_slow<T, SRC, DP>(a, piece(), RT * 16);
    }
}

// Partial rows into output rows: LANES lanes a row.
struct JoinArgs {
    const KvJoin *joins;
    const float *part_acc, *part_ml;
    char *out;
    uint64_t out_token, out_head;
    uint32_t group, head_dim;
    Divider by_group;
};

// Bound by reading the partial rows: 4 to 5 us behind single tokens, 11.6 us where two chunks of 700 tokens were cut
// (36 MB), of which some 2 us are the launch.
//
// The lanes of a row look at the pieces' maxima and sums side by side; then the pieces' rows are added up, a few
// loads in flight at a time.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void kvm_join_kernel(const JoinArgs a)
{
    const KvJoin j = a.joins[blockIdx.x];
    const int lane = threadIdx.x % LANES, d = lane * 8;
    const int r = blockIdx.y * (256 / LANES) + threadIdx.x / LANES;
    if (r >= j.rows) return;                       // a row's lanes leave together
    auto part_row = [&](int p) { return (uint64_t)(uint32_t)(p == 0 ? j.part_row : j.next_row + (p - 1) * j.pitch) + r; };
    float top = -INFINITY, sum = 0.0f;
    for (int p = lane; p < j.pieces; p += LANES) {
        const f32x2 ml = *(const f32x2 *)(a.part_ml + part_row(p) * 2);
        const float m = fmaxf(top, ml[0]);
        const float safe = m == -INFINITY ? 0.0f : m;
        sum = sum * exp2_of(top - safe) + ml[1] * exp2_of(ml[0] - safe);
        top = m;
    }
    float all = top;
#pragma unroll
    for (int x = 1; x < LANES; x <<= 1) all = fmaxf(all, __shfl_xor(all, x));
    const float safe = all == -INFINITY ? 0.0f : all;
    sum *= exp2_of(top - safe);
#pragma unroll
    for (int x = 1; x < LANES; x <<= 1) sum += __shfl_xor(sum, x);
    if (d >= (int)a.head_dim) return;
    f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll 4
    for (int p = 0; p < j.pieces; ++p) {
        const uint64_t at = part_row(p);
        const float f = exp2_of(a.part_ml[at * 2] - safe);
        const f32x4 *from = (const f32x4 *)(a.part_acc + at * a.head_dim + d);
        x += f * from[0];
        y += f * from[1];
    }
    const uint32_t row = (uint32_t)(j.row0 + r), token = div_by(row, a.by_group), g = row - token * a.group;
    typedef typename Elem<T>::V4 V4;
    V4 *o = (V4 *)(a.out + (uint64_t)(j.q_start + token) * a.out_token + (uint64_t)((uint32_t)j.head * a.group + g) * a.out_head +
                   d * sizeof(T));
    const float inverse = 1.0f / sum;
    o[0] = output4<T>(x * inverse);
    o[1] = output4<T>(y * inverse);
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

int check_seal(const KvmStep *step)
{
    if (!step || step->seal != kvm_step_seal(*step)) return refuse(KVM_EINVAL, "the step is not one kvm_plan_step made");
    return KVM_OK;
}

// `need` bytes at p, on *device if that is known: by what the caller vouches for, or by asking the runtime.
int check_memory(const KvmStep *step, const void *p, uint64_t need, int64_t extent, const char *what, int *device)
{
    if (!p) return refuse(KVM_EINVAL, "%s is null", what);
    if (step->device >= 0) {
        *device = (int)step->device;
        if (extent < 0 || need > (uint64_t)extent)
            return refuse(KVM_ERANGE, "%s needs %llu bytes but has %lld", what, (unsigned long long)need, (long long)extent);
        return KVM_OK;
    }
    int dev = -1;
    if (int rc = kvm_internal_pool(p, need, what, &dev)) return rc;
    if (*device >= 0 && dev != *device) return refuse(KVM_EINVAL, "%s is on device %d, the plan on device %d", what, dev, *device);
    *device = dev;
    return KVM_OK;
}

int check_words(const KvmStep *step, const int32_t *words, int *device)
{
    const uint64_t need = (uint64_t)step->words * 4;
    *device = -1;
    if ((uintptr_t)words % 16 != 0) return refuse(KVM_EINVAL, "the plan's words must be 16-byte aligned");
    return check_memory(step, words, need, (int64_t)need, "the plan's words", device);
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
    if (c->format != step->format)
        return refuse(KVM_EMISMATCH, "the pools are of format %d, the plan is for format %d", c->format, (int)step->format);
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
    // (2^26 bytes of a slab, 2^20 heads and 2^31 slots at most, but any number of layers)
    const unsigned __int128 all = (unsigned __int128)(out->head_stride * (uint64_t)c->num_kv_heads) * (uint64_t)c->num_layers;
    if (all > (uint64_t)INT64_MAX || all * (uint64_t)c->num_blocks > (uint64_t)INT64_MAX)
        return refuse(KVM_ERANGE, "a pool of %lld layers is too large", (long long)c->num_layers);
    out->block_stride = (uint64_t)all;
    const uint64_t bytes = out->block_stride * (uint64_t)c->num_blocks;
    KV_TRY(check_memory(step, c->k, bytes, c->extent, "the K pool", &device));
    KV_TRY(check_memory(step, c->v, bytes, c->extent, "the V pool", &device));
    const uint64_t layer = out->head_stride * (uint64_t)(c->num_kv_heads * c->layer);
    out->k = (char *)c->k + layer;
    out->v = (char *)c->v + layer;
    return KVM_OK;
}

// Elements from the first to behind the last one.
unsigned __int128 reach(const KvmRows *r, int64_t tokens, int64_t heads, int64_t head_dim)
{
    return (unsigned __int128)(tokens - 1) * (uint64_t)r->token_stride + (unsigned __int128)(heads - 1) * (uint64_t)r->head_stride +
           (uint64_t)head_dim;
}

int check_rows(const KvmRows *r, const char *what, int64_t tokens, int64_t heads, const KvmStep *step, int device)
{
    const int64_t size = type_bytes(step->dtype);
    if (!r || !r->ptr) return refuse(KVM_EINVAL, "%s is null", what);
    if (r->token_stride < 0 || r->head_stride < 0) return refuse(KVM_EINVAL, "%s has a negative stride", what);
    if ((uintptr_t)r->ptr % 16 != 0 || (uint64_t)r->token_stride * (uint64_t)size % 16 != 0 ||
        (uint64_t)r->head_stride * (uint64_t)size % 16 != 0)
        return refuse(KVM_EINVAL, "%s: rows must start at multiples of 16 bytes (strides %lld and %lld elements)", what,
                      (long long)r->token_stride, (long long)r->head_stride);
    const unsigned __int128 need = reach(r, tokens, heads, step->head_dim) * (uint64_t)size;
    if (need > (uint64_t)INT64_MAX) return refuse(KVM_ERANGE, "%s: strides %lld and %lld are too large", what, (long long)r->token_stride, (long long)r->head_stride);
    return check_memory(step, r->ptr, (uint64_t)need, r->extent, what, &device);
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

bool disjoint(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes)
{
    return (uintptr_t)a + a_bytes <= (uintptr_t)b || (uintptr_t)b + b_bytes <= (uintptr_t)a;
}

// Written rows must not lie on rows that the same call reads or writes elsewhere: workgroups come to them in any order.  Rows
// that take turns in memory (slices of one fused projection) are apart.
int check_clear(const KvmRows *out, int64_t out_heads, const KvmRows *in, int64_t in_heads, int64_t tokens, const KvmStep *step,
                const char *what)
{
    const uint64_t size = (uint64_t)type_bytes(step->dtype), row = (uint64_t)step->head_dim * size;
    if (disjoint(out->ptr, (uint64_t)reach(out, tokens, out_heads, step->head_dim) * size, in->ptr,
                 (uint64_t)reach(in, tokens, in_heads, step->head_dim) * size))
        return KVM_OK;
    // both repeat every `period` bytes: `a` bytes of it are out's, from its start, and `b` bytes in's
    auto take_turns = [&](uint64_t period, uint64_t a, uint64_t b) {
        if (period == 0 || a > period || b > period) return false;
        const uint64_t off = ((uintptr_t)in->ptr % period + period - (uintptr_t)out->ptr % period) % period;
        return off >= a && off + b <= period;
    };
    auto width = [&](const KvmRows *r, int64_t heads) { return (uint64_t)(heads - 1) * (uint64_t)r->head_stride * size + row; };
    if (out->token_stride == in->token_stride &&
        take_turns((uint64_t)out->token_stride * size, width(out, out_heads), width(in, in_heads)))
        return KVM_OK;
    const int64_t head = out_heads > 1 ? out->head_stride : in->head_stride;
    if (head > 0 && (out_heads == 1 || out->head_stride == head) && (in_heads == 1 || in->head_stride == head) &&
        out->token_stride % head == 0 && in->token_stride % head == 0 && take_turns((uint64_t)head * size, row, row))
        return KVM_OK;
    return refuse(KVM_EINVAL, "%s share memory", what);
}

// The same for rows (their whole reach) and a stretch of memory: the plan's words, a workspace.
int check_clear_of(const KvmRows *rows, int64_t tokens, int64_t heads, const KvmStep *step, const void *p, uint64_t bytes, const char *what)
{
    const uint64_t need = (uint64_t)reach(rows, tokens, heads, step->head_dim) * (uint64_t)type_bytes(step->dtype);
    return disjoint(rows->ptr, need, p, bytes) ? KVM_OK : refuse(KVM_EINVAL, "%s share memory", what);
}

// The same for rows and whole pools.
int check_clear_of_pools(const KvmRows *rows, int64_t tokens, int64_t heads, const KvmStep *step, const KvmCache *c, const Layer &layer,
                         const char *what)
{
    const uint64_t bytes = layer.block_stride * (uint64_t)c->num_blocks;
    const uint64_t need = (uint64_t)reach(rows, tokens, heads, step->head_dim) * (uint64_t)type_bytes(step->dtype);
    if (disjoint(rows->ptr, need, c->k, bytes) && disjoint(rows->ptr, need, c->v, bytes)) return KVM_OK;
    return refuse(KVM_EINVAL, "%s and a pool share memory", what);
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
    const uint64_t groups = ((uint64_t)a.tokens + 256 / LANES - 1) / (256 / LANES) * a.heads;
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
    const dim3 grid((uint32_t)step->num_row_groups);
    // (more than 16 rows of 16 bits over codes are the kernel for many rows' work: quantised blocks hold 16 tokens or more)
    if constexpr (DP <= 128 && (SRC != kE4m3 || sizeof(T) == 4)) {
        if (step->row_tiles == 2) kvm_rows_kernel<T, SRC, DP, 2><<<grid, 64 * Rows<T, SRC, DP, 2>::kWaves, 0, stream>>>(a);
    }
    if (step->row_tiles == 1) kvm_rows_kernel<T, SRC, DP, 1><<<grid, 64 * Rows<T, SRC, DP, 1>::kWaves, 0, stream>>>(a);
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

template <typename T> int launch_join(const JoinArgs &a, uint32_t num_joins, int64_t join_rows, hipStream_t stream)
{
    const uint32_t lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32, rows = 256 / lanes;
    const dim3 grid(num_joins, (uint32_t)((join_rows + rows - 1) / rows));
    if (lanes == 8) kvm_join_kernel<T, 8><<<grid, 256, 0, stream>>>(a);
    else if (lanes == 16) kvm_join_kernel<T, 16><<<grid, 256, 0, stream>>>(a);
    else kvm_join_kernel<T, 32><<<grid, 256, 0, stream>>>(a);
    return check_launch("attention");
}

// What both attention entry points share.  `source` has filled the pool fields of the arguments.
int attend(const KvmStep *step, const int32_t *words, AttnArgs a, int format, const KvmRows *q, const KvmRows *out,
           float scale, void *workspace, int64_t workspace_bytes, int device, hipStream_t stream)
{
    const float scale_log2 = fabsf(scale) * 1.44269504088896340736f;
    if (!std::isfinite(scale_log2)) return refuse(KVM_EINVAL, "scale is not a finite number, or not one in powers of two (2.3e38 and more)");
    KV_TRY(check_rows(q, "q", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_rows(out, "out", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_apart(out, "out", step->num_tokens, step->num_heads, step->head_dim));
    KV_TRY(check_clear(out, step->num_heads, q, step->num_heads, step->num_tokens, step, "out and q"));
    const int64_t need = kvm_attention_workspace(step);
    if (need > 0) {
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)
            return refuse(KVM_EINVAL, "the workspace has %lld bytes, %lld (16-byte aligned) are needed",
                          (long long)(workspace ? workspace_bytes : 0), (long long)need);
        KV_TRY(check_memory(step, workspace, (uint64_t)need, workspace_bytes, "the workspace", &device));
        KV_TRY(check_clear_of(q, step->num_tokens, step->num_heads, step, workspace, (uint64_t)need, "q and the workspace"));
        KV_TRY(check_clear_of(out, step->num_tokens, step->num_heads, step, workspace, (uint64_t)need, "out and the workspace"));
        if (!disjoint(words, (uint64_t)step->words * 4, workspace, (uint64_t)need))
            return refuse(KVM_EINVAL, "the plan's words and the workspace share memory");
    }
    KV_TRY(check_clear_of(out, step->num_tokens, step->num_heads, step, words, (uint64_t)step->words * 4, "out and the plan's words"));
    const uint64_t tile_groups = (uint64_t)(step->num_tile_items * std::min(step->num_kv_heads, kHeadBlock));
    if (tile_groups > kMaxGroups || (uint64_t)step->num_joins * 16 > kMaxGroups)
        return refuse(KVM_EINVAL, "too many rows for one launch");
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
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
    // a negative scale turns q's signs over; a scale of zero is the smallest one, which keeps masked scores at -infinity and makes
    // no more than 2^-21 of the largest ones
    a.scale_log2 = fmaxf(scale_log2, std::numeric_limits<float>::denorm_min());
    a.q_sign = scale >= 0 ? 0u : size == 4 ? 0x80000000u : 0x80008000u;
    a.part_acc = (float *)workspace;
    a.part_ml = a.part_acc + step->part_rows * step->head_dim;
    a.part_pitch = (uint32_t)(16 * step->row_tiles);
    a.part_starts = (uint32_t)(step->num_row_groups * 16 * step->row_tiles);
    a.part_items = (uint32_t)step->row_part_rows;
    a.part_head = (uint32_t)step->item_part_rows;
    OnDevice on(device);
    KV_TRY(on.status);
    a.tiles = (const KvTile *)(words + step->row_tiles_at);
    a.starts = (const KvStart *)(words + step->row_starts_at);
    a.items = (const KvItem *)(words + step->tile_items_at);
    if (step->num_tile_items > 0)
        KV_TRY(kvm_launch_tiles(a, (int)step->dtype, format, (uint32_t)tile_groups, stream));
    if (step->num_row_groups > 0) {
        if (format == kPacked) KV_TRY(launch_rows_t<kPacked>(a, step, stream));
        else if (format == kE4m3) KV_TRY(launch_rows_t<kE4m3>(a, step, stream));
        else KV_TRY(launch_rows_t<kPlain>(a, step, stream));
    }
    if (step->num_joins == 0) return KVM_OK;
    JoinArgs j;
    j.joins = (const KvJoin *)(words + step->joins_at);
    j.part_acc = a.part_acc;
    j.part_ml = a.part_ml;
    j.out = a.out;
    j.out_token = a.out_token;
    j.out_head = a.out_head;
    j.group = a.group;
    j.head_dim = a.head_dim;
    j.by_group = a.by_group;
    if (step->dtype == KVM_F16) return launch_join<_Float16>(j, (uint32_t)step->num_joins, step->join_rows, stream);
    if (step->dtype == KVM_BF16) return launch_join<__bf16>(j, (uint32_t)step->num_joins, step->join_rows, stream);
    return launch_join<float>(j, (uint32_t)step->num_joins, step->join_rows, stream);
}

}  // namespace

extern "C" {

int kvm_write_kv(const KvmStep *step, const int32_t *words, const KvmCache *cache, const KvmRows *k, const KvmRows *v,
                 void *stream)
{
    int device = 0;
    KV_TRY(check_seal(step));
    if (step->num_tokens == 0) return KVM_OK;
    KV_TRY(check_words(step, words, &device));
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    KV_TRY(check_rows(k, "k", step->num_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(v, "v", step->num_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_clear_of_pools(k, step->num_tokens, step->num_kv_heads, step, cache, layer, "k"));
    KV_TRY(check_clear_of_pools(v, step->num_tokens, step->num_kv_heads, step, cache, layer, "v"));
    const uint64_t pool = layer.block_stride * (uint64_t)cache->num_blocks;
    if (!disjoint(cache->k, pool, cache->v, pool)) return refuse(KVM_EINVAL, "the K pool and the V pool share memory");
    if (!disjoint(cache->k, pool, words, (uint64_t)step->words * 4) || !disjoint(cache->v, pool, words, (uint64_t)step->words * 4))
        return refuse(KVM_EINVAL, "a pool and the plan's words share memory");
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

int kvm_read_kv(const KvmStep *step, const int32_t *words, const KvmCache *cache, const KvmRows *k_out,
                const KvmRows *v_out, void *stream)
{
    int device = 0;
    KV_TRY(check_seal(step));
    if (step->num_kv_tokens == 0) return KVM_OK;
    KV_TRY(check_words(step, words, &device));
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    KV_TRY(check_rows(k_out, "k_out", step->num_kv_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(v_out, "v_out", step->num_kv_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_apart(k_out, "k_out", step->num_kv_tokens, step->num_kv_heads, step->head_dim));
    KV_TRY(check_apart(v_out, "v_out", step->num_kv_tokens, step->num_kv_heads, step->head_dim));
    KV_TRY(check_clear(k_out, step->num_kv_heads, v_out, step->num_kv_heads, step->num_kv_tokens, step, "k_out and v_out"));
    KV_TRY(check_clear_of_pools(k_out, step->num_kv_tokens, step->num_kv_heads, step, cache, layer, "k_out"));
    KV_TRY(check_clear_of_pools(v_out, step->num_kv_tokens, step->num_kv_heads, step, cache, layer, "v_out"));
    for (const KvmRows *r : {k_out, v_out})
        KV_TRY(check_clear_of(r, step->num_kv_tokens, step->num_kv_heads, step, words, (uint64_t)step->words * 4,
                              r == k_out ? "k_out and the plan's words" : "v_out and the plan's words"));
    if (step->num_pages * step->num_kv_heads > INT32_MAX) return refuse(KVM_EINVAL, "too many blocks for one launch");
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    MoveArgs a = {};
    a.slots = words + step->pages_at;
    a.table = words + step->table_at;
    a.src_k = layer.k;
    a.src_v = layer.v;
    a.dst_k = (char *)k_out->ptr;
    a.dst_v = (char *)v_out->ptr;
    a.block_stride = layer.block_stride;
    a.head_stride = layer.head_stride;
    a.k_token = (uint64_t)k_out->token_stride * size;
    a.k_head = (uint64_t)k_out->head_stride * size;
    a.v_token = (uint64_t)v_out->token_stride * size;
    a.v_head = (uint64_t)v_out->head_stride * size;
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
    KV_TRY(check_seal(step));
    if (step->num_tokens == 0) return KVM_OK;
    KV_TRY(check_words(step, words, &device));
    Layer layer;
    KV_TRY(check_cache(step, cache, device, &layer));
    KV_TRY(check_rows(out, "out", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_clear_of_pools(out, step->num_tokens, step->num_heads, step, cache, layer, "out"));
    const uint64_t pool = layer.block_stride * (uint64_t)cache->num_blocks, scratch = (uint64_t)kvm_attention_workspace(step);
    if (scratch > 0 && workspace && (!disjoint(workspace, scratch, cache->k, pool) || !disjoint(workspace, scratch, cache->v, pool)))
        return refuse(KVM_EINVAL, "the workspace and a pool share memory");
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
    KV_TRY(check_seal(step));
    if (!step->all_new) return refuse(KVM_EINVAL, "prompt attention is for sequences without earlier tokens");
    if (step->num_tokens == 0) return KVM_OK;
    KV_TRY(check_words(step, words, &device));
    KV_TRY(check_rows(k, "k", step->num_tokens, step->num_kv_heads, step, device));
    KV_TRY(check_rows(v, "v", step->num_tokens, step->num_kv_heads, step, device));
    const uint64_t size = (uint64_t)type_bytes(step->dtype);
    // the kernels step over 16 rows with 32-bit offsets
    if ((uint64_t)k->token_stride * size >= 1u << 28 || (uint64_t)v->token_stride * size >= 1u << 28)
        return refuse(KVM_EINVAL, "K and V rows 256 MiB apart or more are not supported");
    KV_TRY(check_rows(out, "out", step->num_tokens, step->num_heads, step, device));
    KV_TRY(check_clear(out, step->num_heads, k, step->num_kv_heads, step->num_tokens, step, "out and k"));
    KV_TRY(check_clear(out, step->num_heads, v, step->num_kv_heads, step->num_tokens, step, "out and v"));
    const uint64_t scratch = (uint64_t)kvm_attention_workspace(step);
    if (scratch > 0 && workspace) {
        KV_TRY(check_clear_of(k, step->num_tokens, step->num_kv_heads, step, workspace, scratch, "k and the workspace"));
        KV_TRY(check_clear_of(v, step->num_tokens, step->num_kv_heads, step, workspace, scratch, "v and the workspace"));
    }
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
