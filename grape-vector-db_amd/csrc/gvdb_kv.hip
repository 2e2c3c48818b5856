// gvdb_kv.hip — token cache: keys and values of a model's context, paged and
// held in 4 bits (the gvdb_kv_* entry points of include/gvdb.h).
//
//   k_kv_append : quantise new tokens into their pages, make the pages' key bounds new
//   k_kv_read   : the tokens' values, back in 16 or 32 bits
//   k_kv_attend : softmax attention over a sequence's tokens, or over chosen pages
//   k_kv_score / k_kv_select : the pages that promise each query the largest scores
//   k_kv_combine: joins the parts of a row whose keys were split over workgroups
//
// A tile is 32 tokens of one (page, head), 34 * D bytes:
//   key codes 16 D | key scales D | value codes 16 D | value scales D
// Scales are [D / 32][32 tokens] biased exponents; 255 marks a group that held
// a value that is not finite.  Codes lie in the order in which a wave's lanes
// take them as operands of v_mfma_f32_16x16x32_bf16, 16 bytes a lane at a time:
//   keys  : lane 16 q + m holds tokens 2m, 2m + 1, channels [q D/4, (q+1) D/4)
//   values: lane 16 q + l holds tokens 8q .. 8q + 7, channels [l D/16, (l+1) D/16)
// S^T = K Q^T leaves lane 16 q + n with tokens 8q + 2r + i of query row n, which
// is what O^T = V^T P^T wants of its second operand: the probabilities never
// leave their lane, and every lane keeps the statistics of one query row.
#include "gvdb_device.h"
#include "gvdb_kv.h"

namespace gvdb {
namespace {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -1e38f;  // running maximum before the first key: finite, so that -inf - m is -inf and not NaN
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float bits_f32(uint32_t u) { return __uint_as_float(u); }
__device__ __forceinline__ bf8 as_bf8(u4 v) { return __builtin_bit_cast(bf8, v); }

// Two floats rounded to bf16 (nearest even), packed.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    bf2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float low_bf16(uint32_t u) { return bits_f32(u << 16); }
__device__ __forceinline__ float high_bf16(uint32_t u) { return bits_f32(u & 0xFFFF0000u); }

// A pair of floats as a sum of NP pairs of bf16: 8, 16 or 24 bits of each.
template <int NP>
__device__ __forceinline__ void pack_pieces(float a, float b, uint32_t (&out)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        out[p] = pack_bf16(a, b);
        if (p + 1 < NP) {
            a -= low_bf16(out[p]);
            b -= high_bf16(out[p]);
        }
    }
}

// Largest value over the four lanes that hold one query row (n, n + 16, n + 32, n + 48).
__device__ __forceinline__ float row_max(float v) {
    u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(bits_f32(r[0]), bits_f32(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = bits_f32(r[0]) + bits_f32(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return bits_f32(r[0]) + bits_f32(r[1]);
}

// ---- elements of the caller's tensors ---------------------------------------------------
// Eight neighbouring elements as floats; `wide`: the tensor's base and strides are multiples of 16 bytes.
template <int T>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool wide, float (&x)[8]) {
    if constexpr (T == GVDB_F32) {
        const float* p = (const float*)base + at;
        if (wide) {
            const f4 a = *(const f4*)p, b = *(const f4*)(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    } else {
        const uint16_t* p = (const uint16_t*)base + at;
        uint16_t h[8];
        if (wide) {
            const u4 a = *(const u4*)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) h[2 * i] = (uint16_t)a[i], h[2 * i + 1] = (uint16_t)(a[i] >> 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = T == GVDB_BF16 ? bits_f32((uint32_t)h[i] << 16) : (float)__builtin_bit_cast(_Float16, h[i]);
    }
}

// Eight neighbouring elements, each rounded once.
template <int T>
__device__ __forceinline__ void store8(void* base, int64_t at, bool wide, const float (&x)[8]) {
    if constexpr (T == GVDB_F32) {
        float* p = (float*)base + at;
        if (wide) {
            *(f4*)p = f4{x[0], x[1], x[2], x[3]};
            *(f4*)(p + 4) = f4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = x[i];
        }
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == GVDB_BF16) {
                h[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            } else {
                h[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) |
                       (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16;
            }
        }
        uint16_t* p = (uint16_t*)base + at;
        if (wide) {
            *(u4*)p = u4{h[0], h[1], h[2], h[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(h[i / 2] >> (i % 2 * 16));
        }
    }
}

// ---- the batch --------------------------------------------------------------------------
// Sequence b's rows, held inside the tensors whatever `cu` says.
__device__ __forceinline__ void seq_rows(const KvBatch& bt, uint32_t b, int& r0, int& n) {
    if (bt.cu) {
        r0 = min(max(bt.cu[b], 0), (int)bt.rows);
        n = min(max(bt.cu[b + 1], r0), (int)bt.rows) - r0;
    } else {
        n = (int)(bt.rows / bt.n_seqs);
        r0 = (int)b * n;
    }
}

// Page of the j-th page of sequence b; -1: outside the table or the pool.
__device__ __forceinline__ int64_t page_of(const KvCache& c, const KvBatch& bt, uint32_t b, uint32_t j) {
    if (j >= bt.table_width) return -1;
    const int64_t p = bt.table[(uint64_t)b * bt.table_stride + j];
    return p >= 0 && (uint64_t)p < c.n_pages ? p : -1;
}

template <int D>
__device__ __forceinline__ uint64_t tile_at(const KvCache& c, int64_t page, uint32_t h, uint32_t tile) {
    return (((uint64_t)page * c.heads + h) * (c.page >> 5) + tile) * (uint64_t)(34 * D);
}

// Byte 4 * o of token t's key codes, and of its value codes (D = 64: two halves, each 16 bits).
template <int D>
__device__ __forceinline__ uint32_t key_byte(uint32_t t, uint32_t o) {
    const uint32_t b = 4 * o, at = (t & 1) * (D / 8) + b % (D / 8);
    return (at / 16 * 64 + b / (D / 8) * 16 + t / 2) * 16 + at % 16;
}
template <int D>
__device__ __forceinline__ uint32_t value_byte(uint32_t t, uint32_t b) {
    const uint32_t at = (t & 7) * (D / 32) + b % (D / 32);
    return (at / 16 * 64 + t / 8 * 16 + b / (D / 32)) * 16 + at % 16;
}

// Eight codes as the values that they stand for.
__device__ __forceinline__ void code_values(uint32_t w, uint32_t scale, float (&x)[8]) {
    const float s = scale == 255u ? __builtin_nanf("") : bits_f32(scale << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = (w >> (4 * i)) & 15u;
        // e2m1: subnormal 0, .5, then (2 + m) * 2^(e - 2)
        const uint32_t e = (c >> 1) & 3u, m = c & 1u;
        const float v = e == 0 ? 0.5f * (float)m : bits_f32(((e + 126u) << 23) | (m << 22));
        x[i] = ((c & 8u) ? -v : v) * s;
    }
}

// ---- append -----------------------------------------------------------------------------
// One workgroup a touched page, head and part (keys, values).  D / 8 threads take a token, eight channels
// each; four neighbours share a scale.  Bound by the reads of k and v.
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_append(KvCache c, KvBatch bt, KvRows k, KvRows v, uint32_t slots) {
    constexpr uint32_t TPT = D / 8;       // threads a token
    constexpr uint32_t TPB = 256 / TPT;   // tokens a pass
    __shared__ float s_hi[TPB][D], s_lo[TPB][D];
    __shared__ uint32_t s_bad, s_exp;
    const uint32_t b = blockIdx.x / slots, part = blockIdx.y & 1u, h = blockIdx.y >> 1;
    const uint32_t o = threadIdx.x % TPT, lane_t = threadIdx.x / TPT;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t start = max(bt.lengths[b], 0), end = start + n;
    const KvRows src = part ? v : k;
    for (int64_t pj = start / c.page + blockIdx.x % slots; n > 0 && pj * c.page < end; pj += slots) {
        const int64_t page = pj < (int64_t)bt.table_width ? page_of(c, bt, b, (uint32_t)pj) : -1;
        if (page < 0) continue;  // the same for the whole workgroup
        const int64_t p0 = pj * c.page;
        const uint32_t lo_t = (uint32_t)max(start - p0, (int64_t)0), hi_t = (uint32_t)min(end - p0, (int64_t)c.page);
        float hi[8], lo[8];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
        // tokens that the page holds already count for its bounds; values have none
        for (uint32_t t = (part ? lo_t / TPB * TPB : 0) + lane_t; t < hi_t; t += TPB) {
            uint8_t* tile = c.pool + tile_at<D>(c, page, h, t >> 5) + part * (17 * D);
            const uint32_t t5 = t & 31u, g = o / 4;
            uint8_t* scales = tile + 16 * D + g * 32 + t5;
            float x[8];
            if (t < lo_t) {
                if (part) continue;
                const uint32_t w = *(const uint32_t*)(tile + key_byte<D>(t5, o));
                const uint32_t s = *scales;
                bad |= s == 255u;
                code_values(w, s, x);
            } else {
                load8<T>(src.p, (r0 + (p0 + t - start)) * src.row_stride + (int64_t)h * src.head_stride + 8 * o, src.wide, x);
                uint32_t amax = 0;  // magnitudes order as their bits do; NaN is the largest
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7FFFFFFFu);
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1));
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2));
                // 2^e, the smallest with amax < 7 * 2^e: the fraction's .75 carries into the exponent
                uint32_t s = (amax + 0x200000u) >> 23;
                s = min(max(s, 4u) - 2u, 252u);
                const bool inf = amax >= 0x7F800000u;
                const float up = bits_f32((254u - s) << 23);  // 2^(127 - s), exact
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = fabsf(x[i]) * up;
                    uint32_t code = (uint32_t)(y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) +
                                    (y >= 3.5f) + (y > 5.0f);
                    code |= x[i] < 0.0f ? 8u : 0u;
                    w |= code << (4 * i);
                }
                if (inf) w = 0, s = 255u;
                bad |= inf;
                if (part == 0) {
                    *(uint32_t*)(tile + key_byte<D>(t5, o)) = w;
                } else if constexpr (D == 64) {
                    *(uint16_t*)(tile + value_byte<D>(t5, 4 * o)) = (uint16_t)w;
                    *(uint16_t*)(tile + value_byte<D>(t5, 4 * o + 2)) = (uint16_t)(w >> 16);
                } else {
                    *(uint32_t*)(tile + value_byte<D>(t5, 4 * o)) = w;
                }
                if ((o & 3u) == 0) *scales = (uint8_t)s;
                if (part) continue;
                code_values(w, s, x);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) hi[i] = fmaxf(hi[i], x[i]), lo[i] = fminf(lo[i], x[i]);
        }
        if (part) continue;
        // the page's bounds: over the passes' threads, then one power of two for all channels
        if (threadIdx.x == 0) s_bad = 0, s_exp = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s_hi[lane_t][8 * o + i] = hi[i], s_lo[lane_t][8 * o + i] = lo[i];
        __syncthreads();
        if (bad) s_bad = 1;
        const uint32_t d = threadIdx.x;
        float h1 = -INFINITY, l1 = INFINITY;
        if (d < D) {
            for (uint32_t i = 0; i < TPB; ++i) h1 = fmaxf(h1, s_hi[i][d]), l1 = fminf(l1, s_lo[i][d]);
            atomicMax(&s_exp, __float_as_uint(fmaxf(fabsf(h1), fabsf(l1))));  // LDS; the largest, in any order
        }
        __syncthreads();
        if (d < D) {
            // 2^b, the smallest with amax <= 127 * 2^b (fractions over 127/128 carry), rounded outward
            const uint32_t e = s_bad ? 255u : min(max((s_exp + 0x1FFFFu) >> 23, 7u), 254u);
            const float up = bits_f32((260u - min(e, 254u)) << 23);  // 2^(133 - e)
            int8_t* q = c.bounds + ((uint64_t)page * c.heads + h) * (2 * D);
            q[d] = s_bad ? (int8_t)0 : (int8_t)ceilf(h1 * up);
            q[D + d] = s_bad ? (int8_t)0 : (int8_t)floorf(l1 * up);
            if (d == 0) c.bound_exps[(uint64_t)page * c.heads + h] = (uint8_t)e;
        }
        __syncthreads();
    }
}

// ---- read -------------------------------------------------------------------------------
// A thread takes eight channels of one token and head, keys and values.
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_read(KvCache c, KvBatch bt, KvRows k, KvRows v) {
    constexpr uint32_t TPT = D / 8;
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t o = at % TPT;
    const uint64_t rest = at / TPT;
    const uint32_t h = rest % c.heads;
    const uint64_t row = rest / c.heads;
    if (row >= bt.rows) return;
    uint32_t b;
    if (bt.cu) {  // the last sequence that begins at or before the row
        uint32_t lo = 0, hi = bt.n_seqs;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if ((int64_t)bt.cu[mid + 1] <= (int64_t)row) lo = mid + 1;
            else hi = mid;
        }
        b = lo;
        if (b >= bt.n_seqs) return;  // behind the last sequence: left as it was
    } else {
        b = (uint32_t)(row / (bt.rows / bt.n_seqs));
    }
    int r0, n;
    seq_rows(bt, b, r0, n);
    if ((int64_t)row < r0) return;
    const int64_t pos = (int64_t)max(bt.lengths[b], 0) + ((int64_t)row - r0);
    const int64_t pj = pos / c.page;
    const int64_t page = pj < (int64_t)bt.table_width ? page_of(c, bt, b, (uint32_t)pj) : -1;
    const uint32_t t = (uint32_t)(pos % c.page), t5 = t & 31u;
    float x[8], y[8];
    if (page < 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i] = __builtin_nanf("");
    } else {
        const uint8_t* tile = c.pool + tile_at<D>(c, page, h, t >> 5);
        code_values(*(const uint32_t*)(tile + key_byte<D>(t5, o)), tile[16 * D + o / 4 * 32 + t5], x);
        const uint8_t* tv = tile + 17 * D;
        uint32_t w;
        if constexpr (D == 64) {
            w = *(const uint16_t*)(tv + value_byte<D>(t5, 4 * o)) |
                (uint32_t) * (const uint16_t*)(tv + value_byte<D>(t5, 4 * o + 2)) << 16;
        } else {
            w = *(const uint32_t*)(tv + value_byte<D>(t5, 4 * o));
        }
        code_values(w, tv[16 * D + o / 4 * 32 + t5], y);
    }
    if (k.p) store8<T>(k.p, (int64_t)row * k.row_stride + (int64_t)h * k.head_stride + 8 * o, k.wide, x);
    if (v.p) store8<T>(v.p, (int64_t)row * v.row_stride + (int64_t)h * v.head_stride + 8 * o, v.wide, y);
}

// ---- attention: one wave's part of 16 query rows ---------------------------------------
template <int D>
struct Tile {  // what a lane holds of one tile
    u4 k[D / 64], v[D / 64];
    uint32_t ks[D == 256 ? 2 : 1];  // scales of tokens 2m, 2m + 1
    u2 vs;                          // scales of tokens 8q .. 8q + 7
};

template <int D>
__device__ __forceinline__ void load_tile(const uint8_t* p, uint32_t lane, Tile<D>& t) {
    const uint32_t q = lane >> 4, m = lane & 15u;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        t.k[i] = *(const u4*)(p + (i * 64 + lane) * 16);
        t.v[i] = *(const u4*)(p + 17 * D + (i * 64 + lane) * 16);
    }
    if constexpr (D == 256) {
        t.ks[0] = *(const uint16_t*)(p + 16 * D + (2 * q) * 32 + 2 * m);
        t.ks[1] = *(const uint16_t*)(p + 16 * D + (2 * q + 1) * 32 + 2 * m);
    } else {
        t.ks[0] = *(const uint16_t*)(p + 16 * D + (q * D / 128) * 32 + 2 * m);
    }
    t.vs = *(const u2*)(p + 33 * D + (m * D / 512) * 32 + 8 * q);
}

// A dword of eight codes as eight bf16, exactly: both have the sign, the scale is a power of two.
__device__ __forceinline__ u4 codes_bf16(uint32_t w, float s) {
    u4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    return r;
}
// Two codes (byte `b` of a lane's value codes) as bf16.
template <int N>
__device__ __forceinline__ uint32_t byte_bf16(const u4 (&v)[N], int b, float s) {
    const uint32_t w = v[b / 16][b / 4 % 4];
    switch (b % 4) {
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    }
}

// One wave's state: R tiles of 16 query rows, lane 16 q + n with row n of each.
template <int D, int NP, int R>
struct Rows {
    u4 qf[R][NP][D / 32];  // query pieces, as the second operand
    f4 o[R][D / 16];       // O^T: lane's channels q D/4 + r D/16 + j
    float m[R], l[R];      // largest exponent (base 2) of the row; this lane's share of the sum
};

// Scores of a tile, scaled to base 2: s[rt][i][r] of token 8q + 2r + i.
template <int D, int NP, int R>
__device__ __forceinline__ void tile_scores(const Rows<D, NP, R>& w, const Tile<D>& t, float c2, f4 (&s)[R][2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            const float sc = bits_f32((t.ks[D == 256 ? c / 4 : 0] >> (8 * i) & 255u) << 23);
            const int dw = i * (D / 32) + c;
            const bf8 a = as_bf8(codes_bf16(t.k[dw / 4][dw % 4], sc));
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, as_bf8(w.qf[r][p][c]), s[r][i], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[r][i][e] *= c2;
    }
}

// Scales of 255 mark groups that are not finite: the tile's scores of such keys become NaN.
template <int D, int R>
__device__ __forceinline__ void poison_scores(const Tile<D>& t, uint32_t lane, f4 (&s)[R][2]) {
    const uint32_t q = lane >> 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        bool bad = (t.ks[0] >> (8 * i) & 255u) == 255u;
        if constexpr (D == 256) bad |= (t.ks[1] >> (8 * i) & 255u) == 255u;
        // lane 16 q' + m says it of token 2m + i
        uint64_t b = __ballot(bad);
        b |= b >> 32;
        b |= b >> 16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (b >> (4 * q + e) & 1u) {
#pragma unroll
                for (int r = 0; r < R; ++r) s[r][i][e] = __builtin_nanf("");
            }
    }
}

// Adds a tile's values by the probabilities of its scores (already masked: -inf where a row does not see a token).
// `gone`: the tile's first token that no row sees (32: none); its scales are not read as numbers.
template <int D, int NP, int R>
__device__ __forceinline__ void tile_values(Rows<D, NP, R>& w, Tile<D>& t, f4 (&s)[R][2], uint32_t lane, int gone) {
    const uint32_t q = lane >> 4;
    u4 pf[R][NP];
    bool seen_bad = false;
    // scales of this lane's eight tokens
    float vs[8];
    uint32_t badbits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t b = t.vs[e / 4] >> (8 * (e % 4)) & 255u;
        if ((int)(8 * q + e) >= gone) b = 127u;
        if (b == 255u) badbits |= 1u << e, b = 127u;
        vs[e] = bits_f32(b << 23);
    }
    seen_bad = __ballot(badbits != 0) != 0;
    f4 count[R];
    if (seen_bad) {  // which rows see a value group that is not finite: a product of truth values
        u4 bf, sf;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            bf[r] = ((badbits >> (2 * r) & 1u) ? 0x3F80u : 0u) | ((badbits >> (2 * r + 1) & 1u) ? 0x3F800000u : 0u);
#pragma unroll
        for (int rt = 0; rt < R; ++rt) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sf[r] = (s[rt][0][r] != -INFINITY ? 0x3F80u : 0u) | (s[rt][1][r] != -INFINITY ? 0x3F800000u : 0u);
            count[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(bf), as_bf8(sf), f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        }
    }
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
        float top = w.m[rt];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, s[rt][i][e]);
        top = row_max(top);
        const float a = __builtin_amdgcn_exp2f(w.m[rt] - top);
        w.m[rt] = top;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(s[rt][0][e] - top), p1 = __builtin_amdgcn_exp2f(s[rt][1][e] - top);
            sum += p0 + p1;
            uint32_t pc[NP];
            pack_pieces<NP>(p0, p1, pc);
#pragma unroll
            for (int p = 0; p < NP; ++p) pf[rt][p][e] = pc[p];
        }
        w.l[rt] = w.l[rt] * a + sum;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) w.o[rt][j][e] *= a;
    }
#pragma unroll
    for (int jb = 0; jb < D / 32; ++jb) {  // two channels a byte
        u4 even, odd;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t a = byte_bf16<D / 64>(t.v, (2 * r) * (D / 32) + jb, vs[2 * r]);
            const uint32_t b = byte_bf16<D / 64>(t.v, (2 * r + 1) * (D / 32) + jb, vs[2 * r + 1]);
            even[r] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            odd[r] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                w.o[rt][2 * jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(even), as_bf8(pf[rt][p]), w.o[rt][2 * jb], 0, 0, 0);
                w.o[rt][2 * jb + 1] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(odd), as_bf8(pf[rt][p]), w.o[rt][2 * jb + 1], 0, 0, 0);
            }
    }
    if (seen_bad) {
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (count[rt][e] > 0.f) {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) w.o[rt][j][e] = __builtin_nanf("");
                }
    }
}

// Tiles that a query at `limit` visible tokens reads: one tile beyond the table stands for a length that the
// table does not cover, and poisons the row.
__device__ __forceinline__ uint32_t tiles_of(const KvCache& c, const KvBatch& bt, int64_t limit) {
    const int64_t have = (int64_t)bt.table_width * (c.page >> 5);
    const int64_t want = limit <= 0 ? 0 : (limit + 31) >> 5;
    return (uint32_t)min(want, have + 1);
}

// Query rows of a wave's 16-row tile: row n of the sequence is token n / group, head h * group + n % group.
struct QRow {
    int token;       // row of q; -1: none
    uint32_t head;
    int64_t limit;   // tokens that it sees
};

// ---- attend -----------------------------------------------------------------------------
// A workgroup takes 16 query rows of one sequence (CHOSEN: of one token) and key head and one split of the
// keys; its four waves take the split's tiles in turn, and join their parts through LDS.  With one query
// token a sequence the kernel reads each cached byte once: 34 D / 32 bytes a token and head bound it.
template <int D, int T, bool CHOSEN>
__global__ __launch_bounds__(256) void k_kv_attend(KvCache c, KvBatch bt, AttendArgs a) {
    constexpr int NP = T == GVDB_BF16 ? 1 : T == GVDB_F16 ? 2 : 3;
    __shared__ float s_o[4][16][D];
    __shared__ float s_m[4][16], s_l[4][16];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    const uint32_t h = blockIdx.x % c.heads, split = blockIdx.x / c.heads % a.splits;
    const uint32_t unit = blockIdx.x / c.heads / a.splits;  // (sequence, tile slot), or (token, tile slot)
    const uint32_t slot = unit % a.row_tiles;
    uint32_t b = unit / a.row_tiles;
    int r0, n;
    int chosen_row = 0;
    if constexpr (CHOSEN) {
        chosen_row = (int)b;
        if (!a.row_seq(bt, chosen_row, b)) return;
    }
    seq_rows(bt, b, r0, n);
    const int64_t len = max(bt.lengths[b], 0);
    const uint32_t group = a.q_heads / c.heads;
    const int rows_here = (CHOSEN ? 1 : n) * (int)group;
    const uint32_t per_page = c.page >> 5;
    for (int row_tile = (int)slot; row_tile * 16 < rows_here; row_tile += (int)a.row_tiles) {
        const int first = row_tile * 16;
        // this lane's row
        const int rr = first + (int)n16;
        QRow me;
        me.token = rr < rows_here ? (CHOSEN ? chosen_row : r0 + rr / (int)group) : -1;
        me.head = h * group + (uint32_t)rr % group;
        me.limit = me.token < 0 ? 0 : a.causal ? len - n + (me.token - r0) + 1 : len;
        const int last_token = CHOSEN ? chosen_row : r0 + min(first + 15, rows_here - 1) / (int)group;
        const int first_token = CHOSEN ? chosen_row : r0 + first / (int)group;
        const int64_t most = a.causal ? len - n + (last_token - r0) + 1 : len;    // of the tile's rows
        const int64_t least = a.causal ? len - n + (first_token - r0) + 1 : len;
        const int32_t* list = nullptr;
        uint32_t tiles;
        if constexpr (CHOSEN) {
            list = a.chosen + ((uint64_t)chosen_row * c.heads + h) * a.top;
            tiles = (uint32_t)min((int64_t)a.top, a.pages_seen(c, bt, most)) * per_page;
        } else {
            tiles = tiles_of(c, bt, most);
        }
        const uint32_t t0 = min(split * a.chunk, tiles), t1 = split + 1 == a.splits ? tiles : min(t0 + a.chunk, tiles);
        if (a.splits > 1 && t0 >= t1) continue;  // no part: k_kv_combine does not read it
        Rows<D, NP, 1> w;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) w.o[0][j] = f4{0.f, 0.f, 0.f, 0.f};
        w.m[0] = kLowest;
        w.l[0] = 0.f;
        if (t0 < t1) {
#pragma unroll
            for (int ch = 0; ch < D / 32; ++ch) {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (me.token >= 0)
                    load8<T>(a.q.p, (int64_t)me.token * a.q.row_stride + (int64_t)me.head * a.q.head_stride + q4 * (D / 4) + 8 * ch,
                             a.q.wide, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t pc[NP];
                    pack_pieces<NP>(x[2 * e], x[2 * e + 1], pc);
#pragma unroll
                    for (int p = 0; p < NP; ++p) w.qf[0][p][ch][e] = pc[p];
                }
            }
        }
        for (uint32_t t = t0 + wave; t < t1; t += 4) {
            uint32_t pj = t / per_page;
            if constexpr (CHOSEN) pj = (uint32_t)list[pj];
            const int64_t page = page_of(c, bt, b, pj);
            const int64_t base = (int64_t)pj * c.page + (t % per_page) * 32;
            if (CHOSEN && base >= most) continue;
            Tile<D> tl;
            load_tile<D>(c.pool + tile_at<D>(c, max(page, (int64_t)0), h, t % per_page), lane, tl);
            f4 s[1][2];
            tile_scores<D, NP, 1>(w, tl, a.scale_log2, s);
            bool bad = (tl.ks[0] & 255u) == 255u || (tl.ks[0] >> 8) == 255u;
            if constexpr (D == 256) bad |= (tl.ks[1] & 255u) == 255u || (tl.ks[1] >> 8) == 255u;
            if (__ballot(bad)) poison_scores<D, 1>(tl, lane, s);
            int gone = 32;
            if (page < 0) {
                gone = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) s[0][i] = f4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
            }
            if (base + 32 > least || me.token < 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (base + 8 * q4 + 2 * e + i >= me.limit) s[0][i][e] = -INFINITY;
                gone = (int)min((int64_t)gone, most - base);
            }
            tile_values<D, NP, 1>(w, tl, s, lane, gone);
        }
        // join the four waves
        w.l[0] = row_sum(w.l[0]);
        if (q4 == 0) s_m[wave][n16] = w.m[0], s_l[wave][n16] = w.l[0];
        __syncthreads();
        const float top = fmaxf(fmaxf(s_m[0][n16], s_m[1][n16]), fmaxf(s_m[2][n16], s_m[3][n16]));
        const float f = __builtin_amdgcn_exp2f(w.m[0] - top);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < D / 16; ++j) s_o[wave][n16][q4 * (D / 4) + r * (D / 16) + j] = w.o[0][j][r] * f;
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < 16 * (D / 8); e += 256) {
            const uint32_t r = e / (D / 8), d = e % (D / 8) * 8;
            const int row = first + (int)r;
            if (row >= rows_here) continue;
            const int token = CHOSEN ? chosen_row : r0 + row / (int)group;
            const uint32_t head = h * group + (uint32_t)row % group;
            const float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            float l = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) l += s_l[k][r] * __builtin_amdgcn_exp2f(s_m[k][r] - m);
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (s_o[0][r][d + i] + s_o[1][r][d + i]) + (s_o[2][r][d + i] + s_o[3][r][d + i]);
            const uint64_t at = (uint64_t)token * a.q_heads + head;
            if (a.splits > 1) {
                float* po = a.part_o + (at * a.splits + split) * D + d;
                *(f4*)po = f4{x[0], x[1], x[2], x[3]};
                *(f4*)(po + 4) = f4{x[4], x[5], x[6], x[7]};
                if (d == 0) *(f2*)(a.part_ml + (at * a.splits + split) * 2) = f2{m, l};
            } else {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= inv;
                store8<T>(a.out.p, (int64_t)token * a.out.row_stride + (int64_t)head * a.out.head_stride + d, a.out.wide, x);
                if (a.lse && d == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) / kLog2e;
            }
        }
        __syncthreads();
    }
}

// ---- combine ----------------------------------------------------------------------------
// D / 8 threads join one row's parts: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
template <int D, int T, bool CHOSEN>
__global__ __launch_bounds__(256) void k_kv_combine(KvCache c, KvBatch bt, AttendArgs a) {
    const uint64_t at = (uint64_t)blockIdx.x * (256 / (D / 8)) + threadIdx.x / (D / 8);
    const uint32_t d = threadIdx.x % (D / 8) * 8;
    if (at >= (uint64_t)bt.rows * a.q_heads) return;
    const int token = (int)(at / a.q_heads);
    const uint32_t head = at % a.q_heads;
    uint32_t b;
    if (!a.row_seq(bt, token, b)) return;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t len = max(bt.lengths[b], 0);
    const int64_t limit = a.causal ? len - n + (token - r0) + 1 : len;
    const uint32_t tiles = CHOSEN ? (uint32_t)min((int64_t)a.top, a.pages_seen(c, bt, limit)) * (c.page >> 5) : tiles_of(c, bt, limit);
    const uint32_t parts = min(a.splits, (tiles + a.chunk - 1) / a.chunk);
    float m = kLowest;
    for (uint32_t s = 0; s < parts; ++s) m = fmaxf(m, a.part_ml[(at * a.splits + s) * 2]);
    float l = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t s = 0; s < parts; ++s) {
        const f2 ml = *(const f2*)(a.part_ml + (at * a.splits + s) * 2);
        const float f = __builtin_amdgcn_exp2f(ml[0] - m);
        const float* po = a.part_o + (at * a.splits + s) * D + d;
        const f4 u = *(const f4*)po, v = *(const f4*)(po + 4);
        l += ml[1] * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += u[i] * f, x[4 + i] += v[i] * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
    store8<T>(a.out.p, (int64_t)token * a.out.row_stride + (int64_t)head * a.out.head_stride + d, a.out.wide, x);
    if (a.lse && d == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) / kLog2e;
}

// ---- which pages ------------------------------------------------------------------------
// Score of a page for a query head: 2^(a + b) * sum_d max(q8_d, 0) hi_d + min(q8_d, 0) lo_d with q8 = rint(q / 2^a) and the
// page's bounds hi, lo in units of 2^b.  The sum is a product of whole numbers over 2 D channels: v_mfma_i32_16x16x64_i8,
// exact in any order.  A wave scores 16 pages for 16 columns: `width` columns (a power of two) a token, the group's heads.
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_score(KvCache c, KvBatch bt, AttendArgs a, uint32_t tok_tiles, uint32_t chunks) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    const uint32_t h = blockIdx.x % c.heads, chunk = blockIdx.x / c.heads % chunks;
    const uint32_t unit = blockIdx.x / c.heads / chunks;
    const uint32_t b = unit / tok_tiles;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t len = max(bt.lengths[b], 0);
    const uint32_t group = a.q_heads / c.heads;
    const uint32_t width = min(16u, next_pow2(group)), per = 16 / width;
    for (int tt = (int)(unit % tok_tiles); tt * (int)per < n; tt += (int)tok_tiles) {
        const int tok = tt * (int)per + (int)(n16 / width);
        const bool live = tok < n;
        const int last = min(tt * (int)per + (int)per, n) - 1;
        const int64_t seen = min(a.pages_seen(c, bt, a.causal ? len - n + last + 1 : len), (int64_t)bt.table_width);
        if ((int64_t)chunk * a.score_chunk >= seen) continue;
        const int64_t p_end = chunk + 1 == chunks ? seen : min(seen, ((int64_t)chunk + 1) * a.score_chunk);
        for (int64_t p0 = (int64_t)chunk * a.score_chunk + wave * 16; p0 < p_end; p0 += 64) {
            const int64_t pm = p0 + n16;
            const int64_t page = pm < seen ? page_of(c, bt, b, (uint32_t)pm) : -1;
            u4 bd[D / 32];
            uint32_t e = 255u;
            const int8_t* row = c.bounds + ((uint64_t)max(page, (int64_t)0) * c.heads + h) * (2 * D);
#pragma unroll
            for (int k = 0; k < D / 32; ++k) bd[k] = *(const u4*)(row + k * 64 + q4 * 16);
            if (page >= 0) e = c.bound_exps[(uint64_t)page * c.heads + h];
            float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            for (uint32_t g0 = 0; g0 < group; g0 += width) {
                const uint32_t gh = g0 + n16 % width;
                const bool on = live && gh < group;
                float x[D / 64][16];
                uint32_t amax = 0;
#pragma unroll
                for (int k = 0; k < D / 64; ++k)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                        if (on)
                            load8<T>(a.q.p, (int64_t)(r0 + tok) * a.q.row_stride + (int64_t)(h * group + gh) * a.q.head_stride + k * 64 + q4 * 16 + half * 8,
                                     a.q.wide, y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[k][half * 8 + i] = y[i];
                            amax = max(amax, __float_as_uint(y[i]) & 0x7FFFFFFFu);
                        }
                    }
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
                const uint32_t qe = min(max((amax + 0x1FFFFu) >> 23, 7u), 255u);
                const float up = amax >= 0x7F800000u ? 0.f : bits_f32((260u - qe) << 23);
                i4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < D / 64; ++k) {
                    u4 pos, neg;
#pragma unroll
                    for (int wd = 0; wd < 4; ++wd) {
                        uint32_t pp = 0, nn = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int v = amax >= 0x7F800000u ? 0 : (int)rintf(x[k][wd * 4 + i] * up);
                            pp |= (uint32_t)(max(v, 0) & 255) << (8 * i);
                            nn |= (uint32_t)(min(v, 0) & 255) << (8 * i);
                        }
                        pos[wd] = pp, neg[wd] = nn;
                    }
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, bd[k]), __builtin_bit_cast(i4, pos), acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, bd[D / 64 + k]), __builtin_bit_cast(i4, neg), acc, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t be = (uint32_t)__shfl((int)e, 4 * (int)q4 + r);
                    const int ex = min(max((int)qe + (int)be - 266, -126), 127);
                    float sc = on ? (float)acc[r] * bits_f32((uint32_t)(ex + 127) << 23) : -INFINITY;
                    for (uint32_t x2 = 1; x2 < width; x2 <<= 1) sc = fmaxf(sc, __shfl_xor(sc, (int)x2));
                    best[r] = be == 255u ? 3.402823466e38f : fmaxf(best[r], sc);
                }
            }
            if (live && n16 % width == 0) {
                float* out = a.scores + ((uint64_t)(r0 + tok) * c.heads + h) * bt.table_width + p0 + 4 * q4;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (p0 + 4 * q4 + r < seen) out[r] = best[r];
            }
        }
    }
}

// The `top` pages of one token and key head: the first and the most recent ones, then the largest scores, the
// lowest page among equals; written in order, -1 behind the last.  Four passes over the scores find the
// top-th largest key eight bits at a time.
__global__ __launch_bounds__(256) void k_kv_select(KvCache c, KvBatch bt, AttendArgs a) {
    __shared__ uint32_t hist[256], wsum[4], s_digit, s_above;
    const uint32_t h = blockIdx.x % c.heads;
    const int token = (int)(blockIdx.x / c.heads);
    uint32_t b;
    if (!a.row_seq(bt, token, b)) return;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t len = max(bt.lengths[b], 0);
    const int64_t seen = a.pages_seen(c, bt, a.causal ? len - n + (token - r0) + 1 : len);
    int32_t* out = a.chosen + ((uint64_t)token * c.heads + h) * a.top;
    if (seen <= (int64_t)a.top) {
        for (uint32_t i = threadIdx.x; i < a.top; i += 256) out[i] = (int64_t)i < seen ? (int32_t)i : -1;
        return;
    }
    const float* sc = a.scores + ((uint64_t)token * c.heads + h) * bt.table_width;
    auto key = [&](uint32_t j) -> uint32_t {
        if (j < a.first || (int64_t)j >= seen - (int64_t)a.recent || j >= bt.table_width) return 0xFFFFFFFFu;
        return f32_order(sc[j]);
    };
    const uint32_t N = (uint32_t)seen;
    uint32_t prefix = 0, mask = 0, want = a.top;  // the want-th largest among keys with this prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < N; j += 256) {
            const uint32_t k = key(j);
            if ((k & mask) == prefix) atomicAdd(&hist[255u - (k >> shift & 255u)], 1u);  // LDS counts: any order
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const uint32_t t = wave_find_cum(hist, 256, want);
            const uint32_t above = wave_sum_below(hist, t);
            if (threadIdx.x == 0) s_digit = 255u - t, s_above = above;
        }
        __syncthreads();
        prefix |= s_digit << shift;
        mask |= 255u << shift;
        want -= s_above;
        __syncthreads();
    }
    // keys over the found one, and the first `want` that equal it, in page order
    uint32_t put = 0, ties = 0;
    for (uint32_t j0 = 0; j0 < N; j0 += 256) {
        const uint32_t j = j0 + threadIdx.x;
        const uint32_t k = j < N ? key(j) : 0u;
        const bool over = j < N && k > prefix, same = j < N && k == prefix;
        uint32_t tot_same, tot;
        const uint32_t before = big_prefix(same, wsum, &tot_same);
        const bool take = over || (same && ties + before < want);
        const uint32_t at = big_prefix(take, wsum, &tot);
        if (take && put + at < a.top) out[put + at] = (int32_t)j;
        put += tot;
        ties += tot_same;
    }
}

}  // namespace

// ---- launches -----------------------------------------------------------------------------
#define KV_DT(D_, T_, body)          \
    {                                \
        constexpr int D = D_, T = T_; \
        body;                        \
    }
#define KV_T(D_, dtype, body)                                  \
    switch (dtype) {                                           \
        case GVDB_F32: KV_DT(D_, GVDB_F32, body) break;        \
        case GVDB_F16: KV_DT(D_, GVDB_F16, body) break;        \
        default: KV_DT(D_, GVDB_BF16, body) break;             \
    }
#define KV_DISPATCH(dim, dtype, body)            \
    switch (dim) {                               \
        case 64: KV_T(64, dtype, body) break;    \
        case 128: KV_T(128, dtype, body) break;  \
        default: KV_T(256, dtype, body) break;   \
    }

namespace {
// Most `n` (at least 1) with n * others blocks near `cap`: the kernels stride over what is left.
uint32_t capped(uint64_t n, uint64_t others, uint64_t cap) {
    const uint64_t most = cap / others + 1;
    return (uint32_t)(n < 1 ? 1 : n > most ? most : n);
}
bool fits(uint64_t blocks) { return blocks > 0 && blocks <= 0x7FFFFFFFull; }
}  // namespace

hipError_t launch_kv_append(const KvCache& c, const KvBatch& bt, const KvRows& k, const KvRows& v, hipStream_t s) {
    const uint32_t slots = capped(((uint64_t)bt.max_new + c.page - 2) / c.page + 1, bt.n_seqs, 1u << 22);
    if (!fits((uint64_t)bt.n_seqs * slots)) return hipErrorInvalidValue;
    const dim3 grid(bt.n_seqs * slots, 2 * c.heads);
    KV_DISPATCH(c.dim, k.dtype, (k_kv_append<D, T><<<grid, 256, 0, s>>>(c, bt, k, v, slots)));
    GVDB_LAUNCH_CHECK();
    return hipSuccess;
}

hipError_t launch_kv_read(const KvCache& c, const KvBatch& bt, const KvRows& k, const KvRows& v, hipStream_t s) {
    const uint64_t blocks = ((uint64_t)bt.rows * c.heads * (c.dim / 8) + 255) / 256;
    if (!fits(blocks)) return hipErrorInvalidValue;
    const uint32_t dtype = k.p ? k.dtype : v.dtype;
    KV_DISPATCH(c.dim, dtype, (k_kv_read<D, T><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, k, v)));
    GVDB_LAUNCH_CHECK();
    return hipSuccess;
}

hipError_t launch_kv_attend(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s) {
    const uint64_t blocks = (uint64_t)c.heads * a.splits * a.row_tiles * bt.n_seqs;
    const uint32_t per = 256 / (c.dim / 8);
    const uint64_t joins = ((uint64_t)bt.rows * a.q_heads + per - 1) / per;
    if (!fits(blocks) || !fits(joins)) return hipErrorInvalidValue;
    KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend<D, T, false><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    GVDB_LAUNCH_CHECK();
    if (a.splits > 1) {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_combine<D, T, false><<<(uint32_t)joins, 256, 0, s>>>(c, bt, a)));
        GVDB_LAUNCH_CHECK();
    }
    return hipSuccess;
}

hipError_t launch_kv_attend_topk(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s) {
    const uint32_t group = a.q_heads / c.heads;
    const uint32_t per = 16 / (group >= 16 ? 16 : next_pow2(group));
    const uint32_t chunks = (kv_max_pages(c, bt) + a.score_chunk - 1) / a.score_chunk;
    const uint64_t others = (uint64_t)c.heads * chunks * bt.n_seqs;
    const uint32_t tok_tiles = capped(((uint64_t)bt.max_new + per - 1) / per, others, 1u << 22);
    const uint64_t blocks = (uint64_t)c.heads * a.splits * a.row_tiles * bt.rows;
    const uint32_t pb = 256 / (c.dim / 8);
    const uint64_t joins = ((uint64_t)bt.rows * a.q_heads + pb - 1) / pb;
    if (!fits(others * tok_tiles) || !fits(blocks) || !fits(joins) || !fits((uint64_t)bt.rows * c.heads)) return hipErrorInvalidValue;
    KV_DISPATCH(c.dim, a.q.dtype, (k_kv_score<D, T><<<(uint32_t)(others * tok_tiles), 256, 0, s>>>(c, bt, a, tok_tiles, chunks)));
    GVDB_LAUNCH_CHECK();
    k_kv_select<<<bt.rows * c.heads, 256, 0, s>>>(c, bt, a);
    GVDB_LAUNCH_CHECK();
    KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend<D, T, true><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    GVDB_LAUNCH_CHECK();
    if (a.splits > 1) {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_combine<D, T, true><<<(uint32_t)joins, 256, 0, s>>>(c, bt, a)));
        GVDB_LAUNCH_CHECK();
    }
    return hipSuccess;
}

}  // namespace gvdb
