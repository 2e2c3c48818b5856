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
#include <algorithm>

#include "gvdb_device.h"
#include "gvdb_kv.h"

namespace gvdb {
namespace {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -3e38f;  // running maximum before the first key: finite, so that -inf - m is -inf and not NaN
// Pieces of 8 bits that a type's values are split into for the products.
constexpr int pieces(int dtype) { return dtype == GVDB_BF16 ? 1 : dtype == GVDB_F16 ? 2 : 3; }
// Pieces of a probability, on every path alike: 16 bits for rows of 16 bits, 24 for those of 32.  Rows of 16 bits are as far from 64 bits
// as with 32 (0.0017 relative in bf16, 0.00021 in f16, an output's own rounding); with one piece for bf16 rows 0.0023 by 128 rows, and
// the size of a launch would decide how many bits a row gets.
template <int NP>
constexpr int kProbPieces = NP < 2 ? 2 : NP;
// The value, as one that the compiler knows nothing of: what is reckoned from it in a branch that is seldom taken stays in
// that branch, and takes no registers outside.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
template <int V>
struct Const {
    static constexpr int value = V;
};
// A row's sums are rescaled only when a score passes the reference by so much (base 2): probabilities reach 2^8 instead of 1,
// which no rounding notices, and a new largest score, which some row of a wave has in half of all steps, seldom costs anything.
constexpr float kSlack = 8.f;
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

// A pair of bf16 whose infinities become NaN: a query's infinity times keys of one sign would be scores of -inf, which read as masked.
// (In more pieces the second is inf - inf.)
__device__ __forceinline__ uint32_t inf_to_nan(uint32_t w) { return w | ((w & 0x7F807F80u) + 0x00800080u & 0x80008000u) >> 9; }

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
    const float s = bits_f32(scale << 23);
    const f2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const f2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    const bool bad = scale == 255u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[i] = bad ? __builtin_nanf("") : v0[i], x[2 + i] = bad ? __builtin_nanf("") : v1[i];
        x[4 + i] = bad ? __builtin_nanf("") : v2[i], x[6 + i] = bad ? __builtin_nanf("") : v3[i];
    }
}

// Largest over the lanes that differ in their lowest two bits, and over a wave.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    x = max(x, dpp<0xB1>(x));
    return max(x, dpp<0x4E>(x));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = quad_max(x);
    x = max(x, dpp<0x141>(x));
    x = max(x, dpp<0x140>(x));
    u2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(r[0], r[1]);
}

// Eight neighbouring elements as they lie in memory.
template <int T>
struct Raw8 {
    u4 r[T == GVDB_F32 ? 2 : 1];

    __device__ __forceinline__ void load(const void* base, int64_t at, bool wide) {
        constexpr int N = T == GVDB_F32 ? 2 : 1;
        if (wide) {
            const u4* p = (const u4*)((const char*)base + at * (T == GVDB_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = p[i];
        } else if constexpr (T == GVDB_F32) {
            const uint32_t* p = (const uint32_t*)base + at;
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i / 4][i % 4] = p[i];
        } else {
            const uint16_t* p = (const uint16_t*)base + at;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[0][i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
    }
    // The largest magnitude's bits as a float's: magnitudes order as their bits do, NaN above all.
    __device__ __forceinline__ uint32_t amax() const {
        if constexpr (T == GVDB_F32) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, r[i / 4][i % 4] & 0x7FFFFFFFu);
            return m;
        } else {
            us2 m = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, r[0][i] & 0x7FFF7FFFu));
            const uint16_t x = max(m[0], m[1]);
            return T == GVDB_BF16 ? (uint32_t)x << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, x));
        }
    }
    // The codes at 2^(scale - 127): the conversion rounds to nearest, ties to the even code.
    __device__ __forceinline__ uint32_t codes(uint32_t scale) const {
        const float s = bits_f32(scale << 23);
        uint32_t w = 0;
        const uint32_t x0 = r[0][0], x1 = r[0][1], x2 = r[0][2], x3 = r[0][3];  // a bit cast of a vector's element reads its first
        if constexpr (T == GVDB_F32) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, bits_f32(x0), bits_f32(x1), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, bits_f32(x2), bits_f32(x3), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, bits_f32(r[1][0]), bits_f32(r[1][1]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, bits_f32(r[1][2]), bits_f32(r[1][3]), s, 3);
        } else if constexpr (T == GVDB_F16) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h2, x0), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h2, x1), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h2, x2), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h2, x3), s, 3);
        } else {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x0), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x1), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x2), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x3), s, 3);
        }
        return w;
    }
};

// ---- append -----------------------------------------------------------------------------
// One workgroup a touched page, head and part (keys, values).  D / 8 threads take a token, eight channels each; four neighbours
// share a scale.  Four passes' loads are in flight at once.  Where there are many tokens (16384 of 8 heads of 128 channels, bf16: 28 us,
// 3.0 TB/s read and written) bound by the reads of k and v and by what lies between them: nothing is in flight while a page's bounds are
// reckoned.  Where there is one, by its chain of loads (length, page, rows and the codes that the page's bounds go over): 64 sequences'
// next tokens 8 us.
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_append(KvCache c, KvBatch bt, KvRows k, KvRows v, uint32_t slots) {
    constexpr uint32_t TPT = D / 8;       // threads a token
    constexpr uint32_t TPB = 256 / TPT;   // tokens a pass
    constexpr int AHEAD = 4;
    __shared__ float s_hi[4][D], s_lo[4][D];
    __shared__ uint32_t s_bad[4], s_amax[4];
    const uint32_t b = blockIdx.x / slots, part = blockIdx.y & 1u, h = blockIdx.y >> 1;
    const uint32_t o = threadIdx.x % TPT, lane_t = threadIdx.x / TPT, wave = threadIdx.x >> 6;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t start = max(bt.lengths[b], 0), end = start + n;
    const KvRows src = part ? v : k;
    for (int64_t pj = start / c.page + blockIdx.x % slots; n > 0 && pj * c.page < end; pj += slots) {
        const int64_t page = pj < (int64_t)bt.table_width ? page_of(c, bt, b, (uint32_t)pj) : -1;
        if (page < 0) continue;  // the same for the whole workgroup
        const int64_t p0 = pj * c.page;
        const uint32_t lo_t = (uint32_t)max(start - p0, (int64_t)0), hi_t = (uint32_t)min(end - p0, (int64_t)c.page);
        uint8_t* const tiles = c.pool + tile_at<D>(c, page, h, 0) + part * (17 * D);
        auto code_at = [&](uint32_t t) { return tiles + (t >> 5) * (34 * D) + (part ? value_byte<D>(t & 31u, 4 * o) : key_byte<D>(t & 31u, o)); };
        auto scale_at = [&](uint32_t t) { return tiles + (t >> 5) * (34 * D) + 16 * D + o / 4 * 32 + (t & 31u); };
        float hi[8], lo[8];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
        // tokens that the page holds already count for its bounds; values have none
        for (uint32_t first = (part ? lo_t / TPB * TPB : 0) + lane_t; first < hi_t; first += AHEAD * TPB) {
            Raw8<T> raw[AHEAD];
            uint32_t w[AHEAD], s[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t t = first + i * TPB;
                w[i] = s[i] = 0;
                if (t >= hi_t) continue;
                if (t >= lo_t) {
                    raw[i].load(src.p, (r0 + (p0 + t - start)) * src.row_stride + (int64_t)h * src.head_stride + 8 * o, src.wide);
                } else if (!part) {
                    w[i] = *(const uint32_t*)code_at(t);
                    s[i] = *scale_at(t);
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t t = first + i * TPB;
                if (t >= hi_t || (part && t < lo_t)) continue;
                if (t >= lo_t) {
                    const uint32_t amax = quad_max(raw[i].amax());
                    // 2^e, the smallest with amax < 7 * 2^e: the fraction's .75 carries into the exponent
                    s[i] = min(max((amax + 0x200000u) >> 23, 4u) - 2u, 252u);
                    w[i] = raw[i].codes(s[i]);
                    if (amax >= 0x7F800000u) w[i] = 0, s[i] = 255u;
                    uint8_t* to = code_at(t);
                    if (D == 64 && part) {
                        *(uint16_t*)to = (uint16_t)w[i];
                        *(uint16_t*)(tiles + (t >> 5) * (34 * D) + value_byte<D>(t & 31u, 4 * o + 2)) = (uint16_t)(w[i] >> 16);
                    } else {
                        *(uint32_t*)to = w[i];
                    }
                    if ((o & 3u) == 0) *scale_at(t) = (uint8_t)s[i];
                    if (part) continue;
                }
                bad |= s[i] == 255u;
                float x[8];
                code_values(w[i], s[i], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) hi[e] = fmaxf(hi[e], x[e]), lo[e] = fminf(lo[e], x[e]);
            }
        }
        if (part) continue;
        // the page's bounds: over the wave's tokens, the waves, then one power of two for all channels
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (D == 64) {  // a rotation by 8 of 16 lanes
                hi[e] = fmaxf(hi[e], bits_f32(dpp<0x128>(__float_as_uint(hi[e]))));
                lo[e] = fminf(lo[e], bits_f32(dpp<0x128>(__float_as_uint(lo[e]))));
            }
            if constexpr (D <= 128) {
                u2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(hi[e]), __float_as_uint(hi[e]), false, false);
                hi[e] = fmaxf(bits_f32(r[0]), bits_f32(r[1]));
                r = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo[e]), __float_as_uint(lo[e]), false, false);
                lo[e] = fminf(bits_f32(r[0]), bits_f32(r[1]));
            }
            u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(hi[e]), __float_as_uint(hi[e]), false, false);
            hi[e] = fmaxf(bits_f32(r[0]), bits_f32(r[1]));
            r = __builtin_amdgcn_permlane32_swap(__float_as_uint(lo[e]), __float_as_uint(lo[e]), false, false);
            lo[e] = fminf(bits_f32(r[0]), bits_f32(r[1]));
        }
        const uint64_t any_bad = __ballot(bad);
        if ((threadIdx.x & 63u) < TPT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s_hi[wave][8 * o + e] = hi[e], s_lo[wave][8 * o + e] = lo[e];
        }
        if ((threadIdx.x & 63u) == 0) s_bad[wave] = any_bad != 0;
        __syncthreads();
        const uint32_t d = threadIdx.x;
        float h1 = 0.f, l1 = 0.f;
        if (d < D) {
            h1 = fmaxf(fmaxf(s_hi[0][d], s_hi[1][d]), fmaxf(s_hi[2][d], s_hi[3][d]));
            l1 = fminf(fminf(s_lo[0][d], s_lo[1][d]), fminf(s_lo[2][d], s_lo[3][d]));
        }
        const uint32_t wm = wave_max(__float_as_uint(fmaxf(fabsf(h1), fabsf(l1))));
        if ((threadIdx.x & 63u) == 0) s_amax[wave] = wm;
        __syncthreads();
        if (d < D) {
            const bool any = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
            const uint32_t amax = max(max(s_amax[0], s_amax[1]), max(s_amax[2], s_amax[3]));
            // 2^b, the smallest with amax <= 127 * 2^b (fractions over 127/128 carry), rounded outward
            const uint32_t e = any ? 255u : min(max((amax + 0x1FFFFu) >> 23, 7u), 254u);
            const float up = bits_f32((260u - min(e, 254u)) << 23);  // 2^(133 - e)
            int8_t* q = c.bounds + ((uint64_t)page * c.heads + h) * (2 * D);
            // a product too small for a float is 0, which bounds nothing: outward of it is a step
            q[d] = any ? (int8_t)0 : (int8_t)fmaxf(ceilf(h1 * up), h1 > 0.f ? 1.f : -127.f);
            q[D + d] = any ? (int8_t)0 : (int8_t)fminf(floorf(l1 * up), l1 < 0.f ? -1.f : 127.f);
            if (d == 0) c.bound_exps[(uint64_t)page * c.heads + h] = (uint8_t)e;
        }
        __syncthreads();
    }
}

// ---- read -------------------------------------------------------------------------------
// A thread takes eight channels of one token and head, keys and values; a workgroup several tokens of one head, whose codes lie
// side by side.  Bound by what it writes (the same 16384 tokens: 18.5 us, 4.6 TB/s).
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_read(KvCache c, KvBatch bt, KvRows k, KvRows v) {
    constexpr uint32_t TPT = D / 8;
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t o = at % TPT;
    constexpr uint32_t TPB = 256 / TPT;
    const uint64_t rest = at / 256;
    const uint32_t h = rest % c.heads;
    const uint64_t row = rest / c.heads * TPB + at % 256 / TPT;
    if (row >= bt.rows) return;
    uint32_t b;
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto rest_of = [&](const KvRows& r) {  // behind the last sequence: left as it was, or 0
        if (r.p && r.zero_rest) store8<T>(r.p, (int64_t)row * r.row_stride + (int64_t)h * r.head_stride + 8 * o, r.wide, zero);
    };
    if (bt.cu) {  // the last sequence that begins at or before the row
        uint32_t lo = 0, hi = bt.n_seqs;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if ((int64_t)bt.cu[mid + 1] <= (int64_t)row) lo = mid + 1;
            else hi = mid;
        }
        b = lo;
        if (b >= bt.n_seqs) {
            rest_of(k), rest_of(v);
            return;
        }
    } else {
        b = (uint32_t)(row / (bt.rows / bt.n_seqs));
    }
    int r0, n;
    seq_rows(bt, b, r0, n);
    if ((int64_t)row < r0) {
        rest_of(k), rest_of(v);
        return;
    }
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

// Tiles that a query at `limit` visible tokens reads: one tile beyond the table stands for a length that the
// table does not cover, and poisons the row.
__device__ __forceinline__ uint32_t tiles_of(const KvCache& c, const KvBatch& bt, int64_t limit) {
    const int64_t have = (int64_t)bt.table_width * (c.page >> 5);
    const int64_t want = limit <= 0 ? 0 : (limit + 31) >> 5;
    return (uint32_t)min(want, have + 1);
}

// 16 query rows of a unit (a sequence; CHOSEN: one token) and key head.
template <bool CHOSEN>
struct Job {
    uint32_t b, h, group;
    int r0, n, first, rows;  // the sequence's rows of q; the first row of the 16 and the unit's rows, counted over the group's heads
    int unit;
    int64_t most, least;     // tokens that the last and the first of the 16 see
    // this lane's row
    int token;               // row of q; -1: none
    uint32_t head;
    int64_t limit;           // tokens that it sees

    // false: no sequence has the unit
    __device__ __forceinline__ bool set(const KvCache& c, const KvBatch& bt, const AttendArgs& a, uint32_t u, uint32_t row_tile, uint32_t hh,
                                        uint32_t n16) {
        unit = (int)u, b = u, h = hh, group = a.q_heads / c.heads;
        if (CHOSEN && !a.row_seq(bt, unit, b)) return false;
        seq_rows(bt, b, r0, n);
        const int64_t len = max(bt.lengths[b], 0);
        rows = (CHOSEN ? 1 : n) * (int)group;
        first = (int)row_tile * 16;
        const int rr = first + (int)n16;
        token = rr < rows ? token_of(rr) : -1;
        head = head_of(rr);
        const int64_t before = len - n - r0 + 1;  // a token's limit, less its row
        limit = token < 0 ? 0 : a.causal ? before + token : len;
        most = a.causal ? before + token_of(min(first + 15, rows - 1)) : len;
        least = a.causal ? before + token_of(first) : len;
        return true;
    }
    __device__ __forceinline__ int token_of(int row) const { return CHOSEN ? unit : r0 + row / (int)group; }
    __device__ __forceinline__ uint32_t head_of(int row) const { return h * group + (uint32_t)row % group; }
    // Tiles that the 16 rows read.
    __device__ __forceinline__ uint32_t tiles(const KvCache& c, const KvBatch& bt, const AttendArgs& a) const {
        if (first >= rows) return 0;
        return CHOSEN ? (uint32_t)min((int64_t)a.top, a.pages_seen(c, bt, most)) * (c.page >> 5) : tiles_of(c, bt, most);
    }
    __device__ __forceinline__ const int32_t* list(const KvCache& c, const AttendArgs& a) const {
        return CHOSEN ? a.chosen + ((uint64_t)unit * c.heads + h) * a.top : nullptr;
    }
};

// One wave's state: 16 query rows, lane 16 q + n with row n.
template <int D, int NP>
struct Rows {
    u4 qf[NP][D / 32];  // query pieces, as the second operand
    f4 o[D / 16];       // O^T: lane's channels q D/4 + r D/16 + j
    float m, l;         // largest exponent (base 2) of the row; this lane's share of the sum
};

// Scores of a tile: s[i][r] of token 8q + 2r + i, without the scale.
template <int D, int NP>
__device__ __forceinline__ void tile_scores(const Rows<D, NP>& w, const Tile<D>& t, f4 (&s)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            const float sc = bits_f32((t.ks[D == 256 ? c / 4 : 0] >> (8 * i) & 255u) << 23);
            const int dw = i * (D / 32) + c;
            const bf8 a = as_bf8(codes_bf16(t.k[dw / 4][dw % 4], sc));
#pragma unroll
            for (int p = 0; p < NP; ++p) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, as_bf8(w.qf[p][c]), s[i], 0, 0, 0);
        }
    }
}

// Whether a byte of x is 255: the seven low bits carry where they are all ones.
__device__ __forceinline__ uint32_t all_ones_byte(uint32_t x) { return ((x & 0x7F7F7F7Fu) + 0x01010101u) & x & 0x80808080u; }
template <int D>
__device__ __forceinline__ uint32_t odd_scales(const Tile<D>& t) {
    uint32_t k = t.ks[0];
    if constexpr (D == 256) k |= t.ks[1] << 16;
    return all_ones_byte(k) | all_ones_byte(t.vs[0]) | all_ones_byte(t.vs[1]);
}

// What a tile needs where it is not wholly seen by all 16 rows, or holds what is not finite, or is not there:
// scores of keys that are not finite become NaN and those that a row does not see -inf; rows that see a value that is not
// finite become NaN in that value's channels; and the scales that are left are numbers.
template <int D, int NP, bool CHOSEN>
__device__ __forceinline__ void settle_tile(Rows<D, NP>& w, Tile<D>& t, f4 (&s)[2], const Job<CHOSEN>& j, bool there, int64_t base,
                                            uint32_t lane) {
    const uint32_t q = opaque(lane) >> 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        bool bad = (t.ks[0] >> (8 * i) & 255u) == 255u;
        if constexpr (D == 256) bad |= (t.ks[1] >> (8 * i) & 255u) == 255u;
        // lane 16 q' + m says it of token 2m + i
        uint64_t b = __ballot(bad);
        b |= b >> 32;
        b |= b >> 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!there || (b >> (4 * q + e) & 1u)) s[i][e] = __builtin_nanf("");
            if (base + 8 * q + 2 * e + i >= j.limit) s[i][e] = -INFINITY;
        }
    }
    const int64_t seen = there ? j.most - base : 0;  // tokens behind are seen by no row: their scales may be anything
    uint32_t badbits = 0;
    u2 vs = t.vs;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t byte = vs[e / 4] >> (8 * (e % 4)) & 255u;
        const bool drop = (int64_t)(8 * q + e) >= seen;
        if (!drop && byte == 255u) badbits |= 1u << e;
        if (drop || byte == 255u) vs[e / 4] = (vs[e / 4] & ~(255u << (8 * (e % 4)))) | 127u << (8 * (e % 4));
    }
    t.vs = vs;
    if (__ballot(badbits != 0)) {  // which rows see such a value: a product of truth values
        u4 bf, sf;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bf[r] = ((badbits >> (2 * r) & 1u) ? 0x3F80u : 0u) | ((badbits >> (2 * r + 1) & 1u) ? 0x3F800000u : 0u);
            sf[r] = (s[0][r] != -INFINITY ? 0x3F80u : 0u) | (s[1][r] != -INFINITY ? 0x3F800000u : 0u);
        }
        const f4 count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(bf), as_bf8(sf), f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < D / 16; ++k) w.o[k][e] = count[e] > 0.f ? __builtin_nanf("") : w.o[k][e];
    }
}

// Adds a tile's values by the probabilities pf.
template <int D, int NP, int PP>
__device__ __forceinline__ void tile_values(Rows<D, NP>& w, const Tile<D>& t, const u4 (&pf)[PP]) {
    float vs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) vs[e] = bits_f32((t.vs[e / 4] >> (8 * (e % 4)) & 255u) << 23);
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
        for (int p = 0; p < PP; ++p) {
            w.o[2 * jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(even), as_bf8(pf[p]), w.o[2 * jb], 0, 0, 0);
            w.o[2 * jb + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(odd), as_bf8(pf[p]), w.o[2 * jb + 1], 0, 0, 0);
        }
    }
}

template <int D>
struct Step {  // a tile whose loads were issued
    Tile<D> t;
    bool there;
    int32_t base;  // its first token
};

// One step for 16 rows: the running maximum and sum of a softmax over its 32 tokens.  With two tiles a step, one maximum and one look at
// what is odd serve both, but a wave's first product waits for twice the loads, and its registers leave room for two waves a SIMD: 64
// sequences of 1500 tokens take 26 us so, 22 tile by tile; 4 of 262144 215 and 205.
template <int D, int NP, bool CHOSEN>
__device__ __forceinline__ void work_step(Rows<D, NP>& w, Step<D>& st, const Job<CHOSEN>& j, float c2, uint32_t lane) {
    constexpr int PP = kProbPieces<NP>;
    f4 s[2];
    tile_scores<D, NP>(w, st.t, s);
    const bool plain = st.there && (int64_t)st.base + 32 <= j.least;
    if (!plain || __ballot(odd_scales(st.t) != 0)) settle_tile<D, NP>(w, st.t, s, j, st.there, st.base, lane);
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][e]);
    top = row_max(top) * c2;
    const bool over = top > w.m + kSlack;
    top = over ? top : w.m;
    if (__ballot(over)) {
        const float a = __builtin_amdgcn_exp2f(w.m - top);
        w.m = top;
        w.l *= a;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) w.o[k][e] *= a;
    }
    u4 pf[PP];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][e], c2, -top));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][e], c2, -top));
        uint32_t pc[PP];
        pack_pieces<PP>(p0, p1, pc);
        w.l += p0 + p1;  // of the probabilities as they are: the row's logarithm is given out
#pragma unroll
        for (int p = 0; p < PP; ++p) pf[p][e] = pc[p];
    }
    tile_values<D, NP, PP>(w, st.t, pf);
}

// Where a wave's next 64 tiles lie: lane i keeps the i-th of them, so that no tile's loads wait for the page table.
template <bool CHOSEN>
struct Feed {
    uint32_t lo, hi;  // the tile's number in the pool; hi = ~0: its page is not there
    int32_t pos;      // its first token

    __device__ __forceinline__ void none() { lo = 0, hi = ~0u, pos = 0x7FFFFFFF; }
    // Tile t of sequence b (CHOSEN: of the `top` pages in `list`).
    __device__ __forceinline__ void take(const KvCache& c, const KvBatch& bt, uint32_t b, uint32_t h, const int32_t* list, uint32_t top,
                                         uint32_t t) {
        const uint32_t per_page = c.page >> 5;
        uint32_t pj = t / per_page;
        const uint32_t sub = t % per_page;
        if constexpr (CHOSEN) pj = pj < top ? (uint32_t)list[pj] : ~0u;
        pos = (int32_t)min((uint64_t)pj * c.page + sub * 32u, (uint64_t)0x7FFFFFFF);
        const int64_t page = page_of(c, bt, b, pj);
        if (page < 0) return;
        const uint64_t u = ((uint64_t)page * c.heads + h) * per_page + sub;
        lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    }
    // The loads of the i-th.  A tile that is not there is read as the pool's first, and not used.
    template <int D>
    __device__ __forceinline__ void load(const KvCache& c, uint32_t i, uint32_t lane, Step<D>& st) const {
        const uint32_t l = __builtin_amdgcn_readlane(lo, i), u = __builtin_amdgcn_readlane(hi, i);
        st.there = u != ~0u;
        st.base = (int32_t)__builtin_amdgcn_readlane((uint32_t)pos, i);
        load_tile<D>(c.pool + (st.there ? (uint64_t)u << 32 | l : 0) * (uint64_t)(34 * D), lane, st.t);
    }
};

// A lane's part of its row of q as it lies in memory, so that its loads need not be waited for where they are issued.
template <int D, int T>
struct RawQueries {
    static constexpr int N = T == GVDB_F32 ? 2 : 1;  // dwordx4 to eight channels
    u4 r[D / 32 * N];

    template <bool CHOSEN>
    __device__ __forceinline__ void load(const AttendArgs& a, const Job<CHOSEN>& j, uint32_t q4) {
#pragma unroll
        for (int i = 0; i < D / 32 * N; ++i) r[i] = u4{0, 0, 0, 0};
        if (j.token < 0) return;
        const int64_t at = (int64_t)j.token * a.q.row_stride + (int64_t)j.head * a.q.head_stride + q4 * (D / 4);
        if (a.q.wide) {
            const u4* p = (const u4*)((const char*)a.q.p + at * (T == GVDB_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < D / 32 * N; ++i) r[i] = p[i];
        } else if constexpr (T == GVDB_F32) {
            const uint32_t* p = (const uint32_t*)a.q.p + at;
#pragma unroll
            for (int i = 0; i < D / 32 * N * 4; ++i) r[i / 4][i % 4] = p[i];
        } else {
            const uint16_t* p = (const uint16_t*)a.q.p + at;
#pragma unroll
            for (int i = 0; i < D / 32 * 4; ++i) r[i / 4][i % 4] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
    }
    // The pieces that the products take.
    template <int NP>
    __device__ __forceinline__ void split(bool negate, u4 (&qf)[NP][D / 32]) const {
        const uint32_t sign = negate ? (T == GVDB_F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
        for (int i = 0; i < D / 32 * 4; ++i) {
            uint32_t pc[NP];
            if constexpr (T == GVDB_BF16) {
                pc[0] = inf_to_nan(r[i / 4][i % 4] ^ sign);
            } else if constexpr (T == GVDB_F16) {
                const uint32_t w = r[i / 4][i % 4] ^ sign;
                pack_pieces<NP>((float)__builtin_bit_cast(_Float16, (uint16_t)w), (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)), pc);
            } else {
                pack_pieces<NP>(bits_f32(r[i / 2][i % 2 * 2] ^ sign), bits_f32(r[i / 2][i % 2 * 2 + 1] ^ sign), pc);
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) qf[p][i / 4][i % 4] = pc[p];
        }
    }
};

// Rows of no sequence: left as they were, or (out.zero_rest) 0, their logarithm -inf and their pages -1.
template <int D, int T>
__device__ __forceinline__ void clear_rest(const KvCache& c, const KvBatch& bt, const AttendArgs& a) {
    if (!a.out.zero_rest || !bt.cu) return;
    const int from = min(max(bt.cu[bt.n_seqs], 0), (int)bt.rows), head = min(max(bt.cu[0], 0), from);
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t r = blockIdx.x; r < (int64_t)bt.rows - from + head; r += gridDim.x) {
        const int64_t row = r < head ? r : r - head + from;
        for (uint32_t i = threadIdx.x; i < a.q_heads * (D / 8); i += blockDim.x)
            store8<T>(a.out.p, row * a.out.row_stride + (int64_t)(i / (D / 8)) * a.out.head_stride + i % (D / 8) * 8, a.out.wide, zero);
        if (a.lse)
            for (uint32_t i = threadIdx.x; i < a.q_heads; i += blockDim.x) a.lse[row * a.q_heads + i] = -INFINITY;
        if (a.top)
            for (uint32_t i = threadIdx.x; i < c.heads * a.top; i += blockDim.x) a.chosen[row * c.heads * a.top + i] = -1;
    }
}

template <int D, int NP>
__device__ __forceinline__ void clear(Rows<D, NP>& w) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) w.o[j] = f4{0.f, 0.f, 0.f, 0.f};
    w.m = kLowest;
    w.l = 0.f;
}

template <int D>
struct JoinLds {
    float o[4][16][D + 4];  // rows four banks apart
    float m[4][16], l[4][16];
};

// A row's output: sums over the row's keys, or over a part of them (`part`: its place among the parts).
template <int D, int T, bool CHOSEN>
__device__ __forceinline__ void write_row(const AttendArgs& a, const Job<CHOSEN>& j, int row, uint32_t d, float (&x)[8], float m, float l,
                                          bool parted, uint64_t part) {
    if (parted) {
        float* po = a.part_o + part * D + d;
        *(f4*)po = f4{x[0], x[1], x[2], x[3]};
        *(f4*)(po + 4) = f4{x[4], x[5], x[6], x[7]};
        if (d == 0) *(f2*)(a.part_ml + part * 2) = f2{m, l};
        return;
    }
    const int token = j.token_of(row);
    const uint32_t head = j.head_of(row);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
    store8<T>(a.out.p, (int64_t)token * a.out.row_stride + (int64_t)head * a.out.head_stride + d, a.out.wide, x);
    if (a.lse && d == 0) a.lse[(uint64_t)token * a.q_heads + head] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) / kLog2e;
}

// Joins the four waves' parts of 16 rows and writes them.
template <int D, int T, int NP, bool CHOSEN>
__device__ __forceinline__ void join_waves(JoinLds<D>& s, Rows<D, NP>& w, const Job<CHOSEN>& j, const AttendArgs& a, uint32_t split) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, q4 = lane >> 4, n16 = lane & 15u;
    w.l = row_sum(w.l);
    if (j.token >= 0) {  // the lane's channels: r * (D / 16) + k behind q4 * (D / 4)
        if (q4 == 0) s.m[wave][n16] = w.m, s.l[wave][n16] = w.l;
        f4* to = (f4*)&s.o[wave][n16][q4 * (D / 4)];
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            f4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = w.o[(4 * c + i) % (D / 16)][(4 * c + i) / (D / 16)];
            to[c] = x;
        }
    }
    __syncthreads();
    const uint32_t live = (uint32_t)min(16, j.rows - j.first);
#pragma unroll 1
    for (uint32_t e = threadIdx.x; e < live * (D / 8); e += 256) {
        const uint32_t r = e / (D / 8), d = e % (D / 8) * 8;
        const float m = fmaxf(fmaxf(s.m[0][r], s.m[1][r]), fmaxf(s.m[2][r], s.m[3][r]));
        float l = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = __builtin_amdgcn_exp2f(s.m[k][r] - m);
            const f4 u = *(const f4*)&s.o[k][r][d], v = *(const f4*)&s.o[k][r][d + 4];
            l += s.l[k][r] * f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += u[i] * f, x[4 + i] += v[i] * f;
        }
        const int row = j.first + (int)r;
        write_row<D, T>(a, j, row, d, x, m, l, !CHOSEN && a.splits > 1,
                        ((uint64_t)j.token_of(row) * a.q_heads + j.head_of(row)) * a.splits + split);
    }
    __syncthreads();
}

// Writes one wave's rows from its registers; `part`: the place of the first row's part.
template <int D, int T, int NP, bool CHOSEN>
__device__ __forceinline__ void write_wave(Rows<D, NP>& w, const Job<CHOSEN>& j, const AttendArgs& a, bool parted, uint64_t part,
                                           uint32_t lane) {
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    const float l = row_sum(w.l);
    if (j.token < 0) return;
#pragma unroll
    for (int c = 0; c < D / 4; c += 8) {  // the lane's channels: r * (D / 16) + k behind q4 * (D / 4)
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = w.o[(c + i) % (D / 16)][(c + i) / (D / 16)];
        write_row<D, T>(a, j, j.first + (int)n16, q4 * (D / 4) + c, x, w.m, l, parted, part + n16);
    }
}

// ---- attend -----------------------------------------------------------------------------
// A workgroup takes 16 query rows of a unit and key head and one split of its tiles; its four waves take steps of them in
// turn, one step's loads in flight while another is worked on, and join their parts through LDS.  With one query token a
// sequence each cached byte is read once: 34 D / 32 bytes a token and head bound it where there are many (32 sequences of 32 pages:
// 20 us).  One sequence of 768 tokens takes 9 us, of which its 24 tiles are 4; the rest is the chain of
// loads before the first product (length, table, tiles), the join and the launch.
// 384 tokens' own 40 pages of 32, 4 heads: 46 us, 5.8 TB/s out of the caches and three quarters of the cycles in vector instructions.
template <int D, int T, bool CHOSEN>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 && T == GVDB_F32 ? 2 : 3) void k_kv_attend(KvCache c, KvBatch bt, AttendArgs a) {
    constexpr int NP = pieces(T);
    __shared__ JoinLds<D> s;
    clear_rest<D, T>(c, bt, a);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t splits = CHOSEN ? 1 : a.splits;  // chosen pages go whole here
    const uint32_t h = blockIdx.x % c.heads, split = blockIdx.x / c.heads % splits;
    const uint32_t rest = blockIdx.x / c.heads / splits;
    for (uint32_t row_tile = rest % a.row_tiles;; row_tile += a.row_tiles) {
        Job<CHOSEN> j;
        if (!j.set(c, bt, a, rest / a.row_tiles, row_tile, h, lane & 15u) || j.first >= j.rows) return;
        const uint32_t tiles = j.tiles(c, bt, a), s0 = (uint32_t)min((uint64_t)split * a.chunk, (uint64_t)tiles);
        const uint32_t s1 = split + 1 == splits ? tiles : min(s0 + a.chunk, tiles);
        if (splits > 1 && s0 >= s1) continue;  // no part: k_kv_combine does not read it
        Rows<D, NP> w;
        clear(w);
        RawQueries<D, T> raw;
        raw.load(a, j, lane >> 4);
        const uint32_t mine = s0 + wave < s1 ? (s1 - s0 - wave + 3) / 4 : 0;
        const int32_t* list = j.list(c, a);
        Feed<CHOSEN> feed;
        Step<D> st, next;
        auto fill = [&](uint32_t it) {
            const uint32_t tile = s0 + wave + 4 * (it + lane);
            feed.none();
            if (tile < s1) feed.take(c, bt, j.b, h, list, a.top, tile);
        };
        if (mine) {
            fill(0);
            feed.load(c, 0, lane, next);
        }
        raw.template split<NP>(a.negate, w.qf);
        for (uint32_t it = 0; it < mine; ++it) {
            st = next;
            if (it + 1 < mine) {
                const uint32_t i = (it + 1) % 64;
                if (i == 0) fill(it + 1);
                feed.load(c, i, lane, next);
            }
            work_step<D, NP>(w, st, j, a.scale_log2, lane);
        }
        join_waves<D, T, NP>(s, w, j, a, split);
    }
}

// The same for few rows, whose units would leave the card uneven: the steps of all units (16 rows each) lie end to end,
// and wave w of a head takes the w-th of equal shares of that line, whatever the sequences' lengths are.  A unit that one
// wave takes whole is written at once; the others' parts go to slot w + u (w and u only ever grow along the line: no two
// parts share one) and are joined by k_kv_combine.  Waves never wait for one another, and loads run on over the borders
// of units, the next unit's queries among them.  Bound by the reads: 4 sequences of 262144 tokens, 8 heads of 128 channels, 205 us with
// the join, 5.6 TB/s; 64 of up to 10000, 57 us, 4.1 TB/s, of which the join is 6.
template <int D, int T, bool CHOSEN>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 2 : 3) void k_kv_attend_line(KvCache c, KvBatch bt, AttendArgs a) {
    constexpr int NP = pieces(T);
    __shared__ uint32_t s_wsum[4], s_pref[kMaxUnits + 1];
    clear_rest<D, T>(c, bt, a);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t h = blockIdx.x % c.heads, w_id = blockIdx.x / c.heads * 4 + wave;
    {
        const uint32_t per = (a.units + 255) / 256, u0 = min(threadIdx.x * per, a.units), u1 = min(u0 + per, a.units);
        uint32_t sum = 0;
        for (uint32_t u = u0; u < u1; ++u) {
            s_pref[u] = sum;
            Job<CHOSEN> j;
            if (j.set(c, bt, a, u / a.row_tiles, u % a.row_tiles, h, 0)) sum += j.tiles(c, bt, a);
        }
        uint32_t total;
        const uint32_t before = block_scan_u32(sum, s_wsum, &total);
        for (uint32_t u = u0; u < u1; ++u) s_pref[u] += before;
        if (threadIdx.x == 0) s_pref[a.units] = total;
        __syncthreads();
        if (blockIdx.x == 0)
            for (uint32_t u = threadIdx.x; u <= a.units; u += 256) a.prefix[u] = s_pref[u];
    }
    const uint32_t total = s_pref[a.units], share = max(a.least, (total + a.lanes - 1) / a.lanes);
    const uint32_t at = (uint32_t)min((uint64_t)w_id * share, (uint64_t)total), end = min(at + share, total);
    if (at >= end) return;
    // the unit that holds a step of the line
    auto unit_of = [&](uint32_t t) {
        uint32_t lo = 0, hi = a.units;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (s_pref[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    uint32_t u = __builtin_amdgcn_readfirstlane(unit_of(at));
    Job<CHOSEN> j, jn;
    RawQueries<D, T> raw;
    (void)j.set(c, bt, a, u / a.row_tiles, u % a.row_tiles, h, lane & 15u);
    raw.load(a, j, lane >> 4);
    Feed<CHOSEN> feed;
    auto fill = [&](uint32_t it) {
        const uint32_t tile = at + it + lane;
        feed.none();
        if (tile >= end) return;
        const uint32_t v = unit_of(tile);
        Job<CHOSEN> f;
        f.unit = (int)(v / a.row_tiles), f.h = h, f.b = (uint32_t)f.unit;
        if (!CHOSEN || a.row_seq(bt, f.unit, f.b)) feed.take(c, bt, f.b, h, f.list(c, a), a.top, tile - s_pref[v]);
    };
    Step<D> st, next;
    fill(0);
    feed.load(c, 0, lane, next);
    Rows<D, NP> w;
    raw.template split<NP>(a.negate, w.qf);
    const uint32_t mine = end - at;
    for (uint32_t it = 0;;) {
        const uint32_t p0 = s_pref[u], p1 = s_pref[u + 1], to = min(end, p1);
        uint32_t v = u + 1;
        if (to < end) {
            while (s_pref[v + 1] <= to) ++v;  // units without tiles are left to the join
            v = __builtin_amdgcn_readfirstlane(v);
            (void)jn.set(c, bt, a, v / a.row_tiles, v % a.row_tiles, h, lane & 15u);
            raw.load(a, jn, lane >> 4);
        }
        clear(w);
        for (; it < to - at; ++it) {
            st = next;
            if (it + 1 < mine) {
                const uint32_t i = (it + 1) % 64;
                if (i == 0) fill(it + 1);
                feed.load(c, i, lane, next);
            }
            work_step<D, NP>(w, st, j, a.scale_log2, lane);
        }
        write_wave<D, T, NP>(w, j, a, !(at <= p0 && to == p1), ((uint64_t)h * (a.lanes + a.units) + w_id + u) * a.slot_rows, lane);
        if (to >= end) return;
        u = v;
        j = jn;
        raw.template split<NP>(a.negate, w.qf);
    }
}

// ---- attend, many rows ----------------------------------------------------------------
// A workgroup takes 128 query rows of a sequence and key head and one split of the tokens, 32 rows a wave, 64 tokens a
// step, by v_mfma_f32_32x32x16_bf16.  Keys go from the cache to registers, where every wave expands them for itself; the
// values' expansion, which has to turn them from tokens to channels, is shared: each wave expands a quarter of the step
// into LDS (two buffers, one barrier a step), as [8 tokens][channels][16 bytes], the operand as it is read.
// A row of keys stands for token t(row) with bits 2 and 3 exchanged, so that S^T leaves a lane with eight neighbouring
// tokens of its query row, which O^T = V^T P^T takes as they are.  Channel j of sixteenth l lies at row 16 j + l of V^T.
// Bound by the vector instructions that expand keys and reckon probabilities and their pieces: 2048 tokens of 2 sequences over 10000, 32
// heads on 8 of 128 channels, 837 us, 720 TFLOP/s (with probabilities of 8 bits 639 us); vector instructions issue in 66 % of the cycles,
// the matrix units are busy in 49 %, and two workgroups a CU, all that the registers hold, overlap them no further.
template <int D, int NP>
struct Rows32 {
    u4 qf[NP][D / 16];  // query pieces: lane 32 i + n has row n, channels [i D/2, (i+1) D/2)
    f16v o[D / 32];     // O^T: element e of part k is row 32 k + 8 (e / 4) + 4 i + e % 4 of V^T
    float m, l;
};

template <int D>
struct Keys32 {  // a lane's half of one token's channels
    u4 k[D / 64];
    uint32_t ks[D == 256 ? 4 : D == 128 ? 2 : 1];
};

__device__ __forceinline__ uint32_t token_of_row32(uint32_t r) { return (r & 0x13u) | (r & 4u) << 1 | (r & 8u) >> 1; }

template <int D>
__device__ __forceinline__ void load_keys32(const uint8_t* p, uint32_t i, uint32_t t, Keys32<D>& x) {
    constexpr uint32_t QB = D / 8;  // bytes of a quarter of the channels
#pragma unroll
    for (uint32_t c = 0; c < D / 64; ++c) {
        const uint32_t b = c * 16, q = 2 * i + b / QB;
        if constexpr (D == 64) {  // two quarters, eight bytes each
            const u2 lo = *(const u2*)(p + (q * 16 + t / 2) * 16 + (t & 1) * 8), hi = *(const u2*)(p + ((q + 1) * 16 + t / 2) * 16 + (t & 1) * 8);
            x.k[c] = u4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            const uint32_t at = (t & 1) * QB + b % QB;
            x.k[c] = *(const u4*)(p + (at / 16 * 64 + q * 16 + t / 2) * 16);
        }
    }
#pragma unroll
    for (uint32_t g = 0; g < D / 64; ++g) x.ks[g] = p[16 * D + (i * (D / 64) + g) * 32 + t];
}

// Rows of 16 bits only: in 32 bits the pieces of 32 rows do not fit the registers.
// The bound on workgroups keeps D = 64 within a third of the registers (55 -> 52 us: 2 sequences of up to 500 tokens, f16).
template <int D, int T>
__global__ __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) void k_kv_attend_rows(KvCache c, KvBatch bt, AttendArgs a) {
    constexpr int NP = pieces(T), PP = kProbPieces<NP>, W = D / 16;
    __shared__ u4 s_v[2][8 * D];
    __shared__ uint32_t s_odd[2][4];
    clear_rest<D, T>(c, bt, a);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t i2 = lane >> 5, n32 = lane & 31u, l16 = lane & 15u, kg = lane >> 4;
    const uint32_t h = blockIdx.x % c.heads, split = blockIdx.x / c.heads % a.splits;
    const uint32_t rest = blockIdx.x / c.heads / a.splits, b = rest / a.row_tiles;
    const uint32_t group = a.q_heads / c.heads, per_page = c.page >> 5;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t len = max(bt.lengths[b], 0), before = len - n + 1;
    const int rows = n * (int)group;
    // the last rows first: with `causal` they have the most to read
    const int blocks = (rows + 127) / 128;
    for (int rb = blocks - 1 - (int)(rest % a.row_tiles); rb >= 0; rb -= (int)a.row_tiles) {
        const int w_first = rb * 128 + (int)wave * 32, row = w_first + (int)n32;
        const bool live = row < rows;
        const int64_t limit = !live ? 0 : a.causal ? before + row / (int)group : len;
        const int64_t most = a.causal ? before + (min(rb * 128 + 127, rows - 1)) / (int)group : len;        // of the workgroup's rows
        const int64_t w_least = a.causal ? before + w_first / (int)group : len;
        const uint32_t steps = (tiles_of(c, bt, most) + 1) / 2, chunk = a.chunk / 2;
        const uint32_t s0 = (uint32_t)min((uint64_t)split * chunk, (uint64_t)steps);
        const uint32_t s1 = split + 1 == a.splits ? steps : min(s0 + chunk, steps);
        if (a.splits > 1 && s0 >= s1) continue;  // no part: k_kv_combine does not read it
        Rows32<D, NP> w;
        {
            const uint32_t sign = a.negate ? 0x80000000u : 0u;
#pragma unroll
            for (int ch = 0; ch < D / 16; ++ch) {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (live)
                    load8<T>(a.q.p, (int64_t)(r0 + row / (int)group) * a.q.row_stride + (int64_t)(h * group + (uint32_t)row % group) * a.q.head_stride +
                                        i2 * (D / 2) + 8 * ch,
                             a.q.wide, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t pc[NP];
                    pack_pieces<NP>(bits_f32(__float_as_uint(x[2 * e]) ^ sign), bits_f32(__float_as_uint(x[2 * e + 1]) ^ sign), pc);
#pragma unroll
                    for (int p = 0; p < NP; ++p) w.qf[p][ch][e] = NP == 1 ? inf_to_nan(pc[p]) : pc[p];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) w.o[k][e] = 0.f;
        w.m = kLowest;
        w.l = 0.f;
        Feed<false> feed;
        auto fill = [&](uint32_t step) {
            feed.none();
            if (step + lane / 2 < s1) feed.take(c, bt, b, h, nullptr, 0, (step + lane / 2) * 2 + lane % 2);
        };
        Keys32<D> kn[2];
        u4 vn[D / 64];
        u2 vsn;
        bool there_n[2];
        int32_t base_n = 0;
        bool v_there_n = false;
        auto load = [&](uint32_t i) {  // the i-th step of the feed
            const uint8_t* p[2];
            const uint32_t ln = opaque(lane);  // addresses are reckoned anew: kept, they would take the registers of the sums
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t lo = __builtin_amdgcn_readlane(feed.lo, 2 * i + x), hi = __builtin_amdgcn_readlane(feed.hi, 2 * i + x);
                there_n[x] = hi != ~0u;
                p[x] = c.pool + (there_n[x] ? (uint64_t)hi << 32 | lo : 0) * (uint64_t)(34 * D);
                load_keys32<D>(p[x], ln >> 5, token_of_row32(ln & 31u), kn[x]);
            }
            base_n = (int32_t)__builtin_amdgcn_readlane((uint32_t)feed.pos, 2 * i);
            const uint8_t* v = wave < 2 ? p[0] : p[1];
            v_there_n = wave < 2 ? there_n[0] : there_n[1];
#pragma unroll
            for (int k = 0; k < D / 64; ++k) vn[k] = *(const u4*)(v + 17 * D + (k * 64 + ln) * 16);
            vsn = *(const u2*)(v + 33 * D + ((ln & 15u) * D / 512) * 32 + 8 * (ln >> 4));
        };
        if (s0 < s1) {
            fill(s0);
            load(0);
        }
        for (uint32_t st = s0; st < s1; ++st) {
            const uint32_t buf = st & 1u;
            const int64_t base = base_n;
            const bool there[2] = {there_n[0], there_n[1]};
            // this wave's quarter of the values: tile wave / 2, half of each lane's channels
            {
                const int64_t seen = v_there_n ? most - base - 32 * (int64_t)(wave >> 1) : 0;
                u2 vsb = {opaque(vsn[0]), opaque(vsn[1])};
                uint32_t odd = all_ones_byte(vsb[0]) | all_ones_byte(vsb[1]);
                if (seen < 32 || __ballot(odd != 0)) {
                    odd = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t byte = vsb[e / 4] >> (8 * (e % 4)) & 255u;
                        const bool drop = (int64_t)(8 * kg + e) >= seen;  // seen by no row: it may be anything
                        if (!drop && byte == 255u) odd = 1;
                        if (drop || byte == 255u) vsb[e / 4] = (vsb[e / 4] & ~(255u << (8 * (e % 4)))) | 127u << (8 * (e % 4));
                    }
                }
                const uint64_t any = __ballot(odd != 0);
                if (lane == 0) s_odd[buf][wave] = any != 0;
                float vs[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) vs[e] = bits_f32((vsb[e / 4] >> (8 * (e % 4)) & 255u) << 23);
                auto expand = [&](auto half) {
#pragma unroll
                    for (int k = 0; k < D / 64; ++k) {
                        constexpr int H = decltype(half)::value;
                        const int jb = H * (D / 64) + k;
                        u4 even, odd2;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t x = byte_bf16<D / 64>(vn, (2 * r) * (D / 32) + jb, vs[2 * r]);
                            const uint32_t y = byte_bf16<D / 64>(vn, (2 * r + 1) * (D / 32) + jb, vs[2 * r + 1]);
                            even[r] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                            odd2[r] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                        }
                        u4* to = &s_v[buf][((wave >> 1) * 4 + kg) * D + l16];
                        to[(2 * jb) * 16] = even;
                        to[(2 * jb + 1) * 16] = odd2;
                    }
                };
                if (wave & 1u) expand(Const<1>());
                else expand(Const<0>());
            }
            f16v s[2];
            {
                uint32_t odd = 0;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int g = 0; g < D / 64; ++g) kn[x].ks[g] = opaque(kn[x].ks[g]);  // not reckoned with where it is loaded
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[x][e] = 0.f;
#pragma unroll
                    for (int ch = 0; ch < D / 16; ++ch) {
                        const bf8 k8 = as_bf8(codes_bf16(kn[x].k[ch / 4][ch % 4], bits_f32(kn[x].ks[ch / 4] << 23)));
#pragma unroll
                        for (int p = 0; p < NP; ++p) s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k8, as_bf8(w.qf[p][ch]), s[x], 0, 0, 0);
                    }
#pragma unroll
                    for (int g = 0; g < D / 64; ++g) odd |= kn[x].ks[g] == 255u;
                    __builtin_amdgcn_sched_barrier(0);  // one tile's keys expanded at a time: their registers are needed
                }
                if (base + 64 > w_least || !there[0] || !there[1] || __ballot(odd)) {
                    const uint32_t i2s = opaque(i2);
                    const int see = (int)max(min(limit - base, (int64_t)64), (int64_t)0);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        bool bad = false;
#pragma unroll
                        for (int g = 0; g < D / 64; ++g) bad |= kn[x].ks[g] == 255u;
                        uint64_t bb = __ballot(bad);
                        bb |= bb >> 32;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint32_t r = 8 * (e / 4) + 4 * i2s + e % 4;  // the key's row
                            if (!there[x] || (bb >> r & 1u)) s[x][e] = __builtin_nanf("");
                            if ((int)(32 * x + 16 * (e / 8) + 8 * i2s + e % 8) >= see) s[x][e] = -INFINITY;
                        }
                    }
                }
            }
            {  // behind the last step: the pool's first tile, not used; without a branch, whose copies would wait for the loads
                const uint32_t i = (st + 1 - s0) % 32;
                if (i == 0) fill(st + 1);
                load(i);
            }
            __syncthreads();
            float top = s[0][0];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[x][e]);
            {
                const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = fmaxf(bits_f32(r[0]), bits_f32(r[1])) * a.scale_log2;
            }
            const bool over = top > w.m + kSlack;
            top = over ? top : w.m;
            if (__ballot(over)) {
                const float f = __builtin_amdgcn_exp2f(w.m - top);
                w.m = top;
                w.l *= f;
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) w.o[k][e] *= f;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    u4 v[D / 32], pf[PP];  // the values are read while the probabilities are reckoned
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) v[k] = s_v[buf][(4 * x + 2 * ch + i2) * D + 32 * k + n32];
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][8 * ch + 2 * e], a.scale_log2, -top));
                        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][8 * ch + 2 * e + 1], a.scale_log2, -top));
                        uint32_t pc[PP];
                        pack_pieces<PP>(p0, p1, pc);
                        w.l += p0 + p1;  // of the probabilities as they are: the row's logarithm is given out
#pragma unroll
                        for (int p = 0; p < PP; ++p) pf[p][e] = pc[p];
                    }
#pragma unroll
                    for (int k = 0; k < D / 32; ++k)
#pragma unroll
                        for (int p = 0; p < PP; ++p)
                            w.o[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(v[k]), as_bf8(pf[p]), w.o[k], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (s_odd[buf][0] | s_odd[buf][1] | s_odd[buf][2] | s_odd[buf][3]) {
                // a value that is not finite: its group's channels of the rows that see it
                const uint32_t i2s = opaque(i2);
                for (int t = 0; t < 64; ++t) {
                    if (!(base + t < limit)) continue;
                    const int64_t page = page_of(c, bt, b, (uint32_t)((2 * st + t / 32) / per_page));
                    if (page < 0) continue;
                    const uint8_t* vs = c.pool + tile_at<D>(c, page, h, (2 * st + t / 32) % per_page) + 33 * D + t % 32;
#pragma unroll
                    for (int k = 0; k < D / 32; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint32_t l = 8 * (e / 4 % 2) + 4 * i2s + e % 4;  // sixteenth of the channels
                            if (vs[(l * W / 32) * 32] == 255u) w.o[k][e] = __builtin_nanf("");
                        }
                }
            }
        }
        // each lane has its row's channels [(8 q + 4 i2) W, + 4 W), q = 0, 1
        {
            const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(w.l), __float_as_uint(w.l), false, false);
            w.l = bits_f32(r[0]) + bits_f32(r[1]);
        }
        if (live) {
            const int token = r0 + row / (int)group;
            const uint32_t head = h * group + (uint32_t)row % group;
            const uint64_t at = (uint64_t)token * a.q_heads + head;
            const float inv = a.splits > 1 ? 1.f : w.l == 0.f ? 0.f : 1.f / w.l;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c8 = 0; c8 < 4 * W; c8 += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = (c8 + e) % W, l4 = (c8 + e) / W;
                        x[e] = w.o[j / 2][8 * (j % 2) + 4 * q + l4] * inv;
                    }
                    const uint32_t d = (8 * q + 4 * i2) * W + c8;
                    if (a.splits > 1) {
                        float* po = a.part_o + (at * a.splits + split) * D + d;
                        *(f4*)po = f4{x[0], x[1], x[2], x[3]};
                        *(f4*)(po + 4) = f4{x[4], x[5], x[6], x[7]};
                    } else {
                        store8<T>(a.out.p, (int64_t)token * a.out.row_stride + (int64_t)head * a.out.head_stride + d, a.out.wide, x);
                    }
                }
            if (i2 == 0) {
                if (a.splits > 1) *(f2*)(a.part_ml + (at * a.splits + split) * 2) = f2{w.m, w.l};
                else if (a.lse) a.lse[at] = w.l == 0.f ? -INFINITY : (w.m + __builtin_amdgcn_logf(w.l)) / kLog2e;
            }
        }
        __syncthreads();  // the next rows write the buffers that this one's last step read
    }
}

// ---- combine ----------------------------------------------------------------------------
// Joins a row's parts: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  D / 8 lanes hold the channels.  FEW (parts of whole
// rows, at most 16): each of a wave's 512 / D groups of lanes joins a row of its own.  Else the groups share one row and take
// every so many-th part; the order of the sum is the lanes', alike on every run.  Bound by its chain of loads: 4 to 7 us.
template <int D, int T, bool CHOSEN, bool FEW>
__global__ __launch_bounds__(256) void k_kv_combine(KvCache c, KvBatch bt, AttendArgs a) {
    static_assert(!CHOSEN || !FEW, "chosen pages are joined along the line only");
    constexpr uint32_t L = D / 8, G = 64 / L;
    const uint32_t lane = threadIdx.x & 63u, g = lane / L, d = lane % L * 8;
    const uint64_t wave = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6), at = FEW ? wave * G + g : wave;
    if (at >= (uint64_t)bt.rows * a.q_heads) return;
    const int token = (int)(at / a.q_heads);
    const uint32_t head = at % a.q_heads;
    uint32_t b;
    if (!a.row_seq(bt, token, b)) return;
    int r0, n;
    seq_rows(bt, b, r0, n);
    uint64_t first, step;  // where the parts lie
    uint32_t parts;
    if (CHOSEN || (!FEW && a.lanes > 0)) {  // the line's
        const uint32_t group = a.q_heads / c.heads;
        const uint32_t row = (CHOSEN ? 0u : (uint32_t)(token - r0)) * group + head % group;
        const uint32_t u = (CHOSEN ? (uint32_t)token : b) * a.row_tiles + row / 16;
        const uint32_t p0 = a.prefix[u], p1 = a.prefix[u + 1], total = a.prefix[a.units];
        const uint32_t share = max(a.least, (total + a.lanes - 1) / a.lanes);
        const uint32_t w0 = p0 / share, w1 = p1 > p0 ? (p1 - 1) / share : w0;
        if (p1 > p0 && w0 == w1) return;  // one wave took it whole
        parts = p1 > p0 ? w1 - w0 + 1 : 0;
        step = a.slot_rows;
        first = ((uint64_t)(head / group) * (a.lanes + a.units) + w0 + u) * a.slot_rows + row % 16;
    } else {
        const int64_t len = max(bt.lengths[b], 0);
        const int64_t limit = a.causal ? len - n + (token - r0) + 1 : len;
        const uint32_t tiles = tiles_of(c, bt, limit);
        parts = min(a.splits, (tiles + a.chunk - 1) / a.chunk);
        step = 1;
        first = at * a.splits;
    }
    float m = kLowest;
    if constexpr (FEW) {
        for (uint32_t s = 0; s < parts; ++s) m = fmaxf(m, a.part_ml[(first + s) * 2]);
    } else {
        for (uint32_t s = lane; s < parts; s += 64) m = fmaxf(m, a.part_ml[(first + s * step) * 2]);
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    }
    float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t s = FEW ? 0 : g; s < parts; s += FEW ? 1 : G) {
        const uint64_t p = first + s * step;
        const f2 ml = *(const f2*)(a.part_ml + p * 2);
        const float* po = a.part_o + p * D + d;
        const f4 u = *(const f4*)po, v = *(const f4*)(po + 4);
        const float f = __builtin_amdgcn_exp2f(ml[0] - m);
        l += ml[1] * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += u[i] * f, o[4 + i] += v[i] * f;
    }
    if constexpr (!FEW) {
#pragma unroll
        for (uint32_t x = L; x < 64; x <<= 1) {
            l += __shfl_xor(l, (int)x);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] += __shfl_xor(o[i], (int)x);
        }
        if (g) return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= inv;
    store8<T>(a.out.p, (int64_t)token * a.out.row_stride + (int64_t)head * a.out.head_stride + d, a.out.wide, o);
    if (a.lse && d == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) / kLog2e;
}

// ---- which pages ------------------------------------------------------------------------
// Score of a page for a query head: 2^(a + b) * sum_d max(q8_d, 0) hi_d + min(q8_d, 0) lo_d with q8 = rint(q / 2^a) and the
// page's bounds hi, lo in units of 2^b.  The sum is a product of whole numbers over 2 D channels: v_mfma_i32_16x16x64_i8,
// exact in any order.  A wave scores 16 pages for 16 columns: `width` columns (a power of two) a token, the group's heads.

// Score of a page that holds what is not finite, or is not there: over all others, which end at the largest float.
constexpr float kNotFinite = INFINITY;

template <int D>
struct ScoreCols {  // this lane's column: channels k * 64 + q4 * 16 .. + 16 in 8 bits
    u4 pos[D / 64], neg[D / 64];
    uint32_t e;  // biased exponent of the column's largest magnitude
    bool on;

    template <int T>
    __device__ __forceinline__ void load(const AttendArgs& a, bool live, int64_t at, uint32_t q4) {
        on = live;
        float x[D / 64][16];
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (on) load8<T>(a.q.p, at + k * 64 + q4 * 16 + half * 8, a.q.wide, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[k][half * 8 + i] = y[i];
                    amax = max(amax, __float_as_uint(y[i]) & 0x7FFFFFFFu);
                }
            }
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
        e = min(max((amax + 0x1FFFFu) >> 23, 7u), 255u);
        const bool finite = amax < 0x7F800000u;  // else every score is 0
        const float up = bits_f32((260u - e) << 23);
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int wd = 0; wd < 4; ++wd) {
                uint32_t pp = 0, nn = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int v = finite ? (int)rintf(x[k][wd * 4 + i] * up) : 0;
                    pp |= (uint32_t)(max(v, 0) & 255) << (8 * i);
                    nn |= (uint32_t)(min(v, 0) & 255) << (8 * i);
                }
                pos[k][wd] = pp, neg[k][wd] = nn;
            }
    }
};

// Each lane's values and those of the lane that a DPP control names (quad_perm exchanges of 1 and 2, half and whole row mirrors:
// after the exchanges below them they reach every lane of 4, 8 and 16).
template <int CTRL>
__device__ __forceinline__ void row_max_step(float (&v)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int x = (int)__float_as_uint(v[r]);
        v[r] = fmaxf(v[r], __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false)));
    }
}

// best[r]: the largest score over the columns of this lane's token, of page 4 q4 + r of 16.  Lane 16 q + m holds page m's channels
// q * 16 .. + 16 of every 64 in pb; lane first + m its exponent in e (255: not finite, or not there).
template <int D>
__device__ __forceinline__ void score_pages(const u4 (&pb)[D / 32], uint32_t e, uint32_t first, const ScoreCols<D>& col, uint32_t width,
                                            uint32_t q4, float (&best)[4]) {
    i4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < D / 64; ++k) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, pb[k]), __builtin_bit_cast(i4, col.pos[k]), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, pb[D / 64 + k]), __builtin_bit_cast(i4, col.neg[k]), acc, 0, 0, 0);
    }
    uint32_t be[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) be[r] = (uint32_t)__shfl((int)e, (int)(first + 4 * q4) + r);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int ex = min(max((int)col.e + (int)be[r] - 266, -126), 127);
        best[r] = col.on ? (float)acc[r] * bits_f32((uint32_t)(ex + 127) << 23) : -INFINITY;
    }
    // over the token's columns: pairs, fours, eights, all 16 lanes of a row
    if (width > 1) row_max_step<0xB1>(best);
    if (width > 2) row_max_step<0x4E>(best);
    if (width > 4) row_max_step<0x141>(best);
    if (width > 8) row_max_step<0x140>(best);
#pragma unroll
    for (int r = 0; r < 4; ++r) best[r] = be[r] == 255u ? kNotFinite : fminf(best[r], 3.402823466e38f);
}

// Scores of pages [from, to) for CG times 16 / width tokens, 64 pages a wave at a time, all their bounds in flight at once (D = 256, and
// several times 16 columns: half of them, by half the code); `put` takes four neighbouring pages' scores for the g-th 16 columns.
template <int D, int CG, class Put>
__device__ __forceinline__ void score_range(const KvCache& c, const KvBatch& bt, uint32_t b, uint32_t h, const ScoreCols<D> (&col)[CG],
                                            uint32_t width, int64_t from, int64_t to, uint32_t wave, uint32_t waves, uint32_t lane, Put put) {
    constexpr int NB = D == 256 || CG > 1 ? 2 : 4;
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    auto look = [&](int64_t p) { return p + lane < to ? (int)page_of(c, bt, b, (uint32_t)(p + lane)) : -1; };
    int64_t p = from + wave * 64;
    int page = p < to ? look(p) : -1;
    for (; p < to; p += waves * 64) {
        const uint32_t e = page >= 0 ? c.bound_exps[(uint64_t)page * c.heads + h] : 255u;
        const int now = page;
#pragma unroll 1
        for (int s = 0; s < 4; s += NB) {
            if (p + 16 * s >= to) break;
            u4 pb[NB][D / 32];
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                const int pg = max(__shfl(now, (int)(16 * (s + x) + n16)), 0);  // one that is not there: its exponent says so
                const int8_t* row = c.bounds + ((uint64_t)pg * c.heads + h) * (2 * D) + q4 * 16;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) pb[x][k] = *(const u4*)(row + k * 64);
            }
            if (s + NB == 4) page = look(p + waves * 64);
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int g = 0; g < CG; ++g) {
                    float best[4];
                    score_pages<D>(pb[x], e, 16 * (s + x), col[g], width, q4, best);
                    put(g, p + 16 * (s + x) + 4 * q4, best);
                }
        }
    }
}

// ---- choosing ------------------------------------------------------------------------------
// The `top` of a token's `seen` pages (more than `top`): the first and the most recent ones, then the largest scores, the lowest
// page among equals; in order.
//
// The want-th largest of the lanes' own maxima is no more than the want-th largest of all keys: what is below it is dropped at
// once, and a list little longer than `want` is left.  On it the interval of keys that holds the last one taken is halved until
// it parts the list; one wave, no barrier.  Code that runs once is slow to fetch: the loops are kept rolled.
constexpr uint32_t kListWave = 256;   // list entries a wave
constexpr uint32_t kChooseThreads = 512, kChooseWaves = kChooseThreads / 64;
struct ChooseLds {
    uint32_t key[kChooseWaves * kListWave], page[kChooseWaves * kListWave];
    uint32_t most[kChooseThreads], count[kChooseWaves];
};

// The interval [lo, hi): `want` or more of the n keys are >= lo, fewer (`over`) are >= hi.  true: from `want` to `want` + `slack` are
// >= lo; false: [lo, hi) is one key.
template <class Key>
__device__ __forceinline__ bool halve(Key key, uint32_t n, uint32_t want, uint32_t slack, uint32_t& lo, uint32_t hi, uint32_t& over,
                                      uint32_t lane) {
    constexpr int K = 8;  // keys a lane: the list, or the lanes' maxima
    over = 0;
    uint32_t k[K];
    const bool few = n <= 64 * K;
#pragma unroll
    for (int i = 0; i < K; ++i) k[i] = few && lane + 64 * i < n ? key(lane + 64 * i) : 0;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        uint32_t c = 0;
        if (few) {
#pragma unroll
            for (int i = 0; i < K; ++i) c += (uint32_t)__popcll(__ballot(k[i] >= mid));
        } else {
#pragma unroll 4
            for (uint32_t i = 0; i < n; i += 64) c += (uint32_t)__popcll(__ballot(i + lane < n && key(min(i + lane, n - 1)) >= mid));
        }
        if (c >= want) lo = mid;
        else hi = mid, over = c;
        if (c >= want && c - want <= slack) return true;
    }
    return false;
}

// W waves together (`wave` of them; barriers where W > 1), or one wave by itself.
template <uint32_t W, class Scores>
__device__ __forceinline__ void choose_pages(const AttendArgs& a, Scores sc, uint32_t seen, int32_t* out, ChooseLds& s, uint32_t wave,
                                             uint32_t lane) {
    auto meet = [] {
        if constexpr (W > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    const uint32_t part = W > 1 ? wave : 0, home = W > 1 ? 0 : wave;  // of the pages, and where the list begins
    const uint32_t lo_j = a.first, hi_j = seen - a.recent, want = a.top - a.first - a.recent;
    const uint32_t each = ((hi_j - lo_j + W - 1) / W + 63) / 64 * 64;  // a wave's pages, side by side: the list is in order
    const uint32_t j0 = min(lo_j + part * each, hi_j), j1 = min(j0 + each, hi_j);
    uint32_t* const list_key = s.key + home * kListWave;
    uint32_t* const list_page = s.page + home * kListWave;
    constexpr uint32_t kCap = kListWave * W;
    // the lanes' maxima, and the least and largest of them
    uint32_t most = 0;
#pragma unroll 4
    for (uint32_t j = j0 + lane; j < j1; j += 64) most = max(most, f32_order(sc(j)));
    s.most[wave * 64 + lane] = most;
    meet();
    uint32_t hi = 0, floor = 0;
    auto maxima = [&](uint32_t i) { return s.most[(W > 1 ? 0 : wave * 64) + i]; };
#pragma unroll 1
    for (uint32_t i = lane; i < W * 64; i += 64) hi = max(hi, maxima(i));
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) hi = max(hi, (uint32_t)__shfl_xor((int)hi, x));
    hi = __builtin_amdgcn_readfirstlane(hi);
    uint32_t over;
    if (want > 0 && want <= W * 64) (void)halve(maxima, W * 64, want, 2 * W, floor, hi + 1, over, lane);
    // the list of what is left; where it is too long, the pages themselves are gone over
    uint32_t at = 0, n = 0;
    if constexpr (W > 1) {  // each wave's pages go behind those of the waves before
        uint32_t mine = 0;
#pragma unroll 2
        for (uint32_t j = j0; j < j1; j += 64) mine += (uint32_t)__popcll(__ballot(j + lane < j1 && f32_order(sc(min(j + lane, j1 - 1))) >= floor));
        if (lane == 0) s.count[wave] = mine;
        meet();
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const uint32_t x = s.count[w];
            if (w < part) at += x;
            n += x;
        }
    }
    if (n <= kCap) {
#pragma unroll 2
        for (uint32_t j = j0; j < j1; j += 64) {
            const uint32_t k = f32_order(sc(min(j + lane, j1 - 1)));
            const bool in = j + lane < j1 && k >= floor;
            const uint64_t m = __ballot(in);
            if (!m) continue;
            const uint32_t to = at + (uint32_t)__popcll(m & ((1ull << lane) - 1ull));
            if (in && to < kCap) list_key[to] = k, list_page[to] = j + lane;
            at += (uint32_t)__popcll(m);
        }
    }
    if constexpr (W == 1) n = at;
    const bool listed = n <= kCap;
    meet();
    if (W == 1 || wave == 0) {
        for (uint32_t i = lane; i < a.first; i += 64) out[i] = (int32_t)i;
        for (uint32_t i = lane; i < a.recent; i += 64) out[a.first + want + i] = (int32_t)(hi_j + i);
        if (want > 0) {
            if (!listed) n = hi_j - lo_j, floor = 0;
            auto key = [&](uint32_t i) { return listed ? list_key[i] : f32_order(sc(lo_j + i)); };
            uint32_t lo = floor;
            const bool exact = n > want && halve(key, n, want, 0, lo, hi + 1, over, lane);
            // n == want: all; else those over lo, and the first `ties` that equal it
            const uint32_t ties = n == want ? ~0u : exact ? ~0u : want - over;
            uint32_t put = a.first, tied = 0;
#pragma unroll 1
            for (uint32_t i = 0; i < n; i += 64) {
                const uint32_t k = i + lane < n ? key(i + lane) : 0u;
                const bool same = i + lane < n && k == lo;
                const uint64_t sm = __ballot(same), below = (1ull << lane) - 1ull;
                const bool take = (i + lane < n && k > lo) || (same && tied + (uint32_t)__popcll(sm & below) < ties);
                const uint64_t tm = __ballot(take);
                if (take) out[put + (uint32_t)__popcll(tm & below)] = (int32_t)(listed ? list_page[i + lane] : lo_j + i + lane);
                put += (uint32_t)__popcll(tm);
                tied += (uint32_t)__popcll(sm);
            }
        }
    }
    meet();
}

// One workgroup: the pages of `per` tokens of a sequence (at most CG times 16 / width) and one key head, scored into LDS and chosen
// there.  The tokens share the bounds that it reads, 2 D + 1 bytes a page.  CG > 1: a wave quantises sixteen columns for all of them,
// and hands them on through LDS; with every wave at all of them, and the loop over pages unrolled, it waited for its own code.
// 384 tokens, 4 heads, 1024 pages: 36 us (45 before; 67 by one sixteen columns a workgroup), about a third each for the prologue, the
// scores and the choice, none of them near a rate of the card: 192 workgroups, a chain of short phases.  3800 pages: 95 us.
template <int D, int T, int CG>
__global__ __launch_bounds__(kChooseThreads) void k_kv_choose(KvCache c, KvBatch bt, AttendArgs a, uint32_t tok_tiles, uint32_t per) {
    extern __shared__ float s_sc[];  // [per][table_width]
    // columns, each wave's sixteen for all the waves; then the choice
    struct Cols {
        u4 x[D / 32][64];
        uint32_t e[64];
    };
    __shared__ union Lds {
        ChooseLds choose;
        Cols col[CG];
    } s_lds;
    ChooseLds& s_choose = s_lds.choose;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    const uint32_t h = blockIdx.x % c.heads, unit = blockIdx.x / c.heads, b = unit / tok_tiles;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t before = (int64_t)max(bt.lengths[b], 0) - n + 1;
    const uint32_t group = a.q_heads / c.heads, width = min(16u, next_pow2(group));
    for (int t0 = (int)(unit % tok_tiles) * (int)per; t0 < n; t0 += (int)(tok_tiles * per)) {
        const int toks = min((int)per, n - t0);
        const int64_t have = a.pages_seen(c, bt, before + t0 + toks - 1), seen = min(have, (int64_t)bt.table_width);
        if (have > (int64_t)a.top) {
            const uint32_t my = n16 / width, toks16 = 16 / width;  // this lane's token of each sixteen columns
            for (uint32_t g0 = 0; g0 < group; g0 += width) {
                const uint32_t gh = g0 + n16 % width;
                ScoreCols<D> col[CG];
                auto take = [&](int g, ScoreCols<D>& x) {
                    const int tok = g * (int)toks16 + (int)my;
                    x.template load<T>(a, tok < toks && gh < group,
                                       (int64_t)(r0 + t0 + tok) * a.q.row_stride + (int64_t)(h * group + gh) * a.q.head_stride, q4);
                };
                if constexpr (CG == 1) {
                    take(0, col[0]);
                } else {
                    if (g0) __syncthreads();
                    if (wave < CG) {
                        take((int)wave, col[0]);
#pragma unroll
                        for (int k = 0; k < D / 64; ++k) s_lds.col[wave].x[k][lane] = col[0].pos[k], s_lds.col[wave].x[D / 64 + k][lane] = col[0].neg[k];
                        s_lds.col[wave].e[lane] = col[0].e | (col[0].on ? 256u : 0u);
                    }
                    __syncthreads();
#pragma unroll
                    for (int g = 0; g < CG; ++g) {
#pragma unroll
                        for (int k = 0; k < D / 64; ++k) col[g].pos[k] = s_lds.col[g].x[k][lane], col[g].neg[k] = s_lds.col[g].x[D / 64 + k][lane];
                        const uint32_t e = s_lds.col[g].e[lane];
                        col[g].e = e & 255u, col[g].on = e > 255u;
                    }
                }
                score_range<D, CG>(c, bt, b, h, col, width, 0, seen, wave, kChooseWaves, lane, [&](int g, int64_t p, const float(&best)[4]) {
                    const int tok = g * (int)toks16 + (int)my;
                    if (tok >= toks || n16 % width) return;
                    float* to = &s_sc[tok * bt.table_width + p];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (p + r < seen) to[r] = g0 ? fmaxf(to[r], best[r]) : best[r];
                });
            }
        }
        __syncthreads();
        const uint32_t in_lds = bt.table_width;
        for (int t = 0; t < toks; ++t) {
            const int64_t mine = a.pages_seen(c, bt, before + t0 + t);
            int32_t* out = a.chosen + ((uint64_t)(r0 + t0 + t) * c.heads + h) * a.top;
            const float* sc = s_sc + t * bt.table_width;
            // a page beyond the table is the last: it is among the recent ones, or scores as one that is not there
            auto score = [=](uint32_t j) {
                const float x = sc[min(j, in_lds - 1)];
                return j < in_lds ? x : kNotFinite;
            };
            if (mine > (int64_t)a.top && toks == 1) {
                choose_pages<kChooseWaves>(a, score, (uint32_t)mine, out, s_choose, wave, lane);
            } else if ((uint32_t)t % kChooseWaves == wave) {  // each wave its token
                if (mine > (int64_t)a.top) {
                    choose_pages<1>(a, score, (uint32_t)mine, out, s_choose, wave, lane);
                } else {
                    for (uint32_t i = lane; i < a.top; i += 64) out[i] = (int64_t)i < mine ? (int32_t)i : -1;
                }
            }
        }
        __syncthreads();
    }
}

// The same in two kernels, scores by way of memory, where few tokens have many pages, or more than LDS holds; for rows [row0, row1),
// as many as the scratch has room for.  One token of 1024 pages, 8 heads: 7 us and 6 to 10, chains of loads; 32 tokens of up to 1563:
// 17 us, 2.8 TB/s of bounds, and 10.
template <int D, int T>
__global__ __launch_bounds__(256) void k_kv_score(KvCache c, KvBatch bt, AttendArgs a, uint32_t per, uint32_t chunks, uint32_t row0, uint32_t row1) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t q4 = lane >> 4, n16 = lane & 15u;
    const uint32_t h = blockIdx.x % c.heads, chunk = blockIdx.x / c.heads % chunks;
    const uint32_t group = a.q_heads / c.heads, width = min(16u, next_pow2(group));
    // `per` rows, at most 16 / width: those of one sequence share the bounds that are read
    int row = (int)(row0 + blockIdx.x / c.heads / chunks * per), toks;
    const int end = (int)min((uint32_t)row + per, row1);
    for (; row < end; row += toks) {
        uint32_t b;
        toks = 1;
        if (!a.row_seq(bt, row, b)) continue;
        int r0, n;
        seq_rows(bt, b, r0, n);
        toks = max(min(end, r0 + n) - row, 1);
        const int64_t limit = (int64_t)max(bt.lengths[b], 0) - n + (row - r0) + toks;  // the last of them sees most
        const int64_t seen = min(a.pages_seen(c, bt, limit), (int64_t)bt.table_width);
        const int64_t from = (int64_t)chunk * a.score_chunk;
        const int64_t to = chunk + 1 == chunks ? seen : min(seen, from + (int64_t)a.score_chunk);
        const uint32_t my = n16 / width;
        for (uint32_t g0 = 0; g0 < group && from < to; g0 += width) {
            const uint32_t gh = g0 + n16 % width;
            ScoreCols<D> col[1];
            col[0].template load<T>(a, (int)my < toks && gh < group,
                                    (int64_t)(row + (int)my) * a.q.row_stride + (int64_t)(h * group + gh) * a.q.head_stride, q4);
            score_range<D, 1>(c, bt, b, h, col, width, from, to, wave, 4, lane, [&](int, int64_t p, const float(&best)[4]) {
                if ((int)my >= toks || n16 % width) return;
                float* out = a.scores + ((uint64_t)(row - (int)row0 + (int)my) * c.heads + h) * bt.table_width + p;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (p + r < to) out[r] = g0 ? fmaxf(out[r], best[r]) : best[r];
            });
        }
    }
}

__global__ __launch_bounds__(kChooseThreads) void k_kv_select(KvCache c, KvBatch bt, AttendArgs a, uint32_t row0) {
    __shared__ ChooseLds s_choose;
    const uint32_t h = blockIdx.x % c.heads;
    const int token = (int)(row0 + blockIdx.x / c.heads);
    uint32_t b;
    if (!a.row_seq(bt, token, b)) return;
    int r0, n;
    seq_rows(bt, b, r0, n);
    const int64_t seen = a.pages_seen(c, bt, (int64_t)max(bt.lengths[b], 0) - n + (token - r0) + 1);
    int32_t* out = a.chosen + ((uint64_t)token * c.heads + h) * a.top;
    if (seen <= (int64_t)a.top) {
        for (uint32_t i = threadIdx.x; i < a.top; i += kChooseThreads) out[i] = (int64_t)i < seen ? (int32_t)i : -1;
        return;
    }
    const float* sc = a.scores + ((uint64_t)(token - (int)row0) * c.heads + h) * bt.table_width;
    const uint32_t width = bt.table_width;
    auto score = [=](uint32_t j) {
        const float x = sc[min(j, width - 1)];
        return j < width ? x : kNotFinite;
    };
    choose_pages<kChooseWaves>(a, score, (uint32_t)seen, out, s_choose,
                               __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), threadIdx.x & 63u);
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
#define KV_T16(D_, dtype, body)                                \
    if ((dtype) == GVDB_F16) KV_DT(D_, GVDB_F16, body)         \
    else KV_DT(D_, GVDB_BF16, body)
#define KV_DISPATCH16(dim, dtype, body)          \
    switch (dim) {                               \
        case 64: KV_T16(64, dtype, body) break;   \
        case 128: KV_T16(128, dtype, body) break; \
        default: KV_T16(256, dtype, body) break;  \
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
// A launch's threads along x are counted in 32 bits.
bool fits(uint64_t blocks, uint64_t threads = 256) { return blocks > 0 && blocks * threads < (1ull << 32); }
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
    const uint32_t tokens = 256 / (c.dim / 8);  // a workgroup
    const uint64_t blocks = ((uint64_t)bt.rows + tokens - 1) / tokens * c.heads;
    if (!fits(blocks)) return hipErrorInvalidValue;
    const uint32_t dtype = k.p ? k.dtype : v.dtype;
    KV_DISPATCH(c.dim, dtype, (k_kv_read<D, T><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, k, v)));
    GVDB_LAUNCH_CHECK();
    return hipSuccess;
}

hipError_t launch_kv_attend(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s) {
    const uint64_t blocks = (uint64_t)c.heads * (a.lanes ? a.lanes / 4 : a.splits * a.row_tiles * bt.n_seqs);
    const bool few = !a.lanes && a.splits <= 16;
    const uint64_t per_join = few ? 4 * (512 / c.dim) : 4, joins = ((uint64_t)bt.rows * a.q_heads + per_join - 1) / per_join;
    if (!fits(blocks) || !fits(joins)) return hipErrorInvalidValue;
    if (a.lanes) {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend_line<D, T, false><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    } else if (a.many) {
        KV_DISPATCH16(c.dim, a.q.dtype, (k_kv_attend_rows<D, T><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    } else {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend<D, T, false><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    }
    GVDB_LAUNCH_CHECK();
    if (a.lanes || a.splits > 1) {
        if (few) {
            KV_DISPATCH(c.dim, a.q.dtype, (k_kv_combine<D, T, false, true><<<(uint32_t)joins, 256, 0, s>>>(c, bt, a)));
        } else {
            KV_DISPATCH(c.dim, a.q.dtype, (k_kv_combine<D, T, false, false><<<(uint32_t)joins, 256, 0, s>>>(c, bt, a)));
        }
        GVDB_LAUNCH_CHECK();
    }
    return hipSuccess;
}

hipError_t launch_kv_attend_topk(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s) {
    const uint32_t group = a.q_heads / c.heads;
    const uint32_t per16 = 16 / (group >= 16 ? 16 : next_pow2(group));
    const bool fused = a.score_chunk == 0;
    // prompts: several times 16 columns a workgroup, eight tokens, one a wave, at most
    const uint32_t groups = c.dim == 256 ? 2 : 4;
    const bool many = fused && bt.max_new >= 2 * per16;
    uint32_t per = many ? std::min(groups * per16, kChooseWaves) : per16;
    if (bt.max_new < per) per = next_pow2(bt.max_new);
    while (fused && per > 1 && per * bt.table_width > kChooseScores) per /= 2;
    const uint64_t blocks = (uint64_t)c.heads * (a.lanes ? a.lanes / 4 : (uint64_t)a.row_tiles * bt.rows);
    if (!fits(blocks)) return hipErrorInvalidValue;
    if (fused) {
        const uint64_t others = (uint64_t)c.heads * bt.n_seqs;
        const uint32_t tok_tiles = capped(((uint64_t)bt.max_new + per - 1) / per, others, 1u << 22);
        if (!fits(others * tok_tiles, kChooseThreads)) return hipErrorInvalidValue;
        const uint32_t lds = per * bt.table_width * 4;
        auto launch = [&](auto cg) {
            constexpr int CG = decltype(cg)::value;
            KV_DISPATCH(c.dim, a.q.dtype, (k_kv_choose<D, T, D == 256 && CG == 4 ? 2 : CG>
                                           <<<(uint32_t)(others * tok_tiles), kChooseThreads, lds, s>>>(c, bt, a, tok_tiles, per)));
        };
        // as many times 16 columns as the workgroup's tokens take: half the table's tokens fit LDS where it has 3800 pages, and the other
        // half's columns would cost as much (384 tokens, 4 heads: 149 us, so 115)
        if (per <= per16) launch(Const<1>());
        else if (per <= 2 * per16) launch(Const<2>());
        else launch(Const<4>());
        GVDB_LAUNCH_CHECK();
    } else {
        const uint32_t chunks = (kv_max_pages(c, bt) + a.score_chunk - 1) / a.score_chunk;
        if (!fits((uint64_t)((a.score_rows + per - 1) / per) * chunks * c.heads) || !fits((uint64_t)a.score_rows * c.heads, kChooseThreads))
            return hipErrorInvalidValue;
        for (uint32_t row0 = 0; row0 < bt.rows; row0 += a.score_rows) {
            const uint32_t rows = std::min(a.score_rows, bt.rows - row0), tiles = (rows + per - 1) / per;
            KV_DISPATCH(c.dim, a.q.dtype, (k_kv_score<D, T><<<tiles * chunks * c.heads, 256, 0, s>>>(c, bt, a, per, chunks, row0, row0 + rows)));
            GVDB_LAUNCH_CHECK();
            k_kv_select<<<rows * c.heads, kChooseThreads, 0, s>>>(c, bt, a, row0);
            GVDB_LAUNCH_CHECK();
        }
    }
    if (a.lanes) {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend_line<D, T, true><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    } else {
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_attend<D, T, true><<<(uint32_t)blocks, 256, 0, s>>>(c, bt, a)));
    }
    GVDB_LAUNCH_CHECK();
    if (a.lanes) {  // few units: a row and head a wave
        const uint32_t joins = (bt.rows * a.q_heads + 3) / 4;
        KV_DISPATCH(c.dim, a.q.dtype, (k_kv_combine<D, T, true, false><<<joins, 256, 0, s>>>(c, bt, a)));
        GVDB_LAUNCH_CHECK();
    }
    return hipSuccess;
}

}  // namespace gvdb
