// gvdb_kv_capi.hip — C ABI of the token cache (include/gvdb.h, gvdb_kv_*):
// checks of arguments, the split of the work, the scratch layout.
#include <algorithm>
#include <cmath>
#include <string>

#include "gvdb_internal.h"
#include "gvdb_kv.h"

using namespace gvdb;

namespace {

gvdb_status invalid(const char* msg) { return report_status(GVDB_ERR_INVALID_ARGUMENT, msg); }

// Entered with the cache's device current, left with the caller's.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) {
            err = hipSetDevice(device);
        } else {
            before = -1;
        }
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// No C++ exception crosses the boundary.
template <class F>
gvdb_status guarded(F&& f) noexcept {
    try {
        return f();
    } catch (...) {
        return GVDB_ERR_OUT_OF_MEMORY;
    }
}

gvdb_status launch(int device, const char* what, hipError_t (*run)(const void*, hipStream_t), const void* args, void* stream) {
    DeviceScope scope(device);
    hipError_t e = scope.err;
    if (e == hipSuccess) e = run(args, (hipStream_t)stream);
    if (e == hipSuccess) return GVDB_OK;
    if (e == hipErrorInvalidValue) return invalid("token cache: more rows and heads than one launch takes");
    return report_status(e == hipErrorOutOfMemory ? GVDB_ERR_OUT_OF_MEMORY : GVDB_ERR_DEVICE,
                         std::string(what) + ": " + hipGetErrorString(e));
}

uint32_t size_of(uint32_t dtype) { return dtype == GVDB_F32 ? 4 : 2; }

gvdb_status take_cache(const gvdb_kv_cache* in, KvCache& c) {
    if (!in) return invalid("token cache: null cache");
    if (in->head_dim != 64 && in->head_dim != 128 && in->head_dim != 256)
        return report_status(GVDB_ERR_INVALID_VECTOR_DIMENSION, "token cache: head_dim is 64, 128 or 256");
    if (in->page_size == 0 || in->page_size % 32 || in->page_size > 1024)
        return invalid("token cache: page_size is a multiple of 32, at most 1024");
    if (in->kv_heads == 0 || in->kv_heads > 4096) return invalid("token cache: kv_heads is 1 .. 4096");
    if (in->n_pages == 0 || in->n_pages > (1ull << 31)) return invalid("token cache: n_pages is 1 .. 2^31");
    if (in->device < 0) return invalid("token cache: negative device");
    if (!in->pool || !in->bounds || !in->bound_exps) return invalid("token cache: null buffer");
    if (((uintptr_t)in->pool | (uintptr_t)in->bounds) & 15u) return invalid("token cache: pool and bounds are 16-byte aligned");
    c = {in->pool, in->bounds, in->bound_exps, in->n_pages, in->kv_heads, in->head_dim, in->page_size};
    return GVDB_OK;
}

gvdb_status take_batch(const gvdb_kv_batch* in, const KvCache& c, KvBatch& bt) {
    if (!in) return invalid("token cache: null batch");
    if (in->rows > 0x7FFFFFFFu) return invalid("token cache: over 2^31 - 1 rows");
    if (in->rows == 0) {
        bt = {};
        return GVDB_OK;
    }
    if (in->n_seqs == 0 || in->n_seqs > 0x7FFFFFFFu) return invalid("token cache: rows without a sequence");
    if (!in->page_table || !in->lengths) return invalid("token cache: null page_table or lengths");
    if (in->table_width == 0 || in->table_width > 0x7FFFFFFFu / c.page) return invalid("token cache: table_width * page_size is 1 .. 2^31 - 1");
    if (in->n_seqs > 1 && in->table_stride < in->table_width) return invalid("token cache: table_stride below table_width");
    if (!in->cu && in->rows % in->n_seqs) return invalid("token cache: without cu, rows is a multiple of n_seqs");
    bt = {in->page_table, in->table_stride, in->table_width, in->n_seqs, in->lengths, in->cu, in->rows, in->max_new, in->max_len};
    // hints: never over what the sizes allow
    if (!bt.cu) bt.max_new = bt.rows / bt.n_seqs;
    if (bt.max_new == 0 || bt.max_new > bt.rows) bt.max_new = bt.rows;
    const uint64_t most = (uint64_t)bt.table_width * c.page;
    if (bt.max_len == 0 || bt.max_len > most) bt.max_len = (uint32_t)most;
    return GVDB_OK;
}

gvdb_status take_rows(const gvdb_kv_rows* in, const char* what, KvRows& r) {
    if (!in || !in->data) return invalid((std::string("token cache: null ") + what).c_str());
    if (in->dtype > GVDB_BF16) return invalid((std::string("token cache: unknown dtype of ") + what).c_str());
    const uint32_t size = size_of(in->dtype);
    if ((uintptr_t)in->data % size) return invalid((std::string("token cache: misaligned ") + what).c_str());
    if (in->flags > GVDB_KV_ZERO_REST) return invalid((std::string("token cache: unknown flags of ") + what).c_str());
    r = {in->data, in->dtype, in->row_stride, in->head_stride, false, in->flags == GVDB_KV_ZERO_REST};
    r.wide = ((uint64_t)(uintptr_t)in->data | (uint64_t)in->row_stride * size | (uint64_t)in->head_stride * size) % 16 == 0;
    return GVDB_OK;
}

// Whether two of [rows][heads] runs of d elements share an element: their starts lie i * rs + j * hs apart, |i| < rows, |j| < heads.
bool overlapping(uint64_t rows, uint64_t heads, int64_t row_stride, int64_t head_stride, uint64_t d) {
    typedef unsigned __int128 wide;
    auto size = [](int64_t x) { return x < 0 ? 0 - (uint64_t)x : (uint64_t)x; };
    const uint64_t rs = size(row_stride), hs = size(head_stride);
    if ((rows > 1 && rs < d) || (heads > 1 && hs < d)) return true;
    if (rows < 2 || heads < 2 || rs >= (wide)(heads - 1) * hs + d || hs >= (wide)(rows - 1) * rs + d) return false;
    // one inside the other, otherwise than [rows][heads] or [heads][rows]: both strides are d or more, so only i and j whose offsets
    // take from one another can meet, and for each head the two rows next to it
    for (uint64_t j = 1; j < heads; ++j) {
        const wide at = (wide)j * hs, i = at / rs;
        if ((i < rows && at - i * rs < d) || (i + 1 < rows && (i + 1) * rs - at < d)) return true;
    }
    return false;
}

// Rows that are written lie apart: two that share an element would be written in any order.
gvdb_status take_out(const gvdb_kv_rows* in, const char* what, const KvCache& c, uint32_t rows, uint32_t heads, KvRows& r) {
    if (gvdb_status s = take_rows(in, what, r)) return s;
    if (overlapping(rows, heads, r.row_stride, r.head_stride, c.dim))
        return invalid((std::string("token cache: overlapping rows of ") + what).c_str());
    return GVDB_OK;
}

uint64_t up256(uint64_t n) { return (n + 255) / 256 * 256; }

// How the work is cut, and where in the scratch each part lies.
struct Plan {
    AttendArgs a{};
    uint64_t scores = 0, chosen = 0, part_o = 0, part_ml = 0, prefix = 0, bytes = 0;
};

gvdb_status plan_attend(const KvCache& c, const KvBatch& bt, uint32_t dtype, uint32_t q_heads, uint32_t top, Plan& p) {
    if (q_heads == 0 || q_heads % c.heads || q_heads > 65536)
        return invalid("token cache: q_heads is a multiple of kv_heads, at most 65536");
    if (top > 65536) return invalid("token cache: top is at most 65536");
    const uint64_t group = q_heads / c.heads;
    AttendArgs& a = p.a;
    a.q_heads = q_heads;
    a.top = top;
    const uint64_t tiles = top ? (uint64_t)std::min(top, bt.table_width) * (c.page / 32) : ((uint64_t)bt.max_len + 31) / 32;
    const uint64_t rows_each = top ? group : bt.max_new * group;
    const uint64_t units0 = top ? bt.rows : bt.n_seqs;
    // Workgroups that have rows, of `w` rows each: with `cu` the sequences are of several lengths, and `rows` says how many there are in all.
    auto busy_of = [&](uint64_t w, uint64_t n_units) { return std::min(n_units, (bt.rows * group / w + bt.n_seqs) * c.heads); };
    // As many workgroups as the card's registers hold at once: three a CU of 64 channels, two of 128, one of 256.  128 channels, 8 heads,
    // 64 sequences of up to 10000 tokens: 64 us with one, 58 with two, 66 with four; 4 x 262144 tokens: 230, 204, 237 us; 256 channels,
    // 4 heads, 64 sequences of up to 20000: 150 us with half a one, 96 with one, 102 with two; 64 channels, 8 heads: 66 us with two, 63
    // with three.
    const uint64_t slots = c.dim == 256 ? 256 : c.dim == 128 ? 512 : 768;
    // Workgroups of 128 rows share the values' expansion, and run in rounds.  A round of m workgroups a CU takes about (m + 1) / 2 times
    // what one of a single one does, 8 tiles' time before its first tile, and a join as much again; in units of half a tile (0.36 us
    // at 64 channels, 0.53 at 128, 0.8 at 256), with the number of parts that takes least (2 sequences of 300 tokens over 5000: 3 parts
    // 109 us, 5 125, 1 160; 6 of 256 over 1500: 1 82, 3 106).
    const uint64_t busy128 = busy_of(128, units0 * c.heads * ((rows_each + 127) / 128));
    uint64_t time128 = ~0ull, parts128 = 1;
    for (uint64_t k = 1; k <= std::max<uint64_t>(1, tiles / 16) && k <= 64; ++k) {
        const uint64_t blocks = busy128 * k, rest = blocks % slots;
        const uint64_t time = ((tiles + k - 1) / k + 8) * (blocks / slots * (slots / 256 + 1) + (rest ? (rest + 255) / 256 + 1 : 0)) + (k > 1 ? 16 : 0);
        if (time < time128) time128 = time, parts128 = k;
    }
    // By 16 rows the card does 800 tiles (64 channels: 1000) in one of these units, 5 go by before a workgroup's first, and a join where
    // they are too few to go whole.  16 sequences of 64 tokens over 900, 4 heads a group: 41 us by 128 rows, 27 by 16; 64 over 300 58 and
    // 90; 2 over 16000 53 and 56; 2 of 2048 over 10000, 8 heads: 837 and 1156.  In 32 bits the pieces do not fit the registers: 130 and
    // 117 us at 512 rows.
    const uint64_t busy16 = busy_of(16, units0 * c.heads * ((rows_each + 15) / 16));
    a.many = !top && dtype != GVDB_F32 && rows_each >= 128 && time128 < 5 + busy16 * (tiles + 5) / (c.dim == 64 ? 1000 : 800) + (busy16 < 512 ? 14 : 0);
    uint64_t row_tiles = a.many ? (rows_each + 127) / 128 : (rows_each + 15) / 16;
    // grids stay below 2^20 tiles of rows where the hints are loose: the kernels stride over the rest
    row_tiles = std::max<uint64_t>(1, std::min<uint64_t>(row_tiles, (1ull << 20) / std::max<uint64_t>(1, units0 * c.heads) + 1));
    const uint64_t units = units0 * c.heads * row_tiles;
    const uint64_t busy = top ? units : busy_of(a.many ? 128 : 16, units);
    // Whole, a unit of 16 rows takes 6 us and 0.17 a tile; shared, all of them 14 us (the join's launch among it) and their share of the
    // card.  Units of one length (chosen pages, one sequence's rows) are shared while few and long: 8 units of 47 tiles 15 us and 14 whole,
    // of 125 15 and 27, 128 of 125 27 and 28, 256 of 188 53 and 48, 192 of 128 chosen 52 and 50.  Sequences of several lengths leave
    // a card of whole units uneven: 512 of up to 63 tiles 25 us and 20 whole, of up to 188 40 and 47, 2000 of up to 125 94 and 91, of up
    // to 313 188 and 209.
    const bool known = !bt.cu || bt.n_seqs == 1;  // how many rows a sequence has
    const bool shared = a.many ? known || (busy < 1024 && tiles > 32)
                        : top || bt.n_seqs == 1 ? units < 200 && tiles * (200 - units) > 9000
                                                : tiles > 48 + units / 8;
    a.row_tiles = (uint32_t)row_tiles;
    a.splits = 1;
    a.chunk = (uint32_t)(tiles + 1) / 2 * 2;
    if (shared) {
        const uint64_t line = units0 * ((rows_each + 15) / 16);
        const uint64_t most = line * (top ? (uint64_t)top : (uint64_t)bt.table_width + 1) * (c.page / 32);
        // chosen pages: fewer than 200 units of at most 65536 pages of 32 tiles, so that a call that shares takes the line
        if (!a.many && (top || !bt.cu) && line <= kMaxUnits && most < (1ull << 31)) {
            // the rows of a unit are known: every wave gets the same share of all tiles, of 4 at least; of long sequences more, for the
            // join's sake, as below (8 heads, one sequence of 125 tiles: 13 us by 4, 16 by 8; of 938 26 and 21)
            a.units = (uint32_t)line;
            a.lanes = (uint32_t)std::max<uint64_t>(1, slots / c.heads) * 4;
            a.least = std::max<uint32_t>(4, (uint32_t)std::sqrt((double)tiles) / 4);
            a.slot_rows = (uint32_t)std::min<uint64_t>(16, rows_each);
            a.row_tiles = (uint32_t)((rows_each + 15) / 16);
        } else if (a.many && known) {
            a.splits = (uint32_t)parts128;
            a.chunk = (uint32_t)((tiles + a.splits - 1) / a.splits + 1) / 2 * 2;
            a.splits = (uint32_t)((tiles + a.chunk - 1) / a.chunk);
        } else {
            // parts for 2048 workgroups of 128 rows, of which about a third find keys (2 sequences of up to 500 tokens over 30000: 421 us,
            // for 1024 of them 447, for 512 525), or 2560 of 16 rows (5 tokens of 32 sequences over up to 20000: 81 us, for 1536 85, for
            // 768 121).  Of 16 tiles at least, for 128 rows; of 16 rows a part's time grows with its tiles and the join's with the parts,
            // so of the square root of all tiles (best of 6 .. 32: 94 tiles 8 to 12, 250 12 to 16, 625 24, 938 32)
            const uint64_t parts = a.many ? 2048 : 2560, least = a.many ? 16 : std::max<uint64_t>(8, (uint64_t)std::sqrt((double)tiles));
            a.chunk = (uint32_t)((std::max(least, (busy * tiles + parts - 1) / parts) + 1) / 2 * 2);  // whole steps
            a.splits = (uint32_t)((tiles + a.chunk - 1) / a.chunk);
        }
    }
    if (units * a.splits > 0x7FFFFFFFull) return invalid("token cache: too many rows and heads for one call");
    const uint64_t qr = (uint64_t)bt.rows * q_heads;
    uint64_t at = 0;
    if (top) {
        // Scores go by way of memory where LDS does not hold them, and where few tokens have many pages: all CUs score, 30 us for one
        // sequence of 1024 pages against 33 by one workgroup a head, 53 against 55 for 32 sequences; 384 tokens of a prompt take 35 us
        // in LDS and 82 by way of memory.
        const bool split = bt.table_width > kChooseScores || (kv_max_pages(c, bt) > 512 && (uint64_t)bt.rows * c.heads <= 1024);
        // 256 pages a workgroup, 64 a wave; 128 where that leaves CUs idle (one sequence of 1024 pages, 8 heads: 31 and 29 us)
        a.score_chunk = !split ? 0 : (uint64_t)bt.rows * c.heads * kv_max_pages(c, bt) < 65536 ? 128 : 256;
        if (split) {
            // tables of over 15360 pages: a prompt's scores would take gigabytes (2048 tokens, 8 heads, 32768 pages: 2 GiB)
            const uint64_t row_bytes = (uint64_t)c.heads * bt.table_width * 4;
            a.score_rows = (uint32_t)std::min<uint64_t>(bt.rows, std::max<uint64_t>(1, kScoreBytes / row_bytes));
            p.scores = at;
            at += up256(a.score_rows * row_bytes);
        }
        p.chosen = at;
        at += up256((uint64_t)bt.rows * c.heads * top * 4);
    }
    const uint64_t parts = a.lanes ? c.heads * (uint64_t)(a.lanes + a.units) * a.slot_rows : a.splits > 1 ? qr * a.splits : 0;
    if (parts) {
        p.part_o = at;
        at += up256(parts * c.dim * 4);
        p.part_ml = at;
        at += up256(parts * 8);
    }
    if (a.lanes) {
        p.prefix = at;
        at += up256((a.units + 1) * 4);
    }
    p.bytes = at;
    return GVDB_OK;
}

struct KvCall {
    KvCache c;
    KvBatch bt;
    KvRows k, v;
    AttendArgs a;
};

gvdb_status attend(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, const gvdb_kv_rows* q, uint32_t q_heads, float scale,
                   int32_t causal, uint32_t top, uint32_t first, uint32_t recent, const gvdb_kv_rows* out, int32_t* chosen,
                   float* lse, void* scratch, uint64_t scratch_bytes, bool choose, void* stream) {
    KvCall call{};
    if (gvdb_status s = take_cache(cache, call.c)) return s;
    if (gvdb_status s = take_batch(batch, call.c, call.bt)) return s;
    if (choose && top == 0) return invalid("token cache: top is at least 1");
    if (choose && (uint64_t)first + recent > top) return invalid("token cache: first + recent is at most top");
    const float base2 = std::fabs(scale) * 1.4426950408889634f;
    if (!std::isfinite(base2)) return invalid("token cache: scale is not finite, or is not times log2(e)");
    if (call.bt.rows == 0) return GVDB_OK;
    Plan p;
    KvRows qr, orow;
    if (gvdb_status s = take_rows(q, "q", qr)) return s;
    if (gvdb_status s = plan_attend(call.c, call.bt, qr.dtype, q_heads, choose ? top : 0, p)) return s;
    if (gvdb_status s = take_out(out, "out", call.c, call.bt.rows, q_heads, orow)) return s;
    p.a.q = qr, p.a.out = orow;
    if (p.a.q.dtype != p.a.out.dtype) return invalid("token cache: q and out are of one dtype");
    if (p.bytes && !scratch) return invalid("token cache: null scratch");
    if (scratch_bytes < p.bytes) return invalid("token cache: scratch below gvdb_kv_scratch_bytes");
    if ((uintptr_t)scratch & 15u) return invalid("token cache: scratch is 16-byte aligned");
    AttendArgs& a = p.a;
    uint8_t* base = (uint8_t*)scratch;
    a.lse = lse;
    // a scale of 0 (every token alike) is the least that there is, which no finite score notices: -inf times it has to stay -inf
    a.scale_log2 = std::max(base2, 0x1p-149f);
    a.negate = scale < 0;
    a.causal = causal != 0;
    a.first = first;
    a.recent = recent;
    a.part_o = (float*)(base + p.part_o);
    a.part_ml = (float*)(base + p.part_ml);
    a.prefix = (uint32_t*)(base + p.prefix);
    a.scores = (float*)(base + p.scores);
    a.chosen = chosen ? chosen : (int32_t*)(base + p.chosen);
    call.a = a;
    if (choose)
        return launch(cache->device, "kv_attend_topk",
                      [](const void* x, hipStream_t s) { auto& k = *(const KvCall*)x; return launch_kv_attend_topk(k.c, k.bt, k.a, s); },
                      &call, stream);
    return launch(cache->device, "kv_attend",
                  [](const void* x, hipStream_t s) { auto& k = *(const KvCall*)x; return launch_kv_attend(k.c, k.bt, k.a, s); }, &call,
                  stream);
}

}  // namespace

extern "C" {

gvdb_status gvdb_kv_append_device(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, const gvdb_kv_rows* k,
                                  const gvdb_kv_rows* v, void* stream) {
    return guarded([&]() -> gvdb_status {
        KvCall call{};
        if (gvdb_status s = take_cache(cache, call.c)) return s;
        if (gvdb_status s = take_batch(batch, call.c, call.bt)) return s;
        if (call.bt.rows == 0) return GVDB_OK;
        if (gvdb_status s = take_rows(k, "k", call.k)) return s;
        if (gvdb_status s = take_rows(v, "v", call.v)) return s;
        if (call.k.dtype != call.v.dtype) return invalid("token cache: k and v are of one dtype");
        return launch(cache->device, "kv_append",
                      [](const void* x, hipStream_t s) { auto& a = *(const KvCall*)x; return launch_kv_append(a.c, a.bt, a.k, a.v, s); },
                      &call, stream);
    });
}

gvdb_status gvdb_kv_read_device(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, const gvdb_kv_rows* k,
                                const gvdb_kv_rows* v, void* stream) {
    return guarded([&]() -> gvdb_status {
        KvCall call{};
        if (gvdb_status s = take_cache(cache, call.c)) return s;
        if (gvdb_status s = take_batch(batch, call.c, call.bt)) return s;
        if (call.bt.rows == 0 || (!k && !v)) return GVDB_OK;
        if (k)
            if (gvdb_status s = take_out(k, "k", call.c, call.bt.rows, call.c.heads, call.k)) return s;
        if (v)
            if (gvdb_status s = take_out(v, "v", call.c, call.bt.rows, call.c.heads, call.v)) return s;
        if (k && v && call.k.dtype != call.v.dtype) return invalid("token cache: k and v are of one dtype");
        return launch(cache->device, "kv_read",
                      [](const void* x, hipStream_t s) { auto& a = *(const KvCall*)x; return launch_kv_read(a.c, a.bt, a.k, a.v, s); },
                      &call, stream);
    });
}

gvdb_status gvdb_kv_scratch_bytes(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, uint32_t q_heads, uint32_t top,
                                  uint64_t* bytes) {
    return guarded([&]() -> gvdb_status {
        if (!bytes) return invalid("token cache: null bytes");
        *bytes = 0;
        KvCache c{};
        KvBatch bt{};
        if (gvdb_status s = take_cache(cache, c)) return s;
        if (gvdb_status s = take_batch(batch, c, bt)) return s;
        if (bt.rows == 0) return GVDB_OK;
        for (uint32_t dtype : {GVDB_F32, GVDB_BF16}) {  // enough for either
            Plan p;
            if (gvdb_status s = plan_attend(c, bt, dtype, q_heads, top, p)) return s;
            *bytes = std::max(*bytes, p.bytes);
        }
        return GVDB_OK;
    });
}

gvdb_status gvdb_kv_attend_path(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, uint32_t dtype, uint32_t q_heads,
                                uint32_t top, uint32_t* path) {
    return guarded([&]() -> gvdb_status {
        if (!path) return invalid("token cache: null path");
        *path = GVDB_KV_UNITS;
        KvCache c{};
        KvBatch bt{};
        if (gvdb_status s = take_cache(cache, c)) return s;
        if (gvdb_status s = take_batch(batch, c, bt)) return s;
        if (dtype > GVDB_BF16) return invalid("token cache: unknown dtype");
        if (bt.rows == 0) return GVDB_OK;
        Plan p;
        if (gvdb_status s = plan_attend(c, bt, dtype, q_heads, top, p)) return s;
        const bool parts = p.a.splits > 1;
        *path = p.a.lanes ? GVDB_KV_LINE : p.a.many ? (parts ? GVDB_KV_ROW_PARTS : GVDB_KV_ROWS) : parts ? GVDB_KV_PARTS : GVDB_KV_UNITS;
        return GVDB_OK;
    });
}

gvdb_status gvdb_kv_attend_device(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, const gvdb_kv_rows* q, uint32_t q_heads,
                                  float scale, int32_t causal, const gvdb_kv_rows* out, float* lse, void* scratch,
                                  uint64_t scratch_bytes, void* stream) {
    return guarded([&] {
        return attend(cache, batch, q, q_heads, scale, causal, 0, 0, 0, out, nullptr, lse, scratch, scratch_bytes, false, stream);
    });
}

gvdb_status gvdb_kv_attend_topk_device(const gvdb_kv_cache* cache, const gvdb_kv_batch* batch, const gvdb_kv_rows* q,
                                       uint32_t q_heads, float scale, uint32_t top, uint32_t first, uint32_t recent,
                                       const gvdb_kv_rows* out, int32_t* chosen, float* lse, void* scratch, uint64_t scratch_bytes,
                                       void* stream) {
    return guarded([&] {
        return attend(cache, batch, q, q_heads, scale, 1, top, first, recent, out, chosen, lse, scratch, scratch_bytes, true, stream);
    });
}

}  // extern "C"
