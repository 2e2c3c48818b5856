// gvdb_kv.h — the token cache's launch interface, between its C ABI
// (gvdb_kv_capi.hip) and its kernels (gvdb_kv.hip).
#pragma once
#include "../../include/gvdb.h"
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gvdb {

constexpr uint32_t kChooseScores = 15360;  // page scores that a choosing workgroup keeps in LDS: two workgroups a CU
constexpr uint64_t kScoreBytes = 64ull << 20;  // page scores that a call keeps in scratch: rows are scored and chosen for in groups that fit
constexpr uint32_t kMaxUnits = 2048;  // sequences or rows that a balanced launch takes

struct KvCache {
    uint8_t* pool;
    int8_t* bounds;
    uint8_t* bound_exps;
    uint64_t n_pages;
    uint32_t heads, dim, page;
};

struct KvBatch {
    const int32_t* table;
    uint64_t table_stride;
    uint32_t table_width, n_seqs;
    const int32_t *lengths, *cu;
    uint32_t rows;
    uint32_t max_new, max_len;  // hints, at least 1: they size the grid, never what is computed
};

struct KvRows {
    void* p;
    uint32_t dtype;
    int64_t row_stride, head_stride;  // elements
    bool wide;                        // base and strides are multiples of 16 bytes
    bool zero_rest;                   // outputs: rows of no sequence become 0
};

struct AttendArgs {
    KvRows q, out;
    float* lse;
    uint32_t q_heads;
    float scale_log2;  // |scale| * log2(e), over 0
    int32_t negate;    // scale < 0: the queries change sign
    int32_t causal;
    uint32_t row_tiles;        // tiles of query rows in the grid, a sequence (chosen pages: a token): 16 rows, `many`: 128
    bool many;
    uint32_t splits, chunk;    // parts along the keys, and the tiles of each
    // the line: `lanes` waves (four a workgroup) a key head share the tiles of `units` units evenly; a unit is 16 rows (slot_rows: fewer,
    // where a sequence or token has fewer) of a sequence, or, over chosen pages, of a token: row_tiles units each
    uint32_t units, lanes, least, slot_rows;  // lanes = 0: one workgroup a tile of rows and split
    uint32_t* prefix;          // [units + 1]: tiles before each unit, left for the join
    float *part_o, *part_ml;   // [rows][q_heads][splits][D]; the line: [heads][lanes + units][slot_rows][D]; and [..][2]
    // chosen pages
    uint32_t top, first, recent;
    uint32_t score_chunk;      // pages a workgroup scores into `scores`; 0: scored and chosen by one workgroup in LDS
    uint32_t score_rows;       // rows whose scores `scores` holds at a time
    int32_t* chosen;           // [rows][heads][top]
    float* scores;             // [score_rows][heads][table_width]

    // Pages that hold a query's visible tokens; one beyond the table where the table is too short.
    __host__ __device__ int64_t pages_seen(const KvCache& c, const KvBatch& bt, int64_t limit) const {
        const int64_t want = limit <= 0 ? 0 : (limit + c.page - 1) / c.page;
        return want <= (int64_t)bt.table_width ? want : (int64_t)bt.table_width + 1;
    }
    // The sequence of a row of q; false: the row lies behind the last sequence.
    __device__ bool row_seq(const KvBatch& bt, int row, uint32_t& b) const {
        if (!bt.cu) {
            b = (uint32_t)row / (bt.rows / bt.n_seqs);
            return true;
        }
        uint32_t lo = 0, hi = bt.n_seqs;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (bt.cu[mid + 1] <= row) lo = mid + 1;
            else hi = mid;
        }
        b = lo;
        return lo < bt.n_seqs && bt.cu[lo] <= row;
    }
};

// Pages that a sequence of max_len tokens takes, within the table.
inline uint32_t kv_max_pages(const KvCache& c, const KvBatch& bt) {
    const uint64_t p = ((uint64_t)bt.max_len + c.page - 1) / c.page;
    return (uint32_t)(p < 1 ? 1 : p > bt.table_width ? bt.table_width : p);
}

hipError_t launch_kv_append(const KvCache& c, const KvBatch& bt, const KvRows& k, const KvRows& v, hipStream_t s);
hipError_t launch_kv_read(const KvCache& c, const KvBatch& bt, const KvRows& k, const KvRows& v, hipStream_t s);
hipError_t launch_kv_attend(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s);
hipError_t launch_kv_attend_topk(const KvCache& c, const KvBatch& bt, const AttendArgs& a, hipStream_t s);

}  // namespace gvdb
