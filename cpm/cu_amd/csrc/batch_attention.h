// What the attention kernels of a batch share (prompt_attention.hip, decode_attention.hip): the call's tensors, and its checks.
#pragma once
#include "common.h"
#include "internal.h"

#include <cmath>

namespace cpmcu {

// Row t of q and out: Hq heads of 128 values from t * stride on.  Request r's rows are [row_offsets[r], row_offsets[r + 1]); its page of
// position x is block_tables[r * table_stride + x / 256].
struct BatchRows {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_stride, out_stride;
    const uint16_t* k_pool;
    const uint16_t* v_pool;
    const int32_t* block_tables;
    const int32_t* row_offsets;  // null: row r is request r's only one
    const int32_t* positions;
    int64_t table_stride;
    int num_requests, max_blocks, num_pages;
    int n, Hq, Hkv, group;
    uint32_t group_inverse;  // 0xffffffff / group (prompts)
    float scale_log2;  // the scores' factor times log2 e: probabilities are powers of two
};

constexpr int kMostRequests = 4096;
constexpr int kMostBlocks = 1 << 18;       // 2^26 positions of a request
constexpr int kMostTableEntries = 1 << 28; // of all requests: 2^30 tiles of 64 keys
constexpr int kTileKeys = 64;              // keys that a workgroup or a wave takes at a time; pages are whole tiles

// A row's position and a page's number as the device finds them, within what the host promised.
__device__ inline int page_within(int page, int num_pages) { return min(max(page, 0), num_pages - 1); }

// x / d and x % d for 0 <= x < 2^31 - 1 without a division: (x + 1) / d by way of d's inverse is less than one too small, so its floor is the quotient or one less.
struct Quotient {
    int q, r;
};
__device__ inline Quotient divide(int x, int d, uint32_t inverse) {
    Quotient a;
    a.q = (int)__umulhi((uint32_t)x + 1u, inverse);
    a.r = x - a.q * d;
    const bool more = a.r >= d;
    a.q += more ? 1 : 0;
    a.r -= more ? d : 0;
    return a;
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Four KB of a wave from memory to LDS, whole lines: each lane's 16 bytes of each from where it says, in lane order; the instructions add 1 KB each to both addresses.  Their arrival is
// counted by hand: written as loads that the compiler knows, every read of LDS would wait for all of them.  One statement: nothing comes between m0 and its use.
__device__ inline void request_4k(const void* base, uint32_t o0, uint32_t o1, uint32_t o2, uint32_t o3, uint32_t lds_at) {
    asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\tglobal_load_lds_dwordx4 %1, %4 offset:1024\n\t"
                 "global_load_lds_dwordx4 %2, %4 offset:2*1024\n\tglobal_load_lds_dwordx4 %3, %4 offset:3*1024"
                 : : "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(base), "s"(lds_at) : "memory", "m0");
}

inline int check_batch_rows(const char* what, const BatchRows& b, float scale) {
    CPMCU_CHECK_ARG(b.n >= 0 && b.n < 1 << 24, "%s: n=%d outside [0, 2^24)", what, b.n);
    CPMCU_CHECK_ARG(b.num_requests >= 1 && b.num_requests <= kMostRequests, "%s: %d requests outside [1, %d]", what, b.num_requests, kMostRequests);
    CPMCU_CHECK_ARG(b.max_blocks >= 1 && b.max_blocks <= kMostBlocks, "%s: max_blocks=%d outside [1, %d]", what, b.max_blocks, kMostBlocks);
    CPMCU_CHECK_ARG(b.table_stride >= b.max_blocks && b.table_stride <= INT32_MAX, "%s: rows of the tables closer than max_blocks=%d, or further apart than 2^31", what, b.max_blocks);
    CPMCU_CHECK_ARG((int64_t)b.num_requests * b.max_blocks <= kMostTableEntries, "%s: block tables of more than %d entries", what, kMostTableEntries);
    CPMCU_CHECK_ARG(b.num_pages >= 1 && b.num_pages <= INT32_MAX / kPage, "%s: num_pages=%d outside [1, %d]", what, b.num_pages, INT32_MAX / kPage);
    CPMCU_CHECK_ARG(b.Hkv >= 1 && b.Hkv <= 1024 && b.Hq >= 1 && b.Hq <= 1024 && b.Hq % b.Hkv == 0, "%s: %d query heads on %d KV heads", what, b.Hq, b.Hkv);
    CPMCU_CHECK_ARG((int64_t)b.n * b.Hq <= INT32_MAX - 4096, "%s: %d rows of %d heads are beyond 32 bits", what, b.n, b.Hq);
    CPMCU_CHECK_ARG(std::isfinite(scale) && scale > 0.f, "%s: scale=%g is not a positive number", what, (double)scale);
    if (b.n == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(b.q && b.out && b.k_pool && b.v_pool && b.block_tables && b.positions, "%s: null pointer argument", what);
    const int64_t row = (int64_t)b.Hq * kHeadDim;
    CPMCU_CHECK_ARG(b.n == 1 || (b.q_stride >= row && b.out_stride >= row), "%s: rows closer than their %d heads", what, b.Hq);
    CPMCU_CHECK_ARG(b.n == 1 || (b.q_stride <= INT32_MAX && b.out_stride <= INT32_MAX), "%s: rows further apart than 2^31 values", what);
    CPMCU_CHECK_ARG(((uintptr_t)b.q | (uintptr_t)b.out | (uintptr_t)b.k_pool | (uintptr_t)b.v_pool) % 16 == 0 && (b.n == 1 || (b.q_stride % 8 == 0 && b.out_stride % 8 == 0)),
                    "%s: rows and pools have to lie on 16 bytes", what);
    // (a page's part of a head is 64 KB; q's rows may be the results' place only row by row: a workgroup reads its own)
    const size_t pool = (size_t)b.num_pages * b.Hkv * kPage * kHeadDim * 2, ints = sizeof(int32_t);
    const size_t q_bytes = 2 * ((size_t)(b.n - 1) * b.q_stride + row), out_bytes = 2 * ((size_t)(b.n - 1) * b.out_stride + row);
    const bool in_place = (const void*)b.q == (const void*)b.out && (b.n == 1 || b.q_stride == b.out_stride);
    // rows of one stride whose columns are apart (the parts of a wider row)
    const int64_t apart = (const char*)b.out - (const char*)b.q, step = 2 * b.q_stride;
    const int64_t column = b.n > 1 && b.q_stride == b.out_stride ? ((apart % step) + step) % step : 0;
    const bool columns = b.n > 1 && b.q_stride == b.out_stride && column >= 2 * row && column + 2 * row <= step;
    CPMCU_CHECK_ARG(in_place || columns || !overlap(b.q, q_bytes, b.out, out_bytes), "%s: the results lie in other rows of q", what);
    CPMCU_CHECK_ARG(!overlap(b.k_pool, pool, b.out, out_bytes) && !overlap(b.v_pool, pool, b.out, out_bytes), "%s: the results lie in the pools", what);
    CPMCU_CHECK_ARG(!overlap(b.block_tables, ints * ((size_t)(b.num_requests - 1) * b.table_stride + b.max_blocks), b.out, out_bytes) && !overlap(b.positions, ints * b.n, b.out, out_bytes) &&
                        !(b.row_offsets && overlap(b.row_offsets, ints * (b.num_requests + 1), b.out, out_bytes)),
                    "%s: the results lie in the tables, offsets or positions", what);
    return CPMCU_OK;
}

}  // namespace cpmcu
