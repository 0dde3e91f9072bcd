// Block tables, slot map and positions of a batch, from the requests' lengths, on the device.
//
// For request r with L cached and n new tokens (n < 0: it has ended and gives its pages back), on a stack of free pages:
//   rows:   its n rows are rows [R, R + n) of the batch, R the sum of max(n, 0) over the requests before it;
//   pages:  it needs max(0, ceil((L + n) / 256) - held) more; the ended ones' pages are pushed first, in request order, then the
//           needed ones are popped in request order, so page j of all that are needed is entry top - 1 - j of the stack;
//   slots:  its row i is at position L + i, in slot table[r][position / 256] * 256 + position % 256.
// That is three running totals over the requests and a search in them for each row.  None of it is work -- 8 bytes written per row --
// so the launch is a chain of round trips, and a second launch, or workgroups that wait for each other, would cost more than the
// totals do: every workgroup makes them for itself in LDS (of at most kMaxRequests requests) and takes its share of the rows and
// pages.  Nothing that a workgroup reads is written by another one: pages that change hands are looked up where they were before
// the call (the ended requests' table rows, the stack below its old top), and every other output is memory of its own.
#include "common.h"

#include <algorithm>

namespace cpmcu {
namespace {

constexpr int kMaxRequests = 4096;
constexpr int kMaxBlocks = 1 << 18;   // 2^26 tokens of a request; the pages of kMaxRequests such requests add up in 32 bits
constexpr int kMaxRows = 1 << 30;     // (the totals of rows stop at the capacity)
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kRowsPerThread = 4;     // one 16-byte piece of positions and one of slots

struct TableParams {
    const int32_t *kv_lens, *new_lens, *held, *counts;
    int32_t *tables, *free_pages, *kv_lens_out, *held_out, *counts_out, *row_offsets, *positions, *slots;
    int B, M, num_pages, max_rows;
    bool wide;  // positions and slots lie on 16 bytes
};

// The first of totals[0..n) above x, n if there is none (totals never fall).
__device__ inline int first_above(const int* totals, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (totals[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The total of the threads before this one, and of all of them, each `cap` at most (totals that stop at a cap can be added up in any grouping).
__device__ inline int block_total(int v, int cap, int* wave_total, int* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v = min(v + o, cap);
    }
    if (lane == 63) wave_total[wave] = v;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) before = sum;
        sum = min(sum + wave_total[w], cap);
    }
    __syncthreads();
    *all = sum;
    v = __shfl_up(v, 1);
    return lane == 0 ? before : min(before + v, cap);
}

__global__ __launch_bounds__(kThreads) void batch_tables_kernel(TableParams p) {
    // running totals of rows, needed pages and pages given back; and each request's cached length, -1 where no row of it has a slot
    __shared__ int row_end[kMaxRequests], need_end[kMaxRequests], back_end[kMaxRequests], length[kMaxRequests];
    __shared__ int wave_total[kWaves], granted, refused;
    const int tid = threadIdx.x, B = p.B, M = p.M;
    const int each = (B + kThreads - 1) / kThreads, r0 = min(tid * each, B), r1 = min(r0 + each, B);  // this thread's requests
    const int row_cap = p.max_rows + 1;  // more rows than there is room for
    const auto held_by = [&](int r) { return min(max(p.held[r], 0), M); };

    int rows = 0, back = 0, need = 0, lacking = 0, all_rows, all_back, all_need;
    for (int r = r0; r < r1; ++r) {
        const int n = p.new_lens[r];
        rows = min(rows + min(max(n, 0), row_cap), row_cap);
        if (n < 0) back += held_by(r);
    }
    if (tid == 0) granted = refused = 0;
    rows = block_total(rows, row_cap, wave_total, &all_rows);
    back = block_total(back, INT32_MAX, wave_total, &all_back);
    const int count = min(max(p.counts[0], 0), p.num_pages);
    const int top = min(count + all_back, p.num_pages);
    for (int r = r0; r < r1; ++r) {
        const int n = p.new_lens[r], h = held_by(r), len = p.kv_lens[r];
        const int64_t blocks = ((int64_t)len + max(n, 0) + kPage - 1) / kPage;
        rows = min(rows + min(max(n, 0), row_cap), row_cap);
        if (n < 0) back += h;
        const bool bad = n >= 0 && (len < 0 || blocks > M || (n > 0 && rows > p.max_rows));
        if (n >= 0 && !bad) need += max(0, (int)blocks - h);
        lacking += bad;
        row_end[r] = rows;
        back_end[r] = back;
        need_end[r] = need;
        length[r] = n < 0 || bad ? -1 : len;
    }
    const int need_before = block_total(need, INT32_MAX, wave_total, &all_need);
    int last = 0, served = 0;
    for (int r = r0; r < r1; ++r) {
        const int end = need_end[r];
        need_end[r] = need_before + end;
        if (end > last) {
            if (need_before + end > top) {
                length[r] = -1;
                ++lacking;
            } else {
                served = need_before + end;
            }
        }
        last = end;
    }
    if (served > 0) atomicMax(&granted, served);
    if (lacking > 0) atomicAdd(&refused, lacking);
    __syncthreads();

    const auto begin = [&](const int* totals, int r) { return r > 0 ? totals[r - 1] : 0; };
    const auto on_stack = [&](int at) {  // entry `at` of the stack with the ended requests' pages on it
        if (at < count) return p.free_pages[at];
        const int i = at - count, r = first_above(back_end, B, i);
        return p.tables[(size_t)r * M + i - begin(back_end, r)];
    };
    const int first = blockIdx.x * kThreads + tid, threads = gridDim.x * kThreads;
    for (int g = first; g * kRowsPerThread < p.max_rows; g += threads) {
        int at[kRowsPerThread], slot[kRowsPerThread];
        const int i0 = g * kRowsPerThread;
        int r = -1, lo = 0, hi = 0, h = 0, b_known = -1, page = -1;  // the request whose rows are [lo, hi), and its page b_known
#pragma unroll
        for (int j = 0; j < kRowsPerThread; ++j) {
            const int i = i0 + j;
            at[j] = slot[j] = -1;
            if (i >= min(all_rows, p.max_rows)) continue;
            if (i >= hi) {
                r = first_above(row_end, B, i);
                lo = begin(row_end, r);
                hi = row_end[r];
                h = held_by(r);
                b_known = -1;
            }
            if (length[r] < 0) continue;
            at[j] = length[r] + (i - lo);
            const int b = at[j] / kPage;
            if (b != b_known) {
                b_known = b;
                page = b < h ? p.tables[(size_t)r * M + b] : on_stack(top - 1 - (begin(need_end, r) + b - h));
            }
            if ((unsigned)page < (unsigned)p.num_pages) slot[j] = page * kPage + at[j] % kPage;
        }
        if (p.wide && i0 + kRowsPerThread <= p.max_rows) {
            *reinterpret_cast<int4*>(p.positions + i0) = make_int4(at[0], at[1], at[2], at[3]);
            *reinterpret_cast<int4*>(p.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
#pragma unroll
            for (int j = 0; j < kRowsPerThread; ++j) {
                if (i0 + j >= p.max_rows) break;
                p.positions[i0 + j] = at[j];
                p.slots[i0 + j] = slot[j];
            }
        }
    }
    for (int i = first; i < all_back; i += threads) {
        const int r = first_above(back_end, B, i);
        if (count + i < p.num_pages) p.free_pages[count + i] = p.tables[(size_t)r * M + i - begin(back_end, r)];
    }
    for (int j = first; j < granted; j += threads) {
        const int r = first_above(need_end, B, j);
        p.tables[(size_t)r * M + held_by(r) + j - begin(need_end, r)] = on_stack(top - 1 - j);
    }
    if (blockIdx.x != 0) return;
    for (int r = tid; r < B; r += kThreads) {
        const int n = p.new_lens[r];
        const bool has = length[r] >= 0;
        p.kv_lens_out[r] = has ? length[r] + n : n < 0 ? 0 : p.kv_lens[r];
        p.held_out[r] = n < 0 ? 0 : held_by(r) + (has ? need_end[r] - begin(need_end, r) : 0);
        p.row_offsets[r + 1] = min(row_end[r], p.max_rows);
    }
    if (tid == 0) {
        p.row_offsets[0] = 0;
        p.counts_out[0] = top - granted;
        p.counts_out[1] = refused;
    }
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const char *x = (const char*)a, *y = (const char*)b;
    return x < y + nb && y < x + na;
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" int cpmcu_batch_tables(const int32_t* kv_lens, const int32_t* new_lens, int num_requests, int32_t* block_tables, int max_blocks,
                                  const int32_t* held, int32_t* free_pages, int num_pages, const int32_t* counts, int32_t* kv_lens_out,
                                  int32_t* held_out, int32_t* counts_out, int32_t* row_offsets, int32_t* positions, int32_t* slots, int max_rows,
                                  void* stream) {
    CPMCU_CHECK_ARG(kv_lens && new_lens && block_tables && held && free_pages && counts && kv_lens_out && held_out && counts_out && row_offsets,
                    "batch_tables: null pointer argument");
    CPMCU_CHECK_ARG(num_requests >= 1 && num_requests <= kMaxRequests, "batch_tables: %d requests outside [1, %d]", num_requests, kMaxRequests);
    CPMCU_CHECK_ARG(max_blocks >= 1 && max_blocks <= kMaxBlocks, "batch_tables: max_blocks=%d outside [1, %d]", max_blocks, kMaxBlocks);
    CPMCU_CHECK_ARG(num_pages >= 1 && num_pages <= INT32_MAX / kPage, "batch_tables: num_pages=%d outside [1, %d]", num_pages, INT32_MAX / kPage);
    CPMCU_CHECK_ARG(max_rows >= 0 && max_rows <= kMaxRows, "batch_tables: max_rows=%d outside [0, %d]", max_rows, kMaxRows);
    CPMCU_CHECK_ARG(max_rows == 0 || (positions && slots), "batch_tables: null pointer argument");
    // Workgroups read these inputs while others write the outputs: none may be the same memory.
    const size_t n = sizeof(int32_t) * (size_t)num_requests;
    const struct { const void* at; size_t bytes; } in[] = {{kv_lens, n}, {new_lens, n}, {held, n}, {counts, 4}, {block_tables, n * max_blocks}, {free_pages, 4 * (size_t)num_pages}},
        out[] = {{kv_lens_out, n}, {held_out, n}, {counts_out, 8}, {row_offsets, n + 4}, {positions, 4 * (size_t)max_rows}, {slots, 4 * (size_t)max_rows}};
    for (const auto& o : out)
        for (const auto& i : in) CPMCU_CHECK_ARG(!overlap(o.at, o.bytes, i.at, i.bytes), "batch_tables: an output is the memory of an input");
    TableParams p{kv_lens, new_lens, held, counts, block_tables, free_pages, kv_lens_out, held_out, counts_out, row_offsets, positions, slots,
                  num_requests, max_blocks, num_pages, max_rows, ((uintptr_t)positions | (uintptr_t)slots) % 16 == 0};
    const int grid = std::min(std::max(ceil_div(max_rows, kThreads * kRowsPerThread), 1), 1024);
    hipLaunchKernelGGL(batch_tables_kernel, dim3(grid), dim3(kThreads), 0, resolve_stream(stream), p);
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
