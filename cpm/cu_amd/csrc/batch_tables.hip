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
constexpr int kMaxRows = 1 << 29;     // (the totals of rows stop behind the capacity; two of them have to add up)

struct TableParams {
    const int32_t *kv_lens, *new_lens, *held, *counts;
    int32_t *tables, *free_pages, *kv_lens_out, *held_out, *counts_out, *row_offsets, *positions, *slots;
    int B, M, num_pages, max_rows;
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

// Inclusive running totals over a wave's lanes, each `cap` at most (totals that stop at a cap can be added up in any grouping).
__device__ inline int wave_totals(int v, int cap) {
    const auto add = [&](int from) { v = min(v + from, cap); };
    add(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // rows of 16 lanes: from 1, 2, 4 and 8 lanes before,
    add(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // lane 15 of rows 0 and 2 to the rows behind,
    add(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // lane 31 to the upper half
    return v;
}

// 256 threads with a request each where there are few, 1024 with one each up to 1024 requests, with four each beyond: a launch of 16
// requests' single rows is the round trip for their lengths, one exchange of totals, and the round trip for their pages.
// A wave looks up RUNS runs of 64 rows at once: the requests of their first rows with the whole wave in two reads of LDS, and each row's by
// halving what lies between, which is nothing where requests have many rows.  One run where a workgroup per CU covers all rows, four beyond
// (the runs' round trips overlap).  4096 requests' single rows 9.0 us with one run and 11.3 with four, a million rows of 4096 requests
// 21.2 and 16.8.  1.1 million rows of 1000 requests: 11.7 us, of which a launch that loads the lengths and ends there takes 2.2, the totals
// 1.4 more, the rows' requests and the stores 4.9 (8.8 MB, 1.8 at a copy's rate), and the loads of their pages the last 3.2.
template <int THREADS, int EACH, int RUNS>
__global__ __launch_bounds__(THREADS) void batch_tables_kernel(TableParams p) {
    constexpr int kMost = THREADS * EACH, kWaves = THREADS / 64;
    // running totals of rows, needed pages and pages given back; and each request's cached length, -1 where no row of it has a slot
    __shared__ int row_end[kMost], need_end[kMost], back_end[kMost], length[kMost], pages[kMost];
    __shared__ int group_end[kMost / 64];  // row_end of every 64th
    __shared__ int wave_total[3][kWaves], served, lacking;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = p.B, M = p.M;
    const int row_cap = p.max_rows + 1;  // more rows than there is room for
    const auto held_by = [&](int r) { return min(max(p.held[r], 0), M); };

    int n[EACH], h[EACH], len[EACH], need[EACH];
    int rows = 0, back = 0, needs = 0, bad = 0;
    const int given = p.counts[0];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int r = tid * EACH + e;
        n[e] = r < B ? p.new_lens[r] : 0;
        h[e] = r < B ? held_by(r) : 0;
        len[e] = r < B ? p.kv_lens[r] : 0;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int64_t blocks = ((int64_t)len[e] + max(n[e], 0) + kPage - 1) / kPage;
        const bool never = n[e] >= 0 && (len[e] < 0 || blocks > M);
        bad |= never ? 1 << e : 0;
        need[e] = n[e] < 0 || never ? 0 : max(0, (int)blocks - h[e]);
        rows = min(rows + min(max(n[e], 0), row_cap), row_cap);
        back += n[e] < 0 ? h[e] : 0;
        needs += need[e];
    }
    if (tid == 0) served = lacking = 0;
    // totals in front of this thread's requests, and of all of them
    int all[3], mine[3] = {rows, back, needs};
    const auto totals = [&](int from, int to) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (k < from || k >= to) continue;
            const int cap = k == 0 ? row_cap : INT32_MAX, upto = wave_totals(mine[k], cap);
            if (lane == 63) wave_total[k][wave] = upto;
            mine[k] = __builtin_amdgcn_update_dpp(0, upto, 0x138, 0xf, 0xf, false);  // the lane before
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (k < from || k >= to) continue;
            const int cap = k == 0 ? row_cap : INT32_MAX;
            int before = 0, sum = 0;
            if constexpr (kWaves > 4) {  // (16 totals one after the other take 0.5 us, the running totals over lanes again 0.2)
                const int upto = wave_totals(lane < kWaves ? wave_total[k][lane] : 0, cap);
                sum = __builtin_amdgcn_readlane(upto, kWaves - 1);
                if (wave > 0) before = __builtin_amdgcn_readlane(upto, __builtin_amdgcn_readfirstlane(wave - 1));
            } else {
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    if (w == wave) before = sum;
                    sum = min(sum + wave_total[k][w], cap);
                }
            }
            mine[k] = min(before + mine[k], cap);
            all[k] = sum;
        }
    };
    totals(0, 3);
    if (all[0] > p.max_rows) {  // some requests' rows have no place: they need no pages
        needs = 0;
        rows = mine[0];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            rows = min(rows + min(max(n[e], 0), row_cap), row_cap);
            if (n[e] > 0 && rows > p.max_rows) {
                bad |= 1 << e;
                need[e] = 0;
            }
            needs += need[e];
        }
        mine[2] = needs;
        __syncthreads();
        totals(2, 3);
    }
    const int all_rows = all[0], all_back = all[1];
    const int count = min(max(given, 0), p.num_pages);
    const int top = min(count + all_back, p.num_pages);
    int last = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int r = tid * EACH + e;
        mine[0] = min(mine[0] + min(max(n[e], 0), row_cap), row_cap);
        mine[1] += n[e] < 0 ? h[e] : 0;
        mine[2] += need[e];
        if (need[e] > 0 && mine[2] > top) bad |= 1 << e;
        else if (need[e] > 0) last = mine[2];
        row_end[r] = mine[0];  // (behind the last request the totals stay)
        if (r % 64 == 63) group_end[r / 64] = mine[0];
        back_end[r] = mine[1];
        need_end[r] = mine[2];
        length[r] = n[e] < 0 || (bad >> e & 1) ? -1 : len[e];
        pages[r] = h[e];
    }
    if (all[2] > top && last > 0) atomicMax(&served, last);
    if (bad) atomicAdd(&lacking, __popc(bad));
    __syncthreads();
    const int granted = all[2] > top ? served : all[2];

    const auto begin = [&](const int* totals, int r) { return r > 0 ? totals[r - 1] : 0; };
    const auto on_stack = [&](int at) {  // entry `at` of the stack with the ended requests' pages on it
        if (at < count) return p.free_pages[at];
        const int i = at - count, r = first_above(back_end, B, i);
        return p.tables[(size_t)r * M + i - begin(back_end, r)];
    };
    const int first = blockIdx.x * THREADS + tid, threads = gridDim.x * THREADS, rows_here = min(all_rows, p.max_rows);
    for (int base = (first - lane) * RUNS; base < p.max_rows; base += threads * RUNS) {
        // The requests of the runs' first rows, by the whole wave: which 64 requests, then which of them.
        int lo[RUNS], hi[RUNS], x[RUNS], at[RUNS], slot[RUNS], span = 0;
#pragma unroll
        for (int j = 0; j <= RUNS; ++j) {
            const int row = max(min(base + 64 * j, rows_here - 1), 0);
            const int group = min(__popcll(__ballot(lane < kMost / 64 && group_end[lane % (kMost / 64)] <= row)), kMost / 64 - 1);
            const int r = min(64 * group + __popcll(__ballot(row_end[64 * group + lane] <= row)), kMost - 1);
            if (j < RUNS) lo[j] = r;
            if (j > 0) {
                hi[j - 1] = r;
                span = max(span, r - lo[j - 1]);
            }
        }
#pragma unroll
        for (int j = 0; j < RUNS; ++j) x[j] = base + 64 * j + lane;
        for (; span > 0; span >>= 1) {  // then each row's between them, the runs' round trips together
#pragma unroll
            for (int j = 0; j < RUNS; ++j) {
                const int mid = (lo[j] + hi[j]) >> 1;
                const bool above = row_end[mid] > x[j];
                hi[j] = above ? mid : hi[j];
                lo[j] = above ? lo[j] : min(mid + 1, hi[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < RUNS; ++j) {
            const int r = lo[j], cached = length[r], held = pages[r];
            const bool has = x[j] < rows_here && cached >= 0;
            at[j] = has ? cached + (x[j] - begin(row_end, r)) : -1;
            const int b = at[j] / kPage;
            int page = -1;
            if (has) page = b < held ? p.tables[(size_t)r * M + b] : on_stack(top - 1 - (begin(need_end, r) + b - held));
            slot[j] = (unsigned)page < (unsigned)p.num_pages ? page * kPage + at[j] % kPage : -1;
        }
#pragma unroll
        for (int j = 0; j < RUNS; ++j) {
            if (x[j] >= p.max_rows) break;
            p.positions[x[j]] = at[j];
            p.slots[x[j]] = slot[j];
        }
    }
    for (int i = first; i < all_back; i += threads) {
        const int r = first_above(back_end, B, i);
        if (count + i < p.num_pages) p.free_pages[count + i] = p.tables[(size_t)r * M + i - begin(back_end, r)];
    }
    for (int j = first; j < granted; j += threads) {
        const int r = first_above(need_end, B, j);
        p.tables[(size_t)r * M + pages[r] + j - begin(need_end, r)] = on_stack(top - 1 - j);
    }
    if (blockIdx.x != 0) return;
    for (int r = tid; r < B; r += THREADS) {
        const int n = p.new_lens[r];
        const bool has = length[r] >= 0;
        p.kv_lens_out[r] = has ? length[r] + n : n < 0 ? 0 : p.kv_lens[r];
        p.held_out[r] = n < 0 ? 0 : pages[r] + (has ? need_end[r] - begin(need_end, r) : 0);
        p.row_offsets[r + 1] = min(row_end[r], p.max_rows);
    }
    if (tid == 0) {
        p.row_offsets[0] = 0;
        p.counts_out[0] = top - granted;
        p.counts_out[1] = lacking;
    }
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
    // Workgroups read the inputs while others write the outputs and, in place, the tables and the stack: what is written has to be memory of its own.
    const size_t n = sizeof(int32_t) * (size_t)num_requests;
    const struct { const void* at; size_t bytes; } all[] = {{kv_lens, n}, {new_lens, n}, {held, n}, {counts, 4}, {block_tables, n * max_blocks}, {free_pages, 4 * (size_t)num_pages},
        {kv_lens_out, n}, {held_out, n}, {counts_out, 8}, {row_offsets, n + 4}, {positions, 4 * (size_t)max_rows}, {slots, 4 * (size_t)max_rows}};
    constexpr int kWritten = 4, kOut = 6, kAll = sizeof(all) / sizeof(all[0]);
    for (int o = kWritten; o < kAll; ++o)
        for (int i = 0; i < o; ++i) {
            const bool shared = overlap(all[o].at, all[o].bytes, all[i].at, all[i].bytes);
            CPMCU_CHECK_ARG(!shared || o < kOut || i >= kOut, "batch_tables: an output is the memory of an input");
            CPMCU_CHECK_ARG(!shared || o >= kOut, "batch_tables: the tables or the stack share memory with another input");
            CPMCU_CHECK_ARG(!shared, "batch_tables: two outputs share memory");
        }
    TableParams p{kv_lens, new_lens, held, counts, block_tables, free_pages, kv_lens_out, held_out, counts_out, row_offsets, positions, slots,
                  num_requests, max_blocks, num_pages, max_rows};
    const int threads = num_requests <= 256 ? 256 : 1024;
    const bool few = max_rows <= 256 * threads;
    auto kernel = num_requests <= 256    ? few ? batch_tables_kernel<256, 1, 1> : batch_tables_kernel<256, 1, 4>
                  : num_requests <= 1024 ? few ? batch_tables_kernel<1024, 1, 1> : batch_tables_kernel<1024, 1, 4>
                                         : few ? batch_tables_kernel<1024, 4, 1> : batch_tables_kernel<1024, 4, 4>;
    const int grid = std::min(std::max(ceil_div(max_rows, threads * (few ? 1 : 4)), 1), 512);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, resolve_stream(stream), p);
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
