// Penalties for repeated tokens, biases and masks of allowed tokens on rows of logits, and their arg-max.
//
// With c the times that token v stands in the row's text:
//   z' = z where c = 0, else (z > 0 ? z / repetition : z * repetition) - frequency c - presence;
//   z'' = z' + bias[v], -infinity where v is not allowed,
// in 32 bits, every operation rounded by itself (no fused products), the result rounded once to the element type; then the largest result's index.
//
// What bounds it: a row is read and written once; the counts are not read from a table of all tokens, which somebody would have to keep and which is
// larger than the row itself: a workgroup has a slice of the vocabulary for some rows and counts the text's tokens that lie in it, in LDS
// (whole numbers: their order does not matter).  So a text is read once for each slice, out of L2.
#include "batch_attention.h"

#include <algorithm>

#pragma clang fp contract(off)

namespace cpmcu {
namespace {

constexpr int kThreads = 512, kSlice = kThreads * 8;
constexpr int kAhead = 7;  // places that a row's slices may lie ahead of another one's, because rows begin anywhere on 2 bytes
constexpr int kMostBiases = 1024;

struct LogitsParams {
    const uint16_t* in;
    uint16_t* out;
    int64_t in_stride, out_stride, allowed_stride;
    int n, V, R, L, biases, mask_words, rows_each, slices;
    const float* penalties;  // [R][3]: repetition, presence, frequency
    const int32_t *tokens, *lens, *requests, *bias_ids, *draft_ids;
    const float* bias_values;
    const uint32_t* allowed;
    const uint64_t* tree_mask;
    uint64_t* best;  // [n][slices]
    int32_t* ids;
};

// Larger for larger values, and for equal ones for lower indexes; 0 below all of them: minus infinity and NaN are no candidates.
template <typename E>
__device__ inline uint64_t rank_of(uint16_t bits, int index) {
    const float v = Elem<E>::from_bits(bits);
    if (!(v > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);  // (both zeros are one value)
    const uint32_t key = u >> 31 ? ~u : u | 0x80000000u;
    return (uint64_t)key << 32 | (0xffffffffu - (uint32_t)index);
}

template <typename E>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitsParams p) {
    __shared__ int count[kSlice + kAhead];
    __shared__ float bias[kSlice + kAhead];
    __shared__ int hits, hit_at[kMostBiases];
    __shared__ uint64_t s_best[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slice = blockIdx.x % p.slices, row_begin = blockIdx.x / p.slices * p.rows_each, row_end = min(row_begin + p.rows_each, p.n);
    int request = -2;  // whose counts and biases are in LDS
    float repetition = 1.f, presence = 0.f, frequency = 0.f;
    // A row's pieces of 16 bytes lie where memory has them: the first one may begin in front of the row, by another number of places than the next row's.
    const int base = slice * kSlice - kAhead;  // what is counted is [base, base + kSlice + kAhead)
    const auto place_of = [&](int v) { return (unsigned)v < (unsigned)p.V && (unsigned)(v - base) < (unsigned)(kSlice + kAhead) ? v - base : -1; };
    for (int t = row_begin; t < row_end; ++t) {
        const uint16_t* const in = p.in + (int64_t)t * p.in_stride;
        uint16_t* const out = p.out + (int64_t)t * p.out_stride;
        const bool together = ((uintptr_t)in & 15) == ((uintptr_t)out & 15);
        const int e0 = slice * kSlice - (int)((uintptr_t)in / 2 & 7) + tid * 8, at = e0 - base;
        const bool whole = together && e0 >= 0 && e0 + 8 <= p.V;
        uint4 words = {0, 0, 0, 0};
        if (whole) words = *reinterpret_cast<const uint4*>(in + e0);
        int r = p.requests ? p.requests[t] : p.R == 1 ? 0 : t;
        if ((unsigned)r >= (unsigned)p.R) r = -1;  // (a row of nobody: only its mask counts)
        if (r != request) {
            request = r;
            __syncthreads();
            for (int i = tid; i < kSlice + kAhead; i += kThreads) {
                count[i] = 0;
                bias[i] = 0.f;
            }
            if (tid == 0) hits = 0;
            __syncthreads();
            repetition = 1.f;
            presence = frequency = 0.f;
            if (r >= 0 && p.penalties) {
                repetition = p.penalties[r * 3];
                presence = p.penalties[r * 3 + 1];
                frequency = p.penalties[r * 3 + 2];
                if (p.tokens) {
                    const int32_t* const text = p.tokens + (size_t)r * p.L;
                    const int len = min(max(p.lens[r], 0), p.L);
                    for (int i = tid; i < len; i += kThreads) {
                        const int v = place_of(text[i]);
                        if (v >= 0) atomicAdd(&count[v], 1);
                    }
                }
            }
            if (r >= 0 && p.bias_ids) {
                for (int i = tid; i < p.biases; i += kThreads) {
                    const int v = place_of(p.bias_ids[(size_t)r * p.biases + i]);
                    if (v >= 0) hit_at[atomicAdd(&hits, 1)] = v << 12 | i;
                }
                __syncthreads();
                // An index that stands several times: who has its first place adds them all up, in their order.
                for (int x = tid; x < hits; x += kThreads) {
                    const int me = hit_at[x], v = me >> 12;
                    bool mine = true;
                    for (int y = 0; y < hits; ++y) mine = mine && !(hit_at[y] >> 12 == v && hit_at[y] < me);
                    if (!mine) continue;
                    float sum = 0.f;
                    for (int last = me - 1;;) {
                        int next = INT32_MAX;
                        for (int y = 0; y < hits; ++y)
                            if (hit_at[y] >> 12 == v && hit_at[y] > last) next = min(next, hit_at[y]);
                        if (next == INT32_MAX) break;
                        sum += p.bias_values[(size_t)r * p.biases + (next & 0xfff)];
                        last = next;
                    }
                    bias[v] = sum;
                }
            }
            __syncthreads();
        }
        // the tokens on a tree node's way count for its row only
        int on_way = -1;
        if (p.draft_ids && tid < p.n && (p.tree_mask[(size_t)t * p.mask_words + (tid >> 6)] >> (tid & 63) & 1)) on_way = place_of(p.draft_ids[tid]);
        if (p.draft_ids) {
            if (on_way >= 0) atomicAdd(&count[on_way], 1);
            __syncthreads();
        }
        uint32_t bits = 0xffu;
        if (p.allowed) {
            const uint32_t* const mask = p.allowed + (int64_t)t * p.allowed_stride;
            const int last = (p.V - 1) >> 5, lo = min(max(e0 >> 5, 0), last), hi = min(max((e0 + 7) >> 5, 0), last);
            // bit j: place e0 + j
            bits = e0 < 0 ? mask[0] << -e0 : (uint32_t)(((uint64_t)(hi > lo ? mask[hi] : 0) << 32 | mask[lo]) >> (e0 & 31));
        }
        uint64_t mine = 0;
        uint16_t z16[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = e0 + j;
            uint16_t x = (uint16_t)((j & 1 ? (&words.x)[j >> 1] >> 16 : (&words.x)[j >> 1]) & 0xffffu);
            if (!whole) {
                if (e < 0 || e >= p.V) continue;
                x = in[e];
            }
            const int c = count[at + j];
            float z = Elem<E>::from_bits(x);
            if (c > 0) {
                const float again = z > 0.f ? z / repetition : z * repetition;
                z = again - frequency * (float)c - presence;
            }
            if (p.bias_ids) z += bias[at + j];
            if (!(bits >> j & 1)) z = -INFINITY;
            const uint16_t y = Elem<E>::to_bits(z);
            z16[j] = y;
            if (!whole) out[e] = y;
            const uint64_t rank = rank_of<E>(y, e);
            mine = rank > mine ? rank : mine;
        }
        if (whole) {
            uint4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) (&y.x)[j] = (uint32_t)z16[2 * j] | (uint32_t)z16[2 * j + 1] << 16;
            *reinterpret_cast<uint4*>(out + e0) = y;
        }
        if (p.best) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint64_t other = __shfl_xor(mine, d);
                mine = other > mine ? other : mine;
            }
            if (lane == 0) s_best[wave] = mine;
        }
        if (p.best || p.draft_ids) __syncthreads();
        if (on_way >= 0) atomicSub(&count[on_way], 1);
        if (p.best) {
            if (tid == 0) {
#pragma unroll
                for (int w = 0; w < kThreads / 64; ++w) mine = s_best[w] > mine ? s_best[w] : mine;
                p.best[(size_t)t * p.slices + slice] = mine;
            }
        }
        if (p.best || p.draft_ids) __syncthreads();
    }
}

// A wave a row.
__global__ __launch_bounds__(256) void adjust_logits_ids_kernel(const uint64_t* best, int n, int slices, int32_t* ids) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= n) return;
    uint64_t mine = 0;
    for (int i = lane; i < slices; i += 64) {
        const uint64_t other = best[(size_t)t * slices + i];
        mine = other > mine ? other : mine;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t other = __shfl_xor(mine, d);
        mine = other > mine ? other : mine;
    }
    if (lane == 0) ids[t] = mine ? (int32_t)(0xffffffffu - (uint32_t)mine) : -1;
}

// (a row that does not begin on 16 bytes reaches up to seven places further)
int slices_of(int V) { return ceil_div(V + 7, kSlice); }

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" size_t cpmcu_adjust_logits_workspace_bytes(int n, int V) {
    if (n < 0 || n >= 1 << 24 || V < 1 || V > 1 << 24) return 0;
    return sizeof(uint64_t) * (size_t)n * slices_of(V);
}

extern "C" int cpmcu_adjust_logits(const void* logits, int64_t logits_stride, int n, int V, const float* penalties, const int32_t* tokens, const int32_t* lens, int num_requests,
                                   int max_tokens, const int32_t* requests, const int32_t* bias_ids, const float* bias_values, int num_biases, const uint32_t* allowed,
                                   int64_t allowed_stride, const int32_t* draft_ids, const uint64_t* tree_mask, int mask_words, void* out, int64_t out_stride, int32_t* ids,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    CPMCU_CHECK_ARG(n >= 0 && n < 1 << 24, "adjust_logits: n=%d outside [0, 2^24)", n);
    CPMCU_CHECK_ARG(V >= 1 && V <= 1 << 24, "adjust_logits: V=%d outside [1, 2^24]", V);
    if (n == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(logits && out, "adjust_logits: null pointer argument");
    CPMCU_CHECK_ARG(n == 1 || (logits_stride >= V && out_stride >= V), "adjust_logits: rows closer than their %d values", V);
    CPMCU_CHECK_ARG(((uintptr_t)logits | (uintptr_t)out) % 2 == 0, "adjust_logits: rows have to lie on 2 bytes");
    const bool any = penalties || bias_ids;
    CPMCU_CHECK_ARG(!any || num_requests >= 1, "adjust_logits: %d requests", num_requests);
    CPMCU_CHECK_ARG(!any || requests || num_requests == 1 || num_requests == n, "adjust_logits: %d rows of %d requests need requests", n, num_requests);
    CPMCU_CHECK_ARG(!tokens || (penalties && lens && max_tokens >= 1), "adjust_logits: tokens go with penalties and lens, one place each at least");
    CPMCU_CHECK_ARG(!bias_ids || (bias_values && num_biases >= 1 && num_biases <= kMostBiases), "adjust_logits: %d biases outside [1, %d], or without values", num_biases, kMostBiases);
    CPMCU_CHECK_ARG(!allowed || allowed_stride == 0 || allowed_stride >= (V + 31) / 32, "adjust_logits: rows of allowed closer than their words");
    CPMCU_CHECK_ARG(!draft_ids || (tree_mask && penalties && num_requests == 1 && !requests), "adjust_logits: draft_ids go with tree_mask and the penalties of one request");
    CPMCU_CHECK_ARG(!draft_ids || (n <= kMaxTree && mask_words >= ceil_div(n, 64)), "adjust_logits: a tree of %d nodes, masks of %d words", n, mask_words);
    const int slices = slices_of(V);
    const size_t need = ids ? sizeof(uint64_t) * (size_t)n * slices : 0;
    CPMCU_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0), "adjust_logits: workspace of %zu bytes, %zu needed, on 8 bytes", workspace_bytes, need);
    const size_t in_bytes = 2 * ((size_t)(n - 1) * logits_stride + V), out_bytes = 2 * ((size_t)(n - 1) * out_stride + V), ints = 4;
    const bool in_place = logits == out && (n == 1 || logits_stride == out_stride);
    CPMCU_CHECK_ARG(in_place || !overlap(logits, in_bytes, out, out_bytes), "adjust_logits: the results lie in other logits");
    const struct { const void* at; size_t bytes; } read[] = {
        {penalties, 12 * (size_t)num_requests}, {tokens, ints * num_requests * max_tokens}, {lens, ints * num_requests}, {requests, ints * n}, {bias_ids, ints * num_requests * num_biases},
        {bias_values, ints * num_requests * num_biases}, {allowed, ints * ((size_t)(n - 1) * allowed_stride + (V + 31) / 32)}, {draft_ids, ints * n}, {tree_mask, 8 * (size_t)n * mask_words}};
    for (const auto& m : read) {
        if (!m.at) continue;
        CPMCU_CHECK_ARG(!overlap(m.at, m.bytes, out, out_bytes) && !overlap(m.at, m.bytes, ids, ids ? ints * n : 0), "adjust_logits: results in the memory of an argument");
    }
    CPMCU_CHECK_ARG(!overlap(ids, ids ? ints * n : 0, out, out_bytes) && !overlap(ids, ids ? ints * n : 0, logits, in_bytes), "adjust_logits: ids in the memory of logits");
    // Rows of one text share its counts: as many of them a workgroup as leave two workgroups a CU.
    const bool shared = any && num_requests == 1 && !requests;
    const int rows_each = shared ? std::max(1, std::min(n, (int)((int64_t)n * slices / 512))) : 1;
    const int64_t grid = (int64_t)ceil_div(n, rows_each) * slices;
    CPMCU_CHECK_ARG(grid <= INT32_MAX, "adjust_logits: %lld workgroups are beyond a launch", (long long)grid);
    LogitsParams p{(const uint16_t*)logits, (uint16_t*)out, logits_stride, out_stride, allowed_stride, n, V, any ? num_requests : 0, max_tokens, num_biases, mask_words, rows_each, slices,
                   penalties, tokens, lens, requests, bias_ids, draft_ids, bias_values, allowed, tree_mask, ids ? (uint64_t*)workspace : nullptr, ids};
    const hipStream_t st = resolve_stream(stream);
    hipLaunchKernelGGL(options().dtype == 1 ? adjust_logits_kernel<bf16> : adjust_logits_kernel<f16>, dim3((int)grid), dim3(kThreads), 0, st, p);
    CPMCU_LAUNCH_CHECK();
    if (ids) {
        hipLaunchKernelGGL(adjust_logits_ids_kernel, dim3(ceil_div(n, 4)), dim3(256), 0, st, p.best, n, slices, ids);
        CPMCU_LAUNCH_CHECK();
    }
    return CPMCU_OK;
}
