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

constexpr int kThreads = 256, kPieces = 2;   // pieces of 8 logits that a thread has of a row
constexpr int kSlice = kThreads * kPieces * 8;
constexpr int kAhead = 8;       // places that a row's slices may lie ahead of another one's, because rows begin anywhere on 2 bytes
constexpr int kCounted = kSlice + kAhead;
constexpr int kTextAtOnce = 8;  // tokens that a thread requests together
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

// 16-bit floats as whole numbers in the same order, two at a time: what is at most key_of(-infinity), or above key_of(infinity), is no candidate (NaN
// is behind either end); the zeros are neighbours.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
__device__ inline u16x2 keys_of(uint32_t w) {
    const i16x2 x = __builtin_bit_cast(i16x2, w);
    return __builtin_bit_cast(u16x2, x ^ ((x >> 15) | (i16x2)(int16_t)0x8000));
}
template <typename E>
struct Ends {
    static constexpr uint16_t kInfinity = Elem<E>::kDtype == 0 ? 0x7c00 : 0x7f80, kMinusInfinity = kInfinity | 0x8000;
    static constexpr uint32_t kHighest = kInfinity | 0x8000, kNone = (uint16_t)~kMinusInfinity;
};

template <typename E>
__global__ __launch_bounds__(kThreads, 6) void adjust_logits_kernel(LogitsParams p) {
    constexpr int kWords = kCounted / 32 + 2;
    __shared__ __attribute__((aligned(16))) int count[kCounted];
    __shared__ uint32_t counted[kWords], biased[kWords];  // places that have a count, or a bias: few pieces of a row have one
    __shared__ int hits, again, hit_at[kMostBiases];      // biases of the slice: place and number in the list
    __shared__ float hit_value[kMostBiases];
    __shared__ uint64_t s_best[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slice = blockIdx.x % p.slices, row_begin = blockIdx.x / p.slices * p.rows_each, row_end = min(row_begin + p.rows_each, p.n);
    int request = -2;  // whose counts and biases are in LDS
    float repetition = 1.f, presence = 0.f, frequency = 0.f;
    // A row's pieces of 16 bytes lie where memory has them: the first one may begin in front of the row, by another number of places than the next row's.
    const int base = slice * kSlice - kAhead;  // what is counted is [base, base + kCounted)
    const auto place_of = [&](int v) { return (unsigned)v < (unsigned)p.V && (unsigned)(v - base) < (unsigned)kCounted ? v - base : -1; };
    const auto count_one = [&](int at) {
        atomicAdd(&count[at], 1);
        atomicOr(&counted[at >> 5], 1u << (at & 31));
    };
    for (int t = row_begin; t < row_end; ++t) {
        const uint16_t* const in = p.in + (int64_t)t * p.in_stride;
        uint16_t* const out = p.out + (int64_t)t * p.out_stride;
        const bool together = ((uintptr_t)in & 15) == ((uintptr_t)out & 15);
        const int row_e0 = slice * kSlice - (int)((uintptr_t)in / 2 & 7);
        // What depends on nothing is requested first: the launch is round trips, one after the other unless they overlap.
        uint4 words[kPieces];
        uint32_t mask_lo[kPieces], mask_hi[kPieces];
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int e0 = row_e0 + (x * kThreads + tid) * 8;
            words[x] = uint4{0, 0, 0, 0};
            mask_lo[x] = mask_hi[x] = ~0u;
            if (together && e0 >= 0 && e0 + 8 <= p.V) words[x] = *reinterpret_cast<const uint4*>(in + e0);
            if (p.allowed) {
                const uint32_t* const mask = p.allowed + (int64_t)t * p.allowed_stride;
                const int last = (p.V - 1) >> 5;
                mask_lo[x] = mask[min(max(e0, 0) >> 5, last)];
                mask_hi[x] = mask[min(max(e0 + 7, 0) >> 5, last)];
            }
        }
        int on_way = -1;  // a token on a tree node's way
        if (p.draft_ids && tid < p.n && (p.tree_mask[(size_t)t * p.mask_words + (tid >> 6)] >> (tid & 63) & 1)) on_way = place_of(p.draft_ids[tid]);
        int r = p.requests ? p.requests[t] : p.R == 1 ? 0 : t;
        if ((unsigned)r >= (unsigned)p.R) r = -1;  // (a row of nobody: only its mask counts)
        if (r != request) {
            request = r;
            const bool texts = r >= 0 && p.tokens, biases = r >= 0 && p.bias_ids;
            const int32_t* const text = texts ? p.tokens + (size_t)r * p.L : nullptr;
            int token[kTextAtOnce], len = 0, bias_id[kMostBiases / kThreads];
            if (texts) {
                len = min(max(p.lens[r], 0), p.L);
#pragma unroll
                for (int u = 0; u < kTextAtOnce; ++u) token[u] = text[min(u * kThreads + tid, p.L - 1)];
            }
#pragma unroll
            for (int x = 0; x < kMostBiases / kThreads; ++x) bias_id[x] = biases && x * kThreads + tid < p.biases ? p.bias_ids[(size_t)r * p.biases + x * kThreads + tid] : -1;
            repetition = 1.f;
            presence = frequency = 0.f;
            if (r >= 0 && p.penalties) {
                repetition = p.penalties[r * 3];
                presence = p.penalties[r * 3 + 1];
                frequency = p.penalties[r * 3 + 2];
            }
            if (t > row_begin) __syncthreads();  // (the last row's have been read)
            if (texts || p.draft_ids)
                for (int i = tid; i < kCounted / 4; i += kThreads) reinterpret_cast<int4*>(count)[i] = int4{0, 0, 0, 0};
            if (tid < kWords) counted[tid] = biased[tid] = 0;
            if (tid == 0) hits = again = 0;
            __syncthreads();
            for (int done = 0; done < len; done += kThreads * kTextAtOnce) {
                if (done > 0) {
#pragma unroll
                    for (int u = 0; u < kTextAtOnce; ++u) token[u] = text[min(done + u * kThreads + tid, p.L - 1)];
                }
#pragma unroll
                for (int u = 0; u < kTextAtOnce; ++u) {
                    if (done + u * kThreads >= len) break;
                    const int v = done + u * kThreads + tid < len ? place_of(token[u]) : -1;
                    if (v >= 0) count_one(v);
                }
            }
            if (biases) {
#pragma unroll
                for (int x = 0; x < kMostBiases / kThreads; ++x) {
                    const int v = place_of(bias_id[x]), i = x * kThreads + tid;
                    if (v < 0) continue;
                    const int h = atomicAdd(&hits, 1);
                    hit_at[h] = v << 10 | i;
                    hit_value[h] = p.bias_values[(size_t)r * p.biases + i];
                    const uint32_t bit = 1u << (v & 31);
                    if (atomicOr(&biased[v >> 5], bit) & bit) again = 1;
                }
            }
            __syncthreads();
            if (again) {  // an index that stands several times: its first place gets all of them, added up in their order
                for (int h = tid; h < hits; h += kThreads) {
                    const int v = hit_at[h] >> 10;
                    bool first = true;
                    for (int x = 0; x < hits && first; ++x) first = !(hit_at[x] >> 10 == v && hit_at[x] < hit_at[h]);
                    if (!first) continue;
                    float sum = 0.f;
                    for (int last = hit_at[h] - 1;;) {
                        int next = INT32_MAX;
                        for (int x = 0; x < hits; ++x)
                            if (hit_at[x] >> 10 == v && hit_at[x] > last) next = min(next, hit_at[x]);
                        if (next == INT32_MAX) break;
                        sum += p.bias_values[(size_t)r * p.biases + (next & 1023)];
                        last = next;
                    }
                    hit_value[h] = sum;
                }
                __syncthreads();
            }
        }
        if (p.draft_ids) {  // (counted for this row only)
            if (on_way >= 0) count_one(on_way);
            __syncthreads();
        }
        uint64_t best = 0;
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int e0 = row_e0 + (x * kThreads + tid) * 8, at = e0 - base;
            const bool whole = together && e0 >= 0 && e0 + 8 <= p.V;
            // bit j: place e0 + j (a word holds 32 places from a multiple of 32 on)
            const uint32_t allowed = e0 < 0 ? mask_lo[x] << -e0 : (uint32_t)(((uint64_t)mask_hi[x] << 32 | mask_lo[x]) >> (e0 & 31));
            const auto bits_at = [&](const uint32_t* set) { return (uint32_t)(((uint64_t)set[(at >> 5) + 1] << 32 | set[at >> 5]) >> (at & 31)) & 0xffu; };
            const uint32_t has_count = bits_at(counted), has_bias = bits_at(biased);
            const auto adjusted = [&](uint16_t bits, int j) {
                float z = Elem<E>::from_bits(bits);
                if (has_count >> j & 1) {
                    const int c = count[at + j];
                    if (c > 0) {  // (the tokens of another row's way have left their bits)
                        const float less = z > 0.f ? z / repetition : z * repetition;
                        z = less - frequency * (float)c - presence;
                    }
                }
                if (has_bias >> j & 1) {
                    int found = INT32_MAX;
                    float value = 0.f;
                    for (int h = 0; h < hits; ++h)
                        if (hit_at[h] >> 10 == at + j && hit_at[h] < found) {
                            found = hit_at[h];
                            value = hit_value[h];
                        }
                    z += value;
                }
                return (allowed >> j & 1) ? Elem<E>::to_bits(z) : Ends<E>::kMinusInfinity;
            };
            uint32_t w[4] = {words[x].x, words[x].y, words[x].z, words[x].w};
            if (whole) {
                // What is masked first, two logits a word; what a text or a bias changes one by one.
                if ((allowed & 0xffu) != 0xffu) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t lo = allowed >> (2 * j) & 1 ? 0xffffu : 0u, hi = allowed >> (2 * j + 1) & 1 ? 0xffff0000u : 0u;
                        w[j] = (w[j] & (lo | hi)) | ((uint32_t)Ends<E>::kMinusInfinity * 0x10001u & ~(lo | hi));
                    }
                }
                for (uint32_t rest = (has_count | has_bias) & allowed; rest; rest &= rest - 1) {
                    const int j = __builtin_ctz(rest), shift = 16 * (j & 1);
                    uint32_t old = w[0];
#pragma unroll
                    for (int i = 1; i < 4; ++i) old = j >> 1 == i ? w[i] : old;
                    const uint32_t y = (old & ~(0xffffu << shift)) | (uint32_t)adjusted((uint16_t)(old >> shift), j) << shift;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = j >> 1 == i ? y : w[i];
                }
                *reinterpret_cast<uint4*>(out + e0) = uint4{w[0], w[1], w[2], w[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (uint32_t)Ends<E>::kMinusInfinity * 0x10001u;
                for (int j = max(-e0, 0); j < min(p.V - e0, 8); ++j) {
                    const uint16_t y = adjusted(in[e0 + j], j);
                    out[e0 + j] = y;
                    const uint32_t keep = j & 1 ? 0xffffu : 0xffff0000u, put = (uint32_t)y << (16 * (j & 1));
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = j >> 1 == i ? (w[i] & keep) | put : w[i];
                }
            }
            if (!p.best) continue;
            // the largest of a piece, of the wave's pieces, and the first place that has it
            u16x2 key[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) key[j] = keys_of(w[j]);
            const u16x2 two = __builtin_elementwise_max(__builtin_elementwise_max(key[0], key[1]), __builtin_elementwise_max(key[2], key[3]));
            uint32_t most = max((uint32_t)two.x, (uint32_t)two.y);
            if (most > Ends<E>::kHighest) {  // a NaN among them
                most = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (key[j].x > Ends<E>::kHighest) key[j].x = 0;
                    if (key[j].y > Ends<E>::kHighest) key[j].y = 0;
                    most = max(most, max((uint32_t)key[j].x, (uint32_t)key[j].y));
                }
            }
            if (most == 0x7fff) most = 0x8000;  // the zeros are one value
            uint32_t top = most;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
            if (top > Ends<E>::kNone && lane == __builtin_ctzll(__ballot(most == top))) {
                int j = 0;
#pragma unroll
                for (int i = 7; i >= 0; --i) {
                    const uint32_t k = i & 1 ? key[i >> 1].y : key[i >> 1].x;
                    if (k == top || (top == 0x8000 && k == 0x7fff)) j = i;
                }
                const uint64_t mine = (uint64_t)top << 32 | (0xffffffffu - (uint32_t)(e0 + j));
                best = mine > best ? mine : best;
            }
        }
        if (p.best) {
            // (one lane of the wave has it for each piece)
            const uint64_t some = __ballot(best != 0);
            uint64_t most = 0;
            for (uint64_t rest = some; rest; rest &= rest - 1) {
                const int from = __builtin_ctzll(rest);
                const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(best >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)best, from);
                most = other > most ? other : most;
            }
            if (lane == 0) s_best[wave] = most;
        }
        if (p.best || p.draft_ids) __syncthreads();
        if (on_way >= 0) atomicSub(&count[on_way], 1);
        if (p.best && tid == 0) {
            uint64_t most = s_best[0];
#pragma unroll
            for (int w = 1; w < kThreads / 64; ++w) most = s_best[w] > most ? s_best[w] : most;
            p.best[(size_t)t * p.slices + slice] = most;
        }
        if ((p.best || p.draft_ids) && t + 1 < row_end) __syncthreads();
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
    CPMCU_CHECK_ARG(max_tokens <= 1 << 30, "adjust_logits: max_tokens=%d beyond 2^30", max_tokens);
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
    // Rows of one text share its counts: as many of them a workgroup as leave four workgroups a CU.
    const bool shared = any && num_requests == 1 && !requests;
    const int rows_each = shared ? std::max(1, std::min(n, (int)((int64_t)n * slices / 1024))) : 1;
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
