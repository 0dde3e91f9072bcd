// Penalties for repeated tokens, biases and masks of allowed tokens on rows of logits, and their arg-max.
//
// With c the times that token v stands in the row's text:
//   z' = z where c = 0, else (z > 0 ? z / repetition : z * repetition) - frequency c - presence;
//   z'' = z' + bias[v], -infinity where v is not allowed,
// in 32 bits, every operation rounded by itself (no fused products), the result rounded once to the element type; then the largest result's index.
//
// What bounds it: a row is read and written once; the counts are not read from a table of all tokens, which somebody would have to keep and which is
// larger than the row itself: a workgroup has a slice of the vocabulary for some rows and counts the text's tokens that lie in it, in LDS
// (whole numbers: their order does not matter).  So a text is read once for each slice, out of L2.  512 rows of 73447 with texts of 1500, 40 biases
// and masks: 44 us, 3.4 TB/s of 150 MB (a plain copy of them takes 32); the instructions that count are what is left, so waves are many (32 a CU: with
// 20 they take 50) and registers and LDS few: the lists of biases have the room that the call's list needs.
#include "batch_attention.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(off)

namespace cpmcu {
namespace {

constexpr int kPieces = 2;      // pieces of 8 logits that a thread has of a row
constexpr int kAhead = 8;       // places that a row's slices may lie ahead of another one's, because rows begin anywhere on 2 bytes
// A slice reads the whole text, so longer texts take larger ones: 4096, 8192 and 16384 logits, two pieces a thread.  512 rows with texts of 300: 28, 29 and 32 us, of 4000 42, 38 and 41,
// of 16000 86, 68 and 61; one row with 100000 42, 27 and 25.  (What the call has room for decides, the lengths are the device's.)  Rows of one text: 8192, 60 tree nodes
// and 20000 tokens 17 us, with the others 21 and 19.
constexpr int kSmall = 256, kMiddle = 512, kLarge = 1024, kShortText = 4096, kMiddleText = 8192;
constexpr int slice_of(int threads) { return threads * kPieces * 8; }
constexpr int kTextAtOnce = 8;  // tokens that a thread requests together
constexpr int kMostBiases = 1024, kCountBits = 21, kMostTokens = 1 << 20;  // (a draft tree's 128 besides)

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

// The largest of a wave's values, within rows of 16 lanes and then from row to row, without LDS.
__device__ inline uint32_t wave_most(uint32_t v) {
    const auto with = [&](auto from) { v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(from)::value, 0xf, 0xf, false)); };
    with(std::integral_constant<int, 0x111>{});  // a lane takes its neighbour's, then that of two, four and eight lanes before it
    with(std::integral_constant<int, 0x112>{});
    with(std::integral_constant<int, 0x114>{});
    with(std::integral_constant<int, 0x118>{});
    with(std::integral_constant<int, 0x142>{});  // a row takes the last lane's of the row before it, the upper half that of lane 31
    with(std::integral_constant<int, 0x143>{});
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// SHARED: rows of one text, one after the other, a text's draft tree among them; else a row a workgroup.
template <typename E, bool SHARED, int THREADS>
__global__ __launch_bounds__(THREADS, SHARED ? 6 : 8) void adjust_logits_kernel(LogitsParams p) {
    constexpr int kThreads = THREADS, kSlice = slice_of(THREADS), kCounted = kSlice + kAhead, kWords = kCounted / 32 + 2, kBiases = kMostBiases / kThreads;
    extern __shared__ int bias_at[];  // the list of biases: each one's place in the slice, or -1; behind them their values
    float* const bias_value = reinterpret_cast<float*>(bias_at + p.biases);
    __shared__ __attribute__((aligned(16))) uint32_t count[kCounted];  // of a place: its count, and above it the number of its bias in the list, from 1 on
    __shared__ uint32_t counted[kWords], biased[kWords], twice[kWords];  // places that have either: few pieces of a row have one; with a bias; with several
    __shared__ int again;
    __shared__ uint64_t s_best[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slice = blockIdx.x % p.slices, row_begin = blockIdx.x / p.slices * (SHARED ? p.rows_each : 1), row_end = SHARED ? min(row_begin + p.rows_each, p.n) : row_begin + 1;
    // A row's pieces of 16 bytes lie where memory has them: the first one may begin in front of the row, by another number of places than the next row's.
    const int base = slice * kSlice - kAhead;  // what is counted is [base, base + kCounted)
    const int first_place = max(base, 0), places = min(base + kCounted, p.V) - first_place;
    const auto place_of = [&](int v) { return (unsigned)(v - first_place) < (unsigned)places ? v - base : -1; };
    const auto count_one = [&](int at) {
        atomicAdd(&count[at], 1u);
        atomicOr(&counted[at >> 5], 1u << (at & 31));
    };
    struct Row {
        uint4 words[kPieces];
        uint32_t mask_lo[kPieces], mask_hi[kPieces];
        int e0, on_way;  // where the slice begins; a token on a tree node's way
    };
    const auto request_row = [&](int t, Row& x) {
        const uint16_t* const in = p.in + (int64_t)t * p.in_stride;
        x.e0 = slice * kSlice - (int)((uintptr_t)in / 2 & 7);
        const uint32_t* const mask = p.allowed + (p.allowed ? (int64_t)t * p.allowed_stride : 0);
        const int last = (p.V - 1) >> 5;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e0 = x.e0 + (i * kThreads + tid) * 8;
            x.mask_lo[i] = x.mask_hi[i] = ~0u;
            if (p.allowed) {
                x.mask_lo[i] = mask[min(max(e0, 0) >> 5, last)];
                x.mask_hi[i] = mask[min(max(e0 + 7, 0) >> 5, last)];
            }
            if (e0 >= 0 && e0 + 8 <= p.V) {
                x.words[i] = *reinterpret_cast<const uint4*>(in + e0);
            } else {  // a row's first and last piece; -infinity where it has none
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (uint32_t)Ends<E>::kMinusInfinity * 0x10001u;
#pragma unroll 1
                for (int j = max(-e0, 0); j < min(p.V - e0, 8); ++j) {
                    const uint32_t keep = j & 1 ? 0xffffu : 0xffff0000u, put = (uint32_t)in[e0 + j] << (16 * (j & 1));
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = j >> 1 == k ? (w[k] & keep) | put : w[k];
                }
                x.words[i] = uint4{w[0], w[1], w[2], w[3]};
            }
        }
        x.on_way = -1;
        if (SHARED && p.draft_ids && tid < p.n && (p.tree_mask[(size_t)t * p.mask_words + (tid >> 6)] >> (tid & 63) & 1)) x.on_way = place_of(p.draft_ids[tid]);
    };
    // What depends on nothing is requested first: the launch is round trips, one after the other unless they overlap.
    Row x;
    request_row(row_begin, x);
    int r = SHARED ? 0 : p.requests ? p.requests[row_begin] : p.R == 1 ? 0 : row_begin;
    if ((unsigned)r >= (unsigned)p.R) r = -1;  // (a row of nobody: only its mask counts)
    const bool texts = r >= 0 && p.tokens, biases = r >= 0 && p.bias_ids, draft = SHARED && p.draft_ids;
    float repetition = 1.f, presence = 0.f, frequency = 0.f;
    if (texts || draft || biases) {
        const int32_t* const text = texts ? p.tokens + (size_t)r * p.L : nullptr;
        int token[kTextAtOnce], len = 0, bias_id[kBiases];
        if (texts) {
            len = min(max(p.lens[r], 0), p.L);
#pragma unroll
            for (int u = 0; u < kTextAtOnce; ++u) token[u] = text[min(u * kThreads + tid, p.L - 1)];
        }
#pragma unroll
        for (int i = 0; i < kBiases; ++i) {
            if (!biases || i * kThreads >= p.biases) break;
            bias_id[i] = i * kThreads + tid < p.biases ? p.bias_ids[(size_t)r * p.biases + i * kThreads + tid] : -1;
        }
        if (p.penalties) {
            repetition = p.penalties[r * 3];
            presence = p.penalties[r * 3 + 1];
            frequency = p.penalties[r * 3 + 2];
        }
#pragma unroll
        for (int i = 0; i < kCounted / 4; i += kThreads)
            if (i + kThreads <= kCounted / 4 || i + tid < kCounted / 4) reinterpret_cast<int4*>(count)[i + tid] = int4{0, 0, 0, 0};
        if (tid < kWords) counted[tid] = biased[tid] = twice[tid] = 0;
        if (tid == 0) again = 0;
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
            for (int i = 0; i < kBiases; ++i) {
                if (i * kThreads >= p.biases) break;
                const int v = place_of(bias_id[i]), number = i * kThreads + tid;
                if (number < p.biases) bias_at[number] = v;
                if (v < 0) continue;
                bias_value[number] = p.bias_values[(size_t)r * p.biases + number];
                const uint32_t bit = 1u << (v & 31);
                if (atomicOr(&biased[v >> 5], bit) & bit) {
                    again = 1;
                    atomicOr(&twice[v >> 5], bit);
                } else {
                    atomicAdd(&count[v], (uint32_t)(number + 1) << kCountBits);
                    atomicOr(&counted[v >> 5], bit);
                }
            }
        }
        __syncthreads();
        if (biases && again) {  // an index that stands several times: the one that its place names gets all of them, added up in the list's order
#pragma unroll 1
            for (int number = tid; number < p.biases; number += kThreads) {
                const int v = bias_at[number];
                if (v < 0 || !(twice[v >> 5] >> (v & 31) & 1) || (int)(count[v] >> kCountBits) != number + 1) continue;
                float sum = 0.f;
#pragma unroll 8
                for (int i = 0; i < p.biases; ++i) {
                    const float next = sum + bias_value[i];  // (another place's may be anything)
                    sum = bias_at[i] == v ? next : sum;
                }
                bias_value[number] = sum;
            }
            __syncthreads();
        }
    }
    for (int t = row_begin;;) {
        Row next;
        const bool more = SHARED && t + 1 < row_end;
        if (more) request_row(t + 1, next);
        if (draft) {  // (counted for this row only)
            if (x.on_way >= 0) count_one(x.on_way);
            __syncthreads();
        }
        uint16_t* const out = p.out + (int64_t)t * p.out_stride;
        const bool whole_words = ((uintptr_t)(out + x.e0) & 15) == 0;
        uint32_t largest[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e0 = x.e0 + (i * kThreads + tid) * 8, at = e0 - base;
            uint32_t w[4] = {x.words[i].x, x.words[i].y, x.words[i].z, x.words[i].w};
            // bit j: place e0 + j (a word holds 32 places from a multiple of 32 on)
            uint32_t allowed = 0xff;
            if (p.allowed) {
                allowed = __builtin_amdgcn_alignbit(x.mask_hi[i], x.mask_lo[i], e0);
                if (e0 < 0) allowed = x.mask_lo[i] << -e0;
                if ((allowed & 0xffu) != 0xffu) {  // two logits a word
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t lo = (uint32_t)((int)(allowed << (31 - 2 * j)) >> 31), hi = (uint32_t)((int)(allowed << (30 - 2 * j)) >> 31);
                        const uint32_t keep = (lo & 0xffffu) | (hi & 0xffff0000u);
                        w[j] = (w[j] & keep) | ((uint32_t)Ends<E>::kMinusInfinity * 0x10001u & ~keep);
                    }
                }
            }
            if (texts || draft || biases) {
                const uint32_t has = __builtin_amdgcn_alignbit(counted[(at >> 5) + 1], counted[at >> 5], at) & 0xffu;
                for (uint32_t rest = has & allowed; rest; rest &= rest - 1) {
                    const int j = __builtin_ctz(rest), shift = 16 * (j & 1);
                    uint32_t old = w[0];
#pragma unroll
                    for (int k = 1; k < 4; ++k) old = j >> 1 == k ? w[k] : old;
                    float z = Elem<E>::from_bits((uint16_t)(old >> shift));
                    const uint32_t both = count[at + j], c = both & ((1u << kCountBits) - 1), h = both >> kCountBits;
                    if (c > 0) {  // (the tokens of another row's way have left their bits)
                        const float less = z > 0.f ? z / repetition : z * repetition;
                        z = less - frequency * (float)c - presence;
                    }
                    if (h > 0) z += bias_value[h - 1];
                    const uint32_t y = (old & ~(0xffffu << shift)) | (uint32_t)Elem<E>::to_bits(z) << shift;
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = j >> 1 == k ? y : w[k];
                }
            }
            if (whole_words && e0 >= 0 && e0 + 8 <= p.V) {
                *reinterpret_cast<uint4*>(out + e0) = uint4{w[0], w[1], w[2], w[3]};
            } else {
#pragma unroll 1
                for (int j = max(-e0, 0); j < min(p.V - e0, 8); ++j) out[e0 + j] = (uint16_t)((j & 4 ? j & 2 ? w[3] : w[2] : j & 2 ? w[1] : w[0]) >> (16 * (j & 1)));
            }
            largest[i] = 0;
            if (!p.best) continue;
            // The piece's largest and, behind it, how far in front of the piece's end it lies: of equals the first is the largest.
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t key = __builtin_bit_cast(uint32_t, keys_of(w[j]));
                most = max(most, max(key << 16 | (7 - 2 * j), (key & 0xffff0000u) | (6 - 2 * j)));
            }
            if (most >> 16 > Ends<E>::kHighest || (most >> 16) - 0x7fff <= 1) {  // a NaN among them; or a zero: the two zeros are one value
                most = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const u16x2 two = keys_of(w[j >> 1]);
                    const uint32_t key = j & 1 ? two.y : two.x;
                    if (key <= Ends<E>::kHighest) most = max(most, (key == 0x7fff ? 0x8000 : key) << 16 | (7 - j));
                }
            }
            largest[i] = most;
        }
        if (p.best) {
            // the wave's largest and the first place that has it
            uint32_t all = largest[0];
#pragma unroll
            for (int i = 1; i < kPieces; ++i) all = max(all, largest[i]);
            const uint32_t top = wave_most(all >> 16);
            uint64_t most = 0;
            if (top > Ends<E>::kNone) {
#pragma unroll
                for (int i = kPieces - 1; i >= 0; --i) {
                    const uint64_t have = __ballot(largest[i] >> 16 == top);
                    if (!have) continue;
                    const int first = __builtin_ctzll(have);
                    const int place = x.e0 + (i * kThreads + wave * 64 + first) * 8 + 7 - (__builtin_amdgcn_readlane((int)largest[i], first) & 7);
                    most = (uint64_t)top << 32 | (0xffffffffu - (uint32_t)place);
                }
            }
            if (lane == 0) s_best[wave] = most;
        }
        if (p.best || (draft && more)) __syncthreads();
        if (draft && more && x.on_way >= 0) atomicSub(&count[x.on_way], 1u);
        if (p.best && tid == 0) {
            uint64_t most = s_best[0];
#pragma unroll
            for (int w = 1; w < kThreads / 64; ++w) most = s_best[w] > most ? s_best[w] : most;
            p.best[(size_t)t * p.slices + slice] = most;
        }
        if (!more) break;
        if (p.best || draft) __syncthreads();
        ++t;
        x = next;
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
int slices_of(int V, int threads) { return ceil_div(V + 7, slice_of(threads)); }

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" size_t cpmcu_adjust_logits_workspace_bytes(int n, int V) {
    if (n < 0 || n >= 1 << 24 || V < 1 || V > 1 << 24) return 0;
    return sizeof(uint64_t) * (size_t)n * slices_of(V, kSmall);
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
    CPMCU_CHECK_ARG(!any || (num_requests >= 1 && num_requests < 1 << 24), "adjust_logits: %d requests outside [1, 2^24)", num_requests);
    CPMCU_CHECK_ARG(!any || requests || num_requests == 1 || num_requests == n, "adjust_logits: %d rows of %d requests need requests", n, num_requests);
    CPMCU_CHECK_ARG(max_tokens <= kMostTokens, "adjust_logits: max_tokens=%d beyond 2^20", max_tokens);
    CPMCU_CHECK_ARG(!tokens || (penalties && lens && max_tokens >= 1), "adjust_logits: tokens go with penalties and lens, one place each at least");
    CPMCU_CHECK_ARG(!bias_ids || (bias_values && num_biases >= 1 && num_biases <= kMostBiases), "adjust_logits: %d biases outside [1, %d], or without values", num_biases, kMostBiases);
    CPMCU_CHECK_ARG(!allowed || allowed_stride == 0 || allowed_stride >= (V + 31) / 32, "adjust_logits: rows of allowed closer than their words");
    CPMCU_CHECK_ARG(!draft_ids || (tree_mask && penalties && num_requests == 1 && !requests), "adjust_logits: draft_ids go with tree_mask and the penalties of one request");
    CPMCU_CHECK_ARG(!draft_ids || (n <= kMaxTree && mask_words >= ceil_div(n, 64)), "adjust_logits: a tree of %d nodes, masks of %d words", n, mask_words);
    // Rows of one text share its counts: as many of them a workgroup as leave four workgroups a CU.
    const bool one_text = any && num_requests == 1 && !requests;
    const int rows_each = one_text ? std::max(1, std::min(n, (int)((int64_t)n * slices_of(V, kMiddle) / 1024))) : 1;
    const bool shared = rows_each > 1 || draft_ids;
    const int threads = shared ? kMiddle : !tokens || max_tokens <= kShortText ? kSmall : max_tokens <= kMiddleText ? kMiddle : kLarge, slices = slices_of(V, threads);
    const size_t need = ids ? sizeof(uint64_t) * (size_t)n * slices_of(V, kSmall) : 0;
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
    const int64_t grid = (int64_t)ceil_div(n, rows_each) * slices;
    CPMCU_CHECK_ARG(grid * threads <= UINT32_MAX, "adjust_logits: %lld workgroups of %d threads are beyond a launch", (long long)grid, threads);
    LogitsParams p{(const uint16_t*)logits, (uint16_t*)out, logits_stride, out_stride, allowed_stride, n, V, any ? num_requests : 0, max_tokens, bias_ids ? num_biases : 0, mask_words, rows_each, slices,
                   penalties, tokens, lens, requests, bias_ids, draft_ids, bias_values, allowed, tree_mask, ids ? (uint64_t*)workspace : nullptr, ids};
    const hipStream_t st = resolve_stream(stream);
    const bool bf = options().dtype == 1;
    void (*kernel)(LogitsParams) = bf ? adjust_logits_kernel<bf16, false, kSmall> : adjust_logits_kernel<f16, false, kSmall>;
    if (threads == kMiddle) kernel = bf ? adjust_logits_kernel<bf16, false, kMiddle> : adjust_logits_kernel<f16, false, kMiddle>;
    if (threads == kLarge) kernel = bf ? adjust_logits_kernel<bf16, false, kLarge> : adjust_logits_kernel<f16, false, kLarge>;
    if (shared) kernel = bf ? adjust_logits_kernel<bf16, true, kMiddle> : adjust_logits_kernel<f16, true, kMiddle>;
    hipLaunchKernelGGL(kernel, dim3((int)grid), dim3(threads), 8 * p.biases, st, p);
    CPMCU_LAUNCH_CHECK();
    if (ids) {
        hipLaunchKernelGGL(adjust_logits_ids_kernel, dim3(ceil_div(n, 4)), dim3(256), 0, st, p.best, n, slices, ids);
        CPMCU_LAUNCH_CHECK();
    }
    return CPMCU_OK;
}
