// Rotary positions of query and key rows, and rows appended to the paged cache through a slot map.
//
// Row t at position p turns the pairs (x_i, y_i) of each head's first 2 * half values by the angle p * inv_freq[i]:
//   x' = m (x cos - y sin),  y' = m (x sin + y cos),  the pair being (i, i + half) or, interleaved, (2i, 2i + 1);
// the rest of the head is copied.  The angle is formed in 64 bits and reduced to a turn there -- in 32 bits the product alone is off by
// 0.004 at position 100 000 --, its sine and cosine are 32 bits; each result is rounded once.
#include "common.h"
#include "internal.h"
#include "kv_append.h"

#include <algorithm>

namespace cpmcu {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;    // heads of up to 256 values
constexpr int kMaxHeads = 1024;
constexpr int kRows = 4;         // rows of a workgroup: their angles are formed once for all heads
constexpr int kBatch = 4;        // items of a thread in flight

struct Turns {
    const int32_t* positions;
    const float* inv_freq;
    int half;
    float magnitude, sine;  // sine: the magnitude with the sign of the direction
};
struct HeadRows {
    const void* in;
    void* out;
    long in_stride, out_stride;  // values from row to row; a row's heads follow each other
    int heads;
};

__device__ inline float2 turn_of(const Turns& t, int position, int i) {
    constexpr double kTurnsPerRadian = 0.15915494309189533577;
    double turns = (double)position * (double)t.inv_freq[i] * kTurnsPerRadian;
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    return make_float2(c * t.magnitude, s * t.sine);
}

// An item of a head is eight pairs in two 16-byte pieces, behind the rotated values sixteen values (WIDE); or one pair, two values.
template <typename E, bool IL>
struct WideItem {
    typedef typename Elem<E>::x8 X8;
    static constexpr int kPairs = 8;
    X8 a, b;
    __device__ inline void load(const E* head, int i, int half) {
        a = *reinterpret_cast<const X8*>(head + first(i, half));
        b = *reinterpret_cast<const X8*>(head + second(i, half));
    }
    __device__ inline void store(E* head, int i, int half) const {
        *reinterpret_cast<X8*>(head + first(i, half)) = a;
        *reinterpret_cast<X8*>(head + second(i, half)) = b;
    }
    __device__ static inline int first(int i, int half) { return !IL && 8 * i < half ? 8 * i : 16 * i; }
    __device__ static inline int second(int i, int half) { return !IL && 8 * i < half ? half + 8 * i : 16 * i + 8; }
    __device__ inline void turn(const float2* cs) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (IL) {
                X8& x = j < 4 ? a : b;
                E u = x[2 * (j & 3)], v = x[2 * (j & 3) + 1];
                rotate_pair(u, v, cs[j]);
                x[2 * (j & 3)] = u;
                x[2 * (j & 3) + 1] = v;
            } else {
                E u = a[j], v = b[j];
                rotate_pair(u, v, cs[j]);
                a[j] = u;
                b[j] = v;
            }
        }
    }
};
template <typename E, bool IL>
struct NarrowItem {
    static constexpr int kPairs = 1;
    E a, b;
    __device__ inline void load(const E* head, int i, int half) { a = head[first(i, half)], b = head[second(i, half)]; }
    __device__ inline void store(E* head, int i, int half) const { head[first(i, half)] = a, head[second(i, half)] = b; }
    __device__ static inline int first(int i, int half) { return !IL && i < half ? i : 2 * i; }
    __device__ static inline int second(int i, int half) { return !IL && i < half ? half + i : 2 * i + 1; }
    __device__ inline void turn(const float2* cs) { rotate_pair(a, b, cs[0]); }
};

// Rows [r0, r0 + kRows) of q and k, this workgroup's part of their items.  present(r): whether row r has a position and a place.
template <typename E, typename Item, typename Present>
__device__ inline void rope_run(const Turns& t, const HeadRows& q, const HeadRows& k, int n, int head_dim, int r0, int part, int parts, float2* cs, int* there,
                                Present&& present) {
    const int tid = threadIdx.x, half = t.half;
    const int items = head_dim / (2 * Item::kPairs), per_row = (q.heads + k.heads) * items;
    const int rows = min(kRows, n - r0), total = rows * per_row;
    const int start = part * kThreads * kBatch;
    for (int base = start; base < total; base += parts * kThreads * kBatch) {
        Item x[kBatch];
        int row[kBatch], item[kBatch];
        E* to[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = base + u * kThreads + tid;
            row[u] = -1;
            if (i >= total) continue;
            row[u] = i / per_row;
            const int in_row = i - row[u] * per_row;
            int head = in_row / items;
            item[u] = in_row - head * items;
            const bool is_q = head < q.heads;
            if (!is_q) head -= q.heads;
            const E* from = (const E*)(is_q ? q.in : k.in) + (r0 + row[u]) * (is_q ? q.in_stride : k.in_stride) + (long)head * head_dim;
            to[u] = (E*)(is_q ? q.out : k.out) + (r0 + row[u]) * (is_q ? q.out_stride : k.out_stride) + (long)head * head_dim;
            x[u].load(from, item[u], half);
        }
        if (base == start) {
            for (int i = tid; i < rows * half; i += kThreads) cs[i] = turn_of(t, t.positions[r0 + i / half], i % half);
            if (tid < rows) there[tid] = present(r0 + tid);
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (row[u] < 0 || !there[row[u]]) continue;
            if (item[u] * Item::kPairs < half) x[u].turn(cs + row[u] * half + item[u] * Item::kPairs);
            x[u].store(to[u], item[u], half);
        }
    }
}

struct RopeParams {
    Turns t;
    HeadRows q, k;
    int n, head_dim, parts;
};

template <typename E, template <typename, bool> class Item, bool IL>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeParams p) {
    __shared__ float2 cs[kRows * kMaxHalf];
    __shared__ int there[kRows];
    rope_run<E, Item<E, IL>>(p.t, p.q, p.k, p.n, p.head_dim, blockIdx.x * kRows, blockIdx.y, p.parts, cs, there, [&](int r) { return p.t.positions[r] >= 0; });
}

// How many workgroups share kRows rows: enough to give every thread one batch while the launch is small.
int row_parts(int n, int heads, int items) {
    const int most = ceil_div(std::min(n, kRows) * heads * items, kThreads * kBatch);
    return std::min(most, std::max(1, 1024 / ceil_div(n, kRows)));
}

bool on_16_bytes(const HeadRows& x) {
    return x.heads == 0 || (((uintptr_t)x.in | (uintptr_t)x.out) % 16 == 0 && x.in_stride % 8 == 0 && x.out_stride % 8 == 0);
}

int check_rows(const char* op, const char* name, const HeadRows& x, int n, int head_dim) {
    CPMCU_CHECK_ARG(x.heads >= 0 && x.heads <= kMaxHeads, "%s: %d heads of %s outside [0, %d]", op, x.heads, name, kMaxHeads);
    if (x.heads == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(x.in && x.out, "%s: null pointer argument", op);
    const long width = (long)x.heads * head_dim;
    CPMCU_CHECK_ARG(x.in_stride >= width && x.out_stride >= width, "%s: rows of %s closer than their %ld values", op, name, width);
    if (x.in == x.out && x.in_stride == x.out_stride) return CPMCU_OK;
    const char *a = (const char*)x.in, *b = (const char*)x.out;
    CPMCU_CHECK_ARG(a + 2 * ((n - 1) * x.in_stride + width) <= b || b + 2 * ((n - 1) * x.out_stride + width) <= a,
                    "%s: the results of %s are neither in place nor in memory apart", op, name);
    return CPMCU_OK;
}

int check_turns(const char* op, const int32_t* positions, const float* inv_freq, int rotary_dim, int head_dim, float magnitude) {
    CPMCU_CHECK_ARG(positions && inv_freq, "%s: null pointer argument", op);
    CPMCU_CHECK_ARG(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, "%s: rotary_dim=%d is not an even number up to the head's %d values", op, rotary_dim, head_dim);
    CPMCU_CHECK_ARG(magnitude - magnitude == 0.f, "%s: magnitude is not finite", op);
    return CPMCU_OK;
}

// ---- append ----

constexpr int kSpan = 2 * kAppendRows;  // the row before a workgroup's sixteen, they, and the fifteen that may complete a group of slots

struct SlotParams {
    RopeParams rope;       // q alone; rope.t.positions null: rows that come rotated
    f16 *k_pool, *v_pool;
    const int32_t* slots;
    const void *k, *v;
    long k_stride, v_stride;
    int Hkv, heads_per_wg, kv_blocks, num_slots;
};

// Sixteen rows of heads_per_wg KV heads.  K rows go on as 16-byte pieces.  V is transposed through LDS: what a page holds of a dim is
// in aligned groups of 16 slots (two 16-byte pieces), so whoever has the first row of a run of consecutive slots inside such a group
// writes all of the group -- up to fifteen rows beyond its own sixteen -- and pieces are whole wherever the rows of a request follow
// each other, however the sixteen lie to the groups.
template <typename E, bool IL>
__device__ inline void append_run(const SlotParams& p, int block, float2* cs, int* slot, uint16_t* stage) {
    typedef WideItem<E, IL> Item;
    const int tid = threadIdx.x, n = p.rope.n, half = p.rope.t.half;
    const int groups_of_heads = p.Hkv / p.heads_per_wg;
    const int r0 = block / groups_of_heads * kAppendRows, g0 = block % groups_of_heads * p.heads_per_wg;
    const bool rope = p.rope.t.positions != nullptr;
    if (tid < kSpan) {
        const int r = r0 - 1 + tid;
        int s = -1;
        if (r >= 0 && r < n) {
            s = p.slots[r];
            if (s < 0 || s >= p.num_slots || (rope && p.rope.t.positions[r] < 0)) s = -1;
        }
        slot[tid] = s;
    }
    if (rope)
        for (int i = tid; i < min(kAppendRows, n - r0) * half; i += kThreads) cs[i] = turn_of(p.rope.t, p.rope.t.positions[r0 + i / half], i % half);
    __syncthreads();
    const int lane = tid & 63, at = lane & (kSpan - 1);
    // bit i: row r0 - 1 + i has a place; it continues the group of the row before it
    const int mine = slot[at];
    const uint32_t present = (uint32_t)__ballot(mine >= 0);
    const uint32_t joined = (uint32_t)__ballot(mine >= 0 && at > 0 && (mine & 15) != 0 && slot[max(at, 1) - 1] == mine - 1);
    const uint32_t leaders = present & ~joined & 0x1FFFEu;
    if ((present & 0x1FFFEu) == 0) return;
    const auto run_of = [&](int i) { return 1 + __builtin_ctz(~((uint64_t)joined >> (i + 1))); };  // rows of the group that row i leads
    const int last_leader = leaders ? 31 - __builtin_clz(leaders) : 0;
    const int staged = leaders ? max(last_leader + run_of(last_leader) - 1, kAppendRows) : kAppendRows;  // rows r0 .. r0 + staged - 1
    for (int g = g0; g < g0 + p.heads_per_wg; ++g) {
        const int row = tid >> 4, ch = tid & 15;
        for (int r = row; r < staged; r += kAppendRows) {
            if (slot[1 + r] < 0) continue;
            const uint4 vx = *reinterpret_cast<const uint4*>((const uint16_t*)p.v + (r0 + r) * p.v_stride + (long)g * kHeadDim + ch * 8);
            uint2* to = reinterpret_cast<uint2*>(stage + r * kAppendStride + ch * 8);
            to[0] = make_uint2(vx.x, vx.y);
            to[1] = make_uint2(vx.z, vx.w);
        }
        if (tid < kAppendRows * 8) {
            const int r = tid >> 3, i = tid & 7, s = slot[1 + r];
            if (s >= 0) {
                Item x;
                x.load((const E*)p.k + (r0 + r) * p.k_stride + (long)g * kHeadDim, i, half);
                if (rope && 8 * i < half) x.turn(cs + r * half + 8 * i);
                x.store((E*)p.k_pool + (((size_t)(s / kPage) * p.Hkv + g) * kPage + s % kPage) * kHeadDim, i, half);
            }
        }
        __syncthreads();
        const int d = tid >> 1, piece = tid & 1;
        for (uint32_t rest = leaders; rest; rest &= rest - 1) {
            const int i = __builtin_ctz(rest), s = slot[i], len = run_of(i);
            uint16_t* dst = reinterpret_cast<uint16_t*>(p.v_pool) + (((size_t)(s / kPage) * p.Hkv + g) * kHeadDim + d) * kPage + (s % kPage & ~15) + piece * 8;
            uint32_t v[8], in = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = piece * 4 + (j & 3) + (j >> 2) * 8 - (s & 15);  // the token of slot j, counted from the group's leader
                v[j] = stage[(i - 1 + min(max(r, 0), len - 1)) * kAppendStride + d];
                in |= r >= 0 && r < len ? 1u << j : 0u;
            }
            if (in == 0xFFu) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if ((in >> j) & 1u) dst[j] = (uint16_t)v[j];
            }
        }
        __syncthreads();
    }
}

template <typename E, bool IL>
__global__ __launch_bounds__(kThreads) void kv_append_slots_kernel(SlotParams p) {
    __shared__ float2 cs[kAppendRows * kHeadDim / 2];
    __shared__ int slot[kSpan];
    __shared__ __attribute__((aligned(8))) uint16_t stage[kSpan * kAppendStride];
    if ((int)blockIdx.x < p.kv_blocks) {
        append_run<E, IL>(p, blockIdx.x, cs, slot, stage);
        return;
    }
    const int b = blockIdx.x - p.kv_blocks;
    rope_run<E, WideItem<E, IL>>(p.rope.t, p.rope.q, p.rope.k, p.rope.n, kHeadDim, b / p.rope.parts * kRows, b % p.rope.parts, p.rope.parts, cs, slot,
                                 [&](int r) { return p.rope.t.positions[r] >= 0 && p.slots[r] >= 0 && p.slots[r] < p.num_slots; });
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" int cpmcu_rope_rows(const int32_t* positions, const float* inv_freq, int rotary_dim, int interleaved, float magnitude, int transposed,
                               const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int Hq, const void* k, int64_t k_stride, void* k_out,
                               int64_t k_out_stride, int Hkv, int head_dim, int n, void* stream) {
    CPMCU_CHECK_ARG(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 2 * kMaxHalf, "rope_rows: head_dim=%d is not an even number up to %d", head_dim, 2 * kMaxHalf);
    CPMCU_CHECK_ARG(n >= 0, "rope_rows: n=%d", n);
    if (int rc = check_turns("rope_rows", positions, inv_freq, rotary_dim, head_dim, magnitude)) return rc;
    RopeParams p{{positions, inv_freq, rotary_dim / 2, magnitude, transposed ? -magnitude : magnitude}, {q, q_out, q_stride, q_out_stride, Hq}, {k, k_out, k_stride, k_out_stride, Hkv}, n, head_dim, 1};
    if (int rc = check_rows("rope_rows", "q", p.q, std::max(n, 1), head_dim)) return rc;
    if (int rc = check_rows("rope_rows", "k", p.k, std::max(n, 1), head_dim)) return rc;
    if (n == 0 || Hq + Hkv == 0) return CPMCU_OK;
    const bool wide = rotary_dim % 16 == 0 && head_dim % 16 == 0 && on_16_bytes(p.q) && on_16_bytes(p.k);
    p.parts = row_parts(n, Hq + Hkv, head_dim / (wide ? 16 : 2));
    const dim3 grid(ceil_div(n, kRows), p.parts);
    hipStream_t st = resolve_stream(stream);
#define CPMCU_ROPE(E)                                                                                                                      \
    (wide ? interleaved ? rope_rows_kernel<E, WideItem, true> : rope_rows_kernel<E, WideItem, false>                                        \
          : interleaved ? rope_rows_kernel<E, NarrowItem, true> : rope_rows_kernel<E, NarrowItem, false>)
    hipLaunchKernelGGL(options().dtype == 1 ? CPMCU_ROPE(bf16) : CPMCU_ROPE(f16), grid, dim3(kThreads), 0, st, p);
#undef CPMCU_ROPE
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}

extern "C" int cpmcu_kv_append_slots(void* k_pool, void* v_pool, int num_pages, const int32_t* slots, const void* k, int64_t k_stride, const void* v,
                                     int64_t v_stride, int n, int Hkv, const int32_t* positions, const float* inv_freq, int rotary_dim, int interleaved,
                                     float magnitude, const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int Hq, void* stream) {
    CPMCU_CHECK_ARG(k_pool && v_pool && slots && k && v, "kv_append_slots: null pointer argument");
    CPMCU_CHECK_ARG(num_pages >= 1 && num_pages <= INT32_MAX / kPage, "kv_append_slots: num_pages=%d outside [1, %d]", num_pages, INT32_MAX / kPage);
    CPMCU_CHECK_ARG(n >= 0 && Hkv >= 1 && Hkv <= kMaxHeads, "kv_append_slots: n=%d Hkv=%d", n, Hkv);
    const bool rope = positions != nullptr || inv_freq != nullptr;
    if (rope) {
        if (int rc = check_turns("kv_append_slots", positions, inv_freq, rotary_dim, kHeadDim, magnitude)) return rc;
        CPMCU_CHECK_ARG(rotary_dim % 16 == 0, "kv_append_slots: rotary_dim=%d is not a multiple of 16", rotary_dim);
    }
    CPMCU_CHECK_ARG(rope || Hq == 0, "kv_append_slots: q is rotated here or not given");
    SlotParams p{};
    p.rope = RopeParams{{positions, inv_freq, rope ? rotary_dim / 2 : 0, magnitude, magnitude}, {q, q_out, q_stride, q_out_stride, Hq}, {}, n, kHeadDim, 1};
    if (int rc = check_rows("kv_append_slots", "q", p.rope.q, std::max(n, 1), kHeadDim)) return rc;
    const long width = (long)Hkv * kHeadDim;
    CPMCU_CHECK_ARG(k_stride >= width && v_stride >= width, "kv_append_slots: rows closer than their %ld values", width);
    CPMCU_CHECK_ARG(on_16_bytes(p.rope.q) && ((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0,
                    "kv_append_slots: rows and pools have to lie on 16 bytes");
    if (n == 0) return CPMCU_OK;
    p.k_pool = (f16*)k_pool;
    p.v_pool = (f16*)v_pool;
    p.slots = slots;
    p.k = k;
    p.v = v;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.Hkv = Hkv;
    p.num_slots = num_pages * kPage;
    p.heads_per_wg = 1;
    p.kv_blocks = ceil_div(n, kAppendRows) * (Hkv / p.heads_per_wg);
    p.rope.parts = Hq ? row_parts(n, Hq, kHeadDim / 16) : 1;
    const int q_blocks = Hq ? ceil_div(n, kRows) * p.rope.parts : 0;
    hipStream_t st = resolve_stream(stream);
    const dim3 grid(p.kv_blocks + q_blocks);
#define CPMCU_SLOTS(E) (interleaved ? kv_append_slots_kernel<E, true> : kv_append_slots_kernel<E, false>)
    hipLaunchKernelGGL(options().dtype == 1 ? CPMCU_SLOTS(bf16) : CPMCU_SLOTS(f16), grid, dim3(kThreads), 0, st, p);
#undef CPMCU_SLOTS
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
