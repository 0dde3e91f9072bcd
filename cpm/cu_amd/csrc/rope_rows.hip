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
constexpr int kMaxRows = 1 << 24; // of an append kMaxRows * 8 of all V heads (a launch has fewer than 2^32 threads)
constexpr int kRows = 4;         // rows of a workgroup: their angles are formed once for all heads

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

// An item of a head is two 16-byte pieces (WideItem) or two values (NarrowItem) that lie so far apart that neighbouring lanes' pieces are
// neighbours in memory: the two halves of pairs (i, i + half), behind those and with interleaved pairs the two halves of what there is.
struct ItemPlace {
    int first, second;   // values from the head's start
    int turn_a, turn_b;  // the pieces' angles: with pairs (i, i + half) both pieces have turn_a's; -1: none, the piece is copied
};
template <int W, bool IL>
__device__ inline ItemPlace item_place(int i, int half, int head_dim) {
    if constexpr (IL) {
        const int a = W * i, b = head_dim / 2 + W * i;
        return {a, b, a < 2 * half ? a / 2 : -1, b < 2 * half ? b / 2 : -1};
    } else {
        if (W * i < half) return {W * i, half + W * i, W * i, -1};
        const int rest = head_dim - 2 * half, j = W * i - half;
        return {2 * half + j, 2 * half + rest / 2 + j, -1, -1};
    }
}
template <typename E, bool IL>
struct WideItem {
    typedef typename Elem<E>::x8 X8;
    static constexpr int kWidth = 8;
    X8 a, b;
    __device__ static inline ItemPlace place(int i, int half, int head_dim) { return item_place<8, IL>(i, half, head_dim); }
    __device__ inline void load(const E* head, const ItemPlace& at) {
        a = *reinterpret_cast<const X8*>(head + at.first);
        b = *reinterpret_cast<const X8*>(head + at.second);
    }
    __device__ inline void store(E* head, const ItemPlace& at) const {
        __builtin_nontemporal_store(a, reinterpret_cast<X8*>(head + at.first));
        __builtin_nontemporal_store(b, reinterpret_cast<X8*>(head + at.second));
    }
    __device__ static inline void turn_pairs(X8& x, const float2* cs) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            E u = x[2 * j], v = x[2 * j + 1];
            rotate_pair(u, v, cs[j]);
            x[2 * j] = u;
            x[2 * j + 1] = v;
        }
    }
    __device__ inline void turn(const float2* cs, const ItemPlace& at) {
        if constexpr (IL) {
            if (at.turn_a >= 0) turn_pairs(a, cs + at.turn_a);
            if (at.turn_b >= 0) turn_pairs(b, cs + at.turn_b);
        } else if (at.turn_a >= 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                E u = a[j], v = b[j];
                rotate_pair(u, v, cs[at.turn_a + j]);
                a[j] = u;
                b[j] = v;
            }
        }
    }
};
// Rows off 16 bytes and rotary parts that are no whole pieces: two 2-byte values an item, with the same two divisions, and so bound by instructions: 8191 rows
// of 40 heads with 42 of 128 values turned 77 us (2.2 TB/s), with 64 turned in pieces 32.
template <typename E, bool IL>
struct NarrowItem {
    static constexpr int kWidth = 1;
    E a, b;
    // (interleaved pairs are neighbours: the item is the pair)
    __device__ static inline ItemPlace place(int i, int half, int head_dim) { return IL ? ItemPlace{2 * i, 2 * i + 1, i < half ? i : -1, -1} : item_place<1, false>(i, half, head_dim); }
    __device__ inline void load(const E* head, const ItemPlace& at) { a = head[at.first], b = head[at.second]; }
    __device__ inline void store(E* head, const ItemPlace& at) const { head[at.first] = a, head[at.second] = b; }
    __device__ inline void turn(const float2* cs, const ItemPlace& at) {
        if (at.turn_a >= 0) rotate_pair(a, b, cs[at.turn_a]);
    }
};

// Rows [r0, r0 + kRows) of q and k, this workgroup's part of their items.  place_of(r): a number >= 0, if row r has a position and a place;
// k_head(r, place, head): where the result of a key head goes.  Results are stored past the L2, whose dirty lines a launch would have to
// write back at its end (8191 rows of 40 heads 36.3 us, so 29.2); one item a thread at a time leaves most waves in flight (39 with four).
template <typename E, typename Item, typename PlaceOf, typename KHead>
__device__ inline void rope_run(const Turns& t, const HeadRows& q, const HeadRows& k, int n, int head_dim, int r0, int part, int parts, float2* cs, int* there,
                                PlaceOf&& place_of, KHead&& k_head) {
    const int tid = threadIdx.x, half = t.half;
    const int items = head_dim / (2 * Item::kWidth), per_row = (q.heads + k.heads) * items;
    const int rows = min(kRows, n - r0), total = rows * per_row;
    const int start = part * kThreads;
    for (int base = start; base < total; base += parts * kThreads) {
        const int i = base + tid;
        Item x;
        ItemPlace at;
        int row = 0, head = 0;
        if (i < total) {
            row = i / per_row;
            const int in_row = i - row * per_row;
            head = in_row / items;
            at = Item::place(in_row - head * items, half, head_dim);
            x.load(head < q.heads ? (const E*)q.in + (r0 + row) * q.in_stride + (long)head * head_dim : (const E*)k.in + (r0 + row) * k.in_stride + (long)(head - q.heads) * head_dim, at);
        }
        if (base == start) {
            for (int j = tid; j < rows * half; j += kThreads) cs[j] = turn_of(t, t.positions[r0 + j / half], j % half);
            if (tid < rows) there[tid] = place_of(r0 + tid);
            __syncthreads();
        }
        if (i < total && there[row] >= 0) {
            x.turn(cs + row * half, at);
            x.store(head < q.heads ? (E*)q.out + (r0 + row) * q.out_stride + (long)head * head_dim : (E*)k_head(r0 + row, there[row], head - q.heads), at);
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
    rope_run<E, Item<E, IL>>(p.t, p.q, p.k, p.n, p.head_dim, blockIdx.x * kRows, blockIdx.y, p.parts, cs, there, [&](int r) { return p.t.positions[r]; },
                              [&](int r, int, int head) { return (E*)p.k.out + r * p.k.out_stride + (long)head * p.head_dim; });
}

// How many workgroups share kRows rows: enough to give every thread one item while the launch is small.
int row_parts(int n, int heads, int items) {
    const int most = ceil_div(std::min(n, kRows) * heads * items, kThreads);
    return std::min(most, std::max(1, 1024 / ceil_div(n, kRows)));
}

bool on_16_bytes(const HeadRows& x) {
    return x.heads == 0 || (((uintptr_t)x.in | (uintptr_t)x.out) % 16 == 0 && x.in_stride % 8 == 0 && x.out_stride % 8 == 0);
}

// n rows in memory, and whether two such sets share any: never where one ends before the other begins, nor where they are columns apart of rows
// of one stride (the parts of a fused projection); rows of different strides that run through each other are taken to.
struct RowSet {
    const void* at;
    long stride, width;
};
bool share(const RowSet& a, const RowSet& b, int n) {
    const intptr_t d = (intptr_t)b.at - (intptr_t)a.at, s = 2 * a.stride;
    if (n == 0 || a.width == 0 || b.width == 0 || d >= (n - 1) * s + 2 * a.width || -d >= 2 * ((n - 1) * b.stride + b.width)) return false;
    const intptr_t column = (d % s + s) % s;
    return a.stride != b.stride || column < 2 * a.width || column + 2 * b.width > s;
}

int check_rows(const char* op, const char* name, const HeadRows& x, int n, int head_dim) {
    CPMCU_CHECK_ARG(x.heads >= 0 && x.heads <= kMaxHeads, "%s: %d heads of %s outside [0, %d]", op, x.heads, name, kMaxHeads);
    if (x.heads == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(x.in && x.out, "%s: null pointer argument", op);
    const long width = (long)x.heads * head_dim;
    CPMCU_CHECK_ARG(x.in_stride >= width && x.out_stride >= width, "%s: rows of %s closer than their %ld values", op, name, width);
    if (x.in == x.out && x.in_stride == x.out_stride) return CPMCU_OK;
    CPMCU_CHECK_ARG(!share({x.in, x.in_stride, width}, {x.out, x.out_stride, width}, n), "%s: the results of %s are neither in place nor in memory apart", op, name);
    return CPMCU_OK;
}

int check_turns(const char* op, const int32_t* positions, const float* inv_freq, int rotary_dim, int head_dim, float magnitude) {
    CPMCU_CHECK_ARG(positions && inv_freq, "%s: null pointer argument", op);
    CPMCU_CHECK_ARG(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, "%s: rotary_dim=%d is not an even number up to the head's %d values", op, rotary_dim, head_dim);
    CPMCU_CHECK_ARG(magnitude - magnitude == 0.f, "%s: magnitude is not finite", op);
    return CPMCU_OK;
}

// ---- append ----

struct SlotParams {
    RopeParams rope;  // q, and k without a place of its own; rope.t.positions null: rows that come rotated
    f16 *k_pool, *v_pool;
    const int32_t* slots;
    const uint16_t* v;
    long v_stride;
    int v_blocks, num_slots;
};

__device__ inline int slot_of(const SlotParams& p, int r) {
    const int s = p.slots[r];
    return s >= 0 && s < p.num_slots && (p.rope.t.positions == nullptr || p.rope.t.positions[r] >= 0) ? s : -1;
}

// V of ROWS rows and one head.  A page holds a dim in aligned groups of 16 slots (two 16-byte pieces), so V is transposed through LDS, and whoever has
// the first row of a run of consecutive slots inside such a group writes all of the run, up to fifteen rows beyond its own: pieces are
// whole wherever the rows of a request follow each other, however a workgroup's rows lie to the groups.  64 rows fill whole lines of four groups; where
// that leaves CUs idle, 16 rows do.  Everything is requested before anything is known of the slots: a decode step's rows are one round trip.
// 4001 rows of 4 heads: 6.1 us, K's workgroups alone 3.3, V's 5.6; with V's columns read without bank conflicts (65 % of LDS's cycles are) 5.6 and 5.0, with none
// read at all no less: what is left is the way from memory to memory.  8192 rows of 32 + 2 heads do not show it (26.4 us either way).
template <int ROWS>
struct VStage {
    int slot[ROWS + 16];  // [i + 1]: row i of the workgroup's, -1: none
    uint16_t v[(ROWS + 15) * kAppendStride];
};
template <int ROWS>
__device__ inline void append_v(const SlotParams& p, int block, VStage<ROWS>& lds) {
    constexpr int kAll = ROWS + 15, kSide = ROWS / 16;  // rows that may be needed; groups that are written side by side
    const int tid = threadIdx.x, lane = tid & 63, n = p.rope.n, Hkv = p.rope.k.heads;
    const int g = block % Hkv, r0 = block / Hkv * ROWS;
    uint4 v[(kAll * 16 + kThreads - 1) / kThreads];
#pragma unroll
    for (int u = 0; u * kThreads < kAll * 16; ++u) {
        const int r = (u * kThreads + tid) >> 4;
        if (r < kAll && r0 + r < n) v[u] = *reinterpret_cast<const uint4*>(p.v + (r0 + r) * p.v_stride + (long)g * kHeadDim + (tid & 15) * 8);
    }
    if (tid <= kAll) lds.slot[tid] = r0 + tid >= 1 && r0 + tid - 1 < n ? slot_of(p, r0 + tid - 1) : -1;
#pragma unroll
    for (int u = 0; u * kThreads < kAll * 16; ++u) {
        const int r = (u * kThreads + tid) >> 4;
        if (r < kAll && r0 + r < n) {
            uint2* to = reinterpret_cast<uint2*>(lds.v + r * kAppendStride + (tid & 15) * 8);
            to[0] = make_uint2(v[u].x, v[u].y);
            to[1] = make_uint2(v[u].z, v[u].w);
        }
    }
    __syncthreads();
    // bit i: row i has a place; it goes on with the run of the row before it
    const auto joins = [&](int i) { return i < kAll && lds.slot[i + 1] >= 0 && (lds.slot[i + 1] & 15) != 0 && lds.slot[i] == lds.slot[i + 1] - 1; };
    const uint64_t joined = __ballot(joins(lane)), joined_hi = ROWS + 15 > 64 ? __ballot(joins(64 + lane)) : 0;
    const uint64_t leaders = __ballot(lane < ROWS && lds.slot[min(lane, ROWS) + 1] >= 0) & ~joined;
    if (leaders == 0) return;
    const auto run_of = [&](int i) {  // rows of the run that row i leads
        const uint32_t next = (uint32_t)(joined >> i >> 1) | (i >= 32 ? (uint32_t)(joined_hi << (63 - i)) : 0u);
        return 1 + __builtin_ctz(~(next & 0x7FFFu));
    };
    const size_t head = (size_t)g * kHeadDim;
    const auto dim_row = [&](int s, int d) { return reinterpret_cast<uint16_t*>(p.v_pool) + ((size_t)(s / kPage) * Hkv * kHeadDim + head + d) * kPage + (s % kPage & ~15); };
    if (__popcll(leaders) > ROWS / 4) {
        // short runs: value by value, all rows from the first leader's to the last run's end
        const int d = tid & (kHeadDim - 1), last = 63 - __builtin_clzll(leaders), end = last + run_of(last);
        for (int i = __builtin_ctzll(leaders) + (tid >> 7); i < end; i += 2) {
            const int s = lds.slot[i + 1];
            if (s >= 0) dim_row(s, d)[v_slot16(s & 15)] = lds.v[i * kAppendStride + d];
        }
        return;
    }
    const int piece = tid & 1, side = (tid >> 1) % kSide, d0 = tid / (2 * kSide);
    uint64_t rest = leaders;
    while (rest) {
        int i = -1;
#pragma unroll
        for (int k = 0; k < kSide; ++k) {
            if (k == side && rest) i = __builtin_ctzll(rest);
            rest &= rest - 1;  // (of none: none)
        }
        if (i < 0) continue;
        const int s = lds.slot[i + 1], len = run_of(i), first = piece * 4 - (s & 15);  // row i + first + (j & 3) + (j >> 2) * 8 is slot j's
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = first + (j & 3) + (j >> 2) * 8;
            in |= r >= 0 && r < len ? 1u << j : 0u;
        }
        if (in == 0) continue;
        for (int d = d0; d < kHeadDim; d += kThreads / (2 * kSide)) {
            uint32_t y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = lds.v[(i + min(max(first + (j & 3) + (j >> 2) * 8, 0), len - 1)) * kAppendStride + d];
            uint16_t* dst = dim_row(s, d) + piece * 8;
            if (in == 0xFFu) {
                typedef uint32_t U4 __attribute__((ext_vector_type(4)));
                __builtin_nontemporal_store(U4{y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16}, reinterpret_cast<U4*>(dst));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if ((in >> j) & 1u) dst[j] = (uint16_t)y[j];
            }
        }
    }
}

template <typename E, bool IL, int ROWS>
__global__ __launch_bounds__(kThreads) void kv_append_slots_kernel(SlotParams p) {
    __shared__ union {
        VStage<ROWS> v;
        struct {
            float2 cs[kRows * kMaxHalf];
            int there[kRows];
        } rope;
    } lds;
    if ((int)blockIdx.x < p.v_blocks) {
        append_v<ROWS>(p, blockIdx.x, lds.v);
        return;
    }
    const int b = blockIdx.x - p.v_blocks, Hkv = p.rope.k.heads;
    rope_run<E, WideItem<E, IL>>(p.rope.t, p.rope.q, p.rope.k, p.rope.n, kHeadDim, b / p.rope.parts * kRows, b % p.rope.parts, p.rope.parts, lds.rope.cs, lds.rope.there,
                                 [&](int r) { return slot_of(p, r); },
                                 [&](int, int s, int head) { return p.k_pool + (((size_t)(s / kPage) * Hkv + head) * kPage + s % kPage) * kHeadDim; });
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" int cpmcu_rope_rows(const int32_t* positions, const float* inv_freq, int rotary_dim, int interleaved, float magnitude, int transposed,
                               const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int Hq, const void* k, int64_t k_stride, void* k_out,
                               int64_t k_out_stride, int Hkv, int head_dim, int n, void* stream) {
    CPMCU_CHECK_ARG(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 2 * kMaxHalf, "rope_rows: head_dim=%d is not an even number up to %d", head_dim, 2 * kMaxHalf);
    CPMCU_CHECK_ARG(n >= 0 && n < kMaxRows, "rope_rows: n=%d outside [0, %d)", n, kMaxRows);
    if (n == 0) return CPMCU_OK;  // (rows that are not there may have no memory)
    if (int rc = check_turns("rope_rows", positions, inv_freq, rotary_dim, head_dim, magnitude)) return rc;
    RopeParams p{{positions, inv_freq, rotary_dim / 2, magnitude, transposed ? -magnitude : magnitude}, {q, q_out, q_stride, q_out_stride, Hq}, {k, k_out, k_stride, k_out_stride, Hkv}, n, head_dim, 1};
    if (int rc = check_rows("rope_rows", "q", p.q, n, head_dim)) return rc;
    if (int rc = check_rows("rope_rows", "k", p.k, n, head_dim)) return rc;
    const long q_width = (long)Hq * head_dim, k_width = (long)Hkv * head_dim;
    CPMCU_CHECK_ARG(!share({q_out, q_out_stride, q_width}, {k, k_stride, k_width}, n) && !share({k_out, k_out_stride, k_width}, {q, q_stride, q_width}, n) &&
                        !share({q_out, q_out_stride, q_width}, {k_out, k_out_stride, k_width}, n),
                    "rope_rows: results lie in the memory of the other rows");
    if (Hq + Hkv == 0) return CPMCU_OK;
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
    CPMCU_CHECK_ARG(num_pages >= 1 && num_pages <= INT32_MAX / kPage, "kv_append_slots: num_pages=%d outside [1, %d]", num_pages, INT32_MAX / kPage);
    CPMCU_CHECK_ARG(n >= 0 && Hkv >= 1 && Hkv <= kMaxHeads && n < kMaxRows && (int64_t)n * Hkv < kMaxRows * 8, "kv_append_slots: n=%d Hkv=%d", n, Hkv);
    if (n == 0) return CPMCU_OK;  // (rows that are not there may have no memory)
    CPMCU_CHECK_ARG(k_pool && v_pool && slots && k && v, "kv_append_slots: null pointer argument");
    const bool rope = positions != nullptr || inv_freq != nullptr;
    if (rope) {
        if (int rc = check_turns("kv_append_slots", positions, inv_freq, rotary_dim, kHeadDim, magnitude)) return rc;
        CPMCU_CHECK_ARG(rotary_dim % 16 == 0, "kv_append_slots: rotary_dim=%d is not a multiple of 16", rotary_dim);
    }
    CPMCU_CHECK_ARG(rope || Hq == 0, "kv_append_slots: q is rotated here or not given");
    SlotParams p{};
    p.rope = RopeParams{{positions, inv_freq, rope ? rotary_dim / 2 : 0, magnitude, magnitude}, {q, q_out, q_stride, q_out_stride, Hq}, {k, nullptr, k_stride, 0, Hkv}, n, kHeadDim, 1};
    if (int rc = check_rows("kv_append_slots", "q", p.rope.q, n, kHeadDim)) return rc;
    const long width = (long)Hkv * kHeadDim;
    CPMCU_CHECK_ARG(k_stride >= width && v_stride >= width, "kv_append_slots: rows closer than their %ld values", width);
    CPMCU_CHECK_ARG(on_16_bytes(p.rope.q) && ((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0,
                    "kv_append_slots: rows and pools have to lie on 16 bytes");
    const long q_width = (long)Hq * kHeadDim, pool = (long)Hkv * kHeadDim * kPage;
    CPMCU_CHECK_ARG(!share({q_out, q_out_stride, q_width}, {k, k_stride, width}, n) && !share({q_out, q_out_stride, q_width}, {v, v_stride, width}, n),
                    "kv_append_slots: the results of q lie in the memory of k or v");
    CPMCU_CHECK_ARG(!share({k_pool, pool, pool}, {v_pool, pool, pool}, num_pages), "kv_append_slots: the K and the V pool share memory");
    p.k_pool = (f16*)k_pool;
    p.v_pool = (f16*)v_pool;
    p.slots = slots;
    p.v = (const uint16_t*)v;
    p.v_stride = v_stride;
    p.num_slots = num_pages * kPage;
    const bool long_runs = (int64_t)ceil_div(n, 64) * Hkv >= 128;  // (4001 rows of 4 heads 8.3 us in 16s, 6.1 in 64s; 64 rows of 8 heads, a page each, 6.3 and 7.5)
    p.v_blocks = ceil_div(n, long_runs ? 64 : 16) * Hkv;
    p.rope.parts = row_parts(n, Hq + Hkv, kHeadDim / 16);
    hipStream_t st = resolve_stream(stream);
    const dim3 grid(p.v_blocks + ceil_div(n, kRows) * p.rope.parts);
#define CPMCU_SLOTS(E)                                                                                                              \
    (long_runs ? interleaved ? kv_append_slots_kernel<E, true, 64> : kv_append_slots_kernel<E, false, 64>                           \
               : interleaved ? kv_append_slots_kernel<E, true, 16> : kv_append_slots_kernel<E, false, 16>)
    hipLaunchKernelGGL(options().dtype == 1 ? CPMCU_SLOTS(bf16) : CPMCU_SLOTS(f16), grid, dim3(kThreads), 0, st, p);
#undef CPMCU_SLOTS
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
