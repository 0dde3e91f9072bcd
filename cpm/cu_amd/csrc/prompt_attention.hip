// Causal attention of the new rows of several requests over their pages: whole prompts, chunks far into a context, single rows between them.
//
//   out[t][h] = sum_x p_x v[x] / sum_x p_x,  p_x = exp(scale (q[t][h] . k[x] - max)),  x from 0 to the row's own position,
//
// k and v the tokens of the row's request and of the KV head of h.  The rows of a request and the heads on one KV head are one matrix of
// rows (token-major), cut into tiles of 128; a workgroup takes a tile, or a part of its keys, through them 64 at a time, with the running
// reference and sum of its softmax.  What bounds it: 4 * 128 operations a row, head and key on the matrix cores, of which two workgroups a CU keep
// as many busy as the card's power allows (one of them forms products while the other one has its scores in the vector units).
//
// Which tiles there are follows from lengths that only the device knows, so a launch of one workgroup lists them first: longest first, those
// that would outlast the others by much cut into pieces, which a last launch joins.  Where they are few, each workgroup finds its own.
#include "batch_attention.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace cpmcu {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kWaveRows = 32, kTileRows = kWaves * kWaveRows;
constexpr int kStages = 2;
constexpr int kKBytes = kTileKeys * kHeadDim * 2, kStageBytes = 2 * kKBytes;
// Probabilities are powers of two of a score less the softmax's reference, which is kLift below the largest score that it has followed and stays until a lane's 32 of a tile add up to
// more than kMostSum.  fp16 has fewer bits below 2^-14: with a lift of 10 a probability keeps all of them down to e^-16.6 of the largest (without, to e^-9.7: behind one key of e^16.5
// times the weight of each other, the others' sum was 2 % off), and what passes 65504 is infinity, as the sum is then.  bf16 has the range of 32 bits.
template <typename E>
struct Range {
    static constexpr float kLift = Elem<E>::kDtype == 0 ? 10.f : 0.f, kMostSum = Elem<E>::kDtype == 0 ? FLT_MAX : 4096.f;
};

// ---- the list of work ----

// The keys [begin, end) * 64 for rows [128 tile, 128 tile + 128) of the packed rows of a request whose `rows` rows start at row0 of the batch and
// at position p0.  slot: where its part of the results waits for the others, -1 if it has all of its keys.
struct Work {
    int row0, rows, p0, request, tile, begin, end, slot;
};
// A tile in `pieces` parts, from slot on.
struct Join {
    int row0, rows, tile, slot, pieces, pad[3];
};
struct Listed {
    int works, joins, pad[6];
};
// Pieces are made of tiles that have more than 1 / kParts of all keys, on all KV heads, and more than what is worth its part of the join: kLeastKeys tiles of keys where there are
// few tiles of rows, kMostKeys where there are enough for all CUs, by the square of their number in between.  Measured with 8, 16, 24 and 64 throughout (us): 8 rows at 12000 cached
// (2 tiles) 24, 27, 33, 68; 64 rows at 4000 (16) 22, 26, 31, 66; 512 rows at 8000 on 8 heads (128) 90, 89, 92, 97; 1000 rows (250) 28, 24, 24, 24; 4 x 256 rows at 6000 (256)
// 125, 125, 125, 110; 4096 rows (1024) 163, 163, 163, 146.  With this rule 24, 22, 92, 24, 116 and 151.
// (The lengths do not count: 1777 rows of 16 heads, 224 tiles of up to 33 tiles of keys, are not cut, 38.9; with pieces of 8, 12 and 17 at least 46.5, 38.7 and 38.1.)
constexpr int kParts = 896, kLeastKeys = 8, kMostKeys = 64;
constexpr int kMostChunk = 1 << 21;  // longer than any tile's keys
__host__ __device__ inline int64_t least_of(int64_t tiles, int Hkv) {
    const int64_t full = tiles * Hkv, least = full * full / 1024;
    return least < kLeastKeys ? kLeastKeys : least > kMostKeys ? kMostKeys : least;
}

struct PlanParams {
    const int32_t *row_offsets, *positions;
    int num_requests, max_blocks, n, group, Hkv, most_tiles, slots;
    Listed* listed;
    Work* works;
    Join* joins;
};

// A workgroup's threads have EACH requests each, then every THREADS-th tile of rows.
struct Tile {
    int request, tile, keys;  // keys: tiles of 64 of them that the last row sees
};
// A lane's value and those of the lanes before it, added up within rows of 16 lanes and then from row to row, without LDS (0 is nothing).
template <typename T, typename F>
__device__ inline T wave_upto(T v, F add) {
    const auto moved = [&](auto from, auto rows) {
        T x = 0;
#pragma unroll
        for (int part = 0; part < (int)sizeof(T); part += 4)
            x |= (T)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)((unsigned long long)v >> (8 * part)), decltype(from)::value, decltype(rows)::value, 0xf, false) << (part ? 32 : 0);
        return x;
    };
    typedef std::integral_constant<int, 0xf> All;
    v = add(v, moved(std::integral_constant<int, 0x111>{}, All{}));  // the lane one before, two, four, eight
    v = add(v, moved(std::integral_constant<int, 0x112>{}, All{}));
    v = add(v, moved(std::integral_constant<int, 0x114>{}, All{}));
    v = add(v, moved(std::integral_constant<int, 0x118>{}, All{}));
    v = add(v, moved(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}));  // every second row: the last lane's of the row before
    v = add(v, moved(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}));  // the upper half: lane 31's
    return v;
}
template <int THREADS, int EACH>
struct Plan {
    static constexpr int kMost = THREADS * EACH, kPlanWaves = THREADS / 64;
    struct Lds {
        int tile_end[kMost], row0[kMost], rows[kMost], first[kMost];
        unsigned long long wave_sum[2][kPlanWaves];
    };
    const PlanParams& p;
    Lds& lds;
    int tid;

    // What the threads before this one have, and what all of them have.
    template <typename T, typename F>
    __device__ T before(T mine, int part, F add, T& all) const {
        const int lane = tid & 63, wave = tid >> 6;
        const T upto = wave_upto(mine, add);
        if (lane == 63) lds.wave_sum[part][wave] = (unsigned long long)upto;
        T lanes = __shfl_up(upto, 1);
        if (lane == 0) lanes = 0;
        __syncthreads();
        T waves = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) {
            if (w == wave) waves = all;
            all = add(all, (T)lds.wave_sum[part][w]);
        }
        return add(waves, lanes);
    }
    // The requests' rows and tiles: how many tiles there are.  (Totals are most_tiles at most: they stop there, so their grouping does not matter.)
    __device__ int requests() const {
        const auto add = [&](int x, int y) { return min(x + y, p.most_tiles); };
        int tiles[EACH], mine = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int r = tid * EACH + e;
            int lo = 0, count = 0, p0 = -1;
            if (r < p.num_requests) {
                lo = min(max(p.row_offsets[r], 0), p.n);
                count = min(max(p.row_offsets[r + 1], lo), p.n) - lo;
                if (count > 0) p0 = p.positions[lo];
                const int64_t room = (int64_t)p.max_blocks * kPage - p0;
                count = p0 < 0 ? 0 : (int)min((int64_t)count, max(room, (int64_t)0));
            }
            tiles[e] = (int)(((int64_t)count * p.group + kTileRows - 1) / kTileRows);
            mine = add(mine, tiles[e]);
            lds.row0[r] = lo;
            lds.rows[r] = count;
            lds.first[r] = p0;
        }
        int all, upto = before(mine, 0, add, all);
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            upto = add(upto, tiles[e]);
            lds.tile_end[tid * EACH + e] = upto;
        }
        __syncthreads();
        return all;
    }
    __device__ Tile find(int t) const {
        int lo = 0, hi = p.num_requests - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (lds.tile_end[mid] > t) hi = mid;
            else lo = mid + 1;
        }
        Tile f{lo, t - (lo > 0 ? lds.tile_end[lo - 1] : 0), 0};
        const int last = min(lds.rows[lo] - 1, (int)(((uint32_t)(f.tile + 1) * kTileRows - 1) / (uint32_t)p.group));  // (rows times heads: 31 bits)
        f.keys = (lds.first[lo] + last) / kTileKeys + 1;
        return f;
    }
    // How many tiles of keys a piece has at most, from how many tiles of rows there are and what they have together.
    __device__ int chunk_of(int all, unsigned long long cost) const {
        // What is cut fits the slots: of more than 1 / kParts of all keys, a tile of t makes at most 2 t / chunk pieces; else t / chunk + 1, and there are twice as many slots as tiles.
        if (p.slots == 0) return kMostChunk;
        const int64_t share = (int64_t)((cost * p.Hkv + kParts - 1) / kParts);
        const int room = p.slots - all, cap = 2 * ((kParts + p.Hkv - 1) / p.Hkv);
        // (a quotient of 64-bit floats, one tile too long at most, is a fraction of a division of 64-bit whole numbers)
        const int64_t fits = room > 0 && p.slots < cap ? (int64_t)((double)cost / (double)room) + 2 : 0;
        return (int)min(max(max(share, fits), least_of(all, p.Hkv)), (int64_t)kMostChunk);
    }
    __device__ int pieces_of(int keys, int chunk) const { return (int)(((uint32_t)keys + chunk - 1) / (uint32_t)chunk); }
    __device__ Work piece(const Tile& f, int i, int pieces, int slot) const {  // (2^20 tiles of keys, 2^11 pieces)
        const int r = f.request;
        return Work{lds.row0[r], lds.rows[r], lds.first[r], r, f.tile, (int)((uint32_t)f.keys * i / pieces), (int)((uint32_t)f.keys * (i + 1) / pieces), slot < 0 ? -1 : slot + i};
    }
    __device__ Join join(const Tile& f, int slot, int pieces) const { return Join{lds.row0[f.request], lds.rows[f.request], f.tile, slot, pieces, {0, 0, 0}}; }
};

// The launch is round trips -- offsets, positions, the list -- and meetings of its waves: with a request and a tile a thread 4.4 us, with four waves in place of sixteen
// 3.1; 1025 tiles, behind a launch that has taken the clock down, 11.6 with four waves and 9 with sixteen.
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void prompt_plan_kernel(PlanParams p) {
    constexpr int kClasses = 64;
    __shared__ typename Plan<THREADS, EACH>::Lds lds;
    __shared__ int in_class[kClasses], slots, joins;
    const int tid = threadIdx.x;
    const Plan<THREADS, EACH> plan{p, lds, tid};
    if (tid < kClasses) in_class[tid] = 0;
    if (tid == 0) slots = joins = 0;
    const int all = plan.requests();
    const Tile own = tid < all ? plan.find(tid) : Tile{0, 0, 0};  // (most launches have no more)
    unsigned long long mine = own.keys, cost;
    for (int t = tid + THREADS; t < all; t += THREADS) mine += plan.find(t).keys;
    plan.before(mine, 1, [](unsigned long long x, unsigned long long y) { return x + y; }, cost);
    const int chunk = plan.chunk_of(all, cost);
    const auto pieces_of = [&](int keys) { return plan.pieces_of(keys, chunk); };
    // Longest first: counted in classes of a quarter of an octave, then put in their places.
    const auto class_of = [&](int keys, int pieces) {
        const int length = (keys + pieces - 1) / pieces, msb = 31 - __clz(max(length, 1));
        return kClasses - 1 - min(length < 4 ? length : 4 * (msb - 1) + (length >> (msb - 2) & 3), kClasses - 1);
    };
    for (int t = tid; t < all; t += THREADS) {
        const Tile f = t == tid ? own : plan.find(t);
        const int pieces = pieces_of(f.keys);
        atomicAdd(&in_class[class_of(f.keys, pieces)], pieces);
    }
    __syncthreads();
    if (tid < 64) {
        const int here = in_class[tid];
        int sum = here;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int from = __shfl_up(sum, d);
            if (tid >= d) sum += from;
        }
        in_class[tid] = sum - here;  // from here on: the next free place
        if (tid == 63) p.listed->works = sum;
    }
    __syncthreads();
    for (int t = tid; t < all; t += THREADS) {
        const Tile f = t == tid ? own : plan.find(t);
        const int pieces = pieces_of(f.keys), at = atomicAdd(&in_class[class_of(f.keys, pieces)], pieces);
        int slot = -1;
        if (pieces > 1) {
            slot = atomicAdd(&slots, pieces);
            p.joins[atomicAdd(&joins, 1)] = plan.join(f, slot, pieces);
        }
        for (int i = 0; i < pieces; ++i) p.works[at + i] = plan.piece(f, i, pieces, slot);
    }
    __syncthreads();
    if (tid == 0) p.listed->joins = joins;
}

// The same for a workgroup by itself, its own piece only: where the card has room for all tiles at once (two workgroups a CU) their order does not matter, and the launch of the
// list is spared (37 rows 9.9 to 7.9 us, 1777 of 16 heads 43 to 38), for 1.5 us more in each workgroup, those behind the last piece among them: the grid is what tables of max_blocks columns may need, and up
// to twice the card's room is worth it.  Nothing here depends on the order of atomics, so all workgroups find the same.
constexpr int kOwnThreads = 256, kOwnGrid = 512;
struct OwnPlan {
    Plan<kOwnThreads, 1>::Lds lds;
    Work work;
};
__device__ inline Work uniform(const Work& w) {
    return Work{__builtin_amdgcn_readfirstlane(w.row0), __builtin_amdgcn_readfirstlane(w.rows), __builtin_amdgcn_readfirstlane(w.p0), __builtin_amdgcn_readfirstlane(w.request),
                __builtin_amdgcn_readfirstlane(w.tile), __builtin_amdgcn_readfirstlane(w.begin), __builtin_amdgcn_readfirstlane(w.end), __builtin_amdgcn_readfirstlane(w.slot)};
}
__device__ bool own_work(const PlanParams& p, OwnPlan& own, int index, bool writes, Work& work) {
    const int tid = threadIdx.x;
    const Plan<kOwnThreads, 1> plan{p, own.lds, tid};
    const int all = plan.requests();
    const bool has = tid < all;
    const Tile f = has ? plan.find(tid) : Tile{0, 0, 0};
    uint32_t cost;  // (2^8 tiles of 2^20 tiles of keys)
    const auto plus = [](uint32_t x, uint32_t y) { return x + y; };
    plan.before((uint32_t)f.keys, 1, plus, cost);
    const int chunk = plan.chunk_of(all, cost), pieces = plan.pieces_of(f.keys, chunk);
    const bool cut = pieces > 1;
    // pieces (2^8 tiles, 2^11 more pieces) and slots in 16 bits each
    uint32_t total;
    const uint32_t at = plan.before((uint32_t)pieces | (cut ? (uint32_t)pieces << 16 : 0u), 0, plus, total);
    const int works = (int)(total & 0xffff), slot = cut ? (int)(at >> 16) : -1;
    const int x = works - 1 - index - (int)(at & 0xffff);  // the last tiles of a prompt are the longest
    if (x >= 0 && x < pieces) own.work = plan.piece(f, x, pieces, slot);
    if (writes) {  // (by the whole workgroup)
        uint32_t joins;
        const uint32_t join = plan.before((uint32_t)cut, 1, plus, joins);
        if (cut) p.joins[join] = plan.join(f, slot, pieces);
        if (tid == 0) p.listed->joins = (int)joins;
    }
    __syncthreads();
    work = own.work;
    return index < works;
}

// ---- attention ----

struct PromptParams {
    BatchRows b;
    PlanParams plan;
    float4* parts;  // [slot][KV head][wave][16 quads][64 lanes]: sums that have not been divided yet
    float2* stats;  // [slot][KV head][128]: (reference in powers of two, sum)
};

// K: a row of 256 bytes a key, its 16-byte pieces exchanged by the key's number; V: a row of 128 bytes a dim, by half of the dim's (even and
// odd rows are in different halves of the banks).  Both ways the matrix operands are read without conflicts.
__device__ inline int k_at(int key, int piece) { return key * 256 + ((piece ^ (key & 15)) << 4); }
__device__ inline int v_at(int d, int piece) { return kKBytes + d * 128 + ((piece ^ ((d >> 1) & 7)) << 4); }

template <typename E>
__device__ inline bool not_finite(E v) {
    constexpr uint32_t kOnes = Elem<E>::kDtype == 0 ? 0x7c00u : 0x7f80u;
    return (__builtin_bit_cast(uint16_t, v) & kOnes) == kOnes;
}

// A tile of keys is two phases of a wave: its scores become probabilities (vector instructions, 650 cycles), and the product with V and the next tile's scores are formed
// (matrix instructions, 1024).  The CU's two workgroups know nothing of each other, so the one's phases fall beside the other's.  (Eight waves in one workgroup, with
// barriers between the phases that keep one wave of a SIMD on either unit: 2.5 % faster on the largest prompt, and 10 to 35 % slower on small ones, whose tiles are too few;
// all eight in step: 8 % slower than that.)  K and V have two stages each: V(i + 1) and K(i + 2) are requested when everybody is through with tile i - 1's products, and have the
// time of a tile to come.
//
// The softmax's reference is the largest score of a row's first tile (of the first that has any but minus infinities), and follows only when a tile's probabilities add up to more than
// kMostSum: their sum is needed anyway, their largest score is not (30 vector instructions of 130).
// LISTED: the list has been made by a launch before this one.
template <typename E, bool LISTED>
__global__ __launch_bounds__(kThreads, 2) void prompt_attention_kernel(PromptParams p) {
    typedef typename Elem<E>::x8 X8;
    typedef typename Elem<E>::x4 X4;
    typedef typename Elem<E>::x2 X2;
    __shared__ __attribute__((aligned(1024))) char ring[kStages * kStageBytes];
    const BatchRows& b = p.b;
    const int g = blockIdx.x % b.Hkv, index = blockIdx.x / b.Hkv;
    Work w;
    if constexpr (LISTED) {
        // (the entry behind the list is memory too: one round trip for both)
        w = p.plan.works[index];
        if (index >= p.plan.listed->works) return;
    } else {
        static_assert(sizeof(OwnPlan) <= sizeof(ring) && kOwnThreads == kThreads, "in the place of the first tiles");
        if (!own_work(p.plan, *reinterpret_cast<OwnPlan*>(ring), index, blockIdx.x == 0, w)) return;
        w = uniform(w);
        __syncthreads();  // (it has been read)
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qcol = lane & 31, hf = lane >> 5;
    const int packed = w.rows * b.group, base_row = w.tile * kTileRows + wave * kWaveRows;
    const int R = base_row + qcol, Rc = min(R, packed - 1);
    const bool wave_ok = base_row < packed;
    const int pos = w.p0 + divide(Rc, b.group, b.group_inverse).q;
    // Where the rows of a lane's sixteen, four apart, begin: one division for the first of them.
    const Quotient four = divide(4, b.group, b.group_inverse);
    struct Rows {
        int64_t at;
        int head;
    };
    const auto first_row = [&](int R, int64_t stride) {
        const Quotient row = divide(R, b.group, b.group_inverse);
        return Rows{(int64_t)(w.row0 + row.q) * stride + (g * b.group + row.r) * kHeadDim, row.r};
    };
    const auto next_row = [&](Rows& x, int64_t stride) {
        const bool over = x.head + four.r >= b.group;
        x.head += over ? four.r - b.group : four.r;
        x.at += four.q * stride + four.r * kHeadDim + (over ? stride - b.group * kHeadDim : 0);
    };
    const int wave_last = __builtin_amdgcn_readlane(pos, 31);  // the position of the wave's last row
    const int n = w.end - w.begin;

    // Page numbers: 64 of them at a time, one a lane.
    const int32_t* const table = b.block_tables + (size_t)w.request * b.table_stride;
    int pages_from = 0, pages = 0;
    const auto load_pages = [&](int block) {
        pages_from = block;
        pages = page_within(table[min(block + lane, b.max_blocks - 1)], b.num_pages);
    };
    load_pages(w.begin * kTileKeys / kPage);

    // What each lane requests of a tile: 4 KB of K's (16 keys) and of V's (32 dims) a wave.  Four keys or eight dims on, the pieces' exchange differs in bits 2 and 3, or 2; a
    // page has 64 KB a head in either pool.
    uint32_t k_off, v_off;
    {
        const int key = wave * 16 + (lane >> 4), d = wave * 32 + (lane >> 3);
        k_off = (uint32_t)(key * kHeadDim + ((lane & 15) ^ (key & 15)) * 8) * 2u;
        v_off = (uint32_t)(d * kPage + ((lane & 7) ^ ((d >> 1) & 7)) * 8) * 2u;
    }
    const uint32_t ring_at = (uint32_t)(uintptr_t)(lds_ptr_t)ring + wave * 4096;
    const uint32_t v_off1 = (v_off ^ 64u) + 3u * 1024u, v_off2 = v_off + 6u * 1024u, v_off3 = (v_off ^ 64u) + 9u * 1024u;
    static_assert(kPage * kHeadDim * 2 == 1 << 16, "64 KB a page and head");
    uint64_t page_at = 0;  // of the tile whose K has been requested last: V(j) is requested behind K(j), ahead of K(j + 1)
    const auto request_k = [&](int i, int stage) {
        const int block = (w.begin + i) * kTileKeys / kPage;
        if (block - pages_from >= 64) load_pages(block);
        page_at = (uint64_t)(uint32_t)(__builtin_amdgcn_readlane(pages, block - pages_from) * b.Hkv + g) << 16;
        request_4k((const char*)b.k_pool + page_at + (w.begin + i) * kTileKeys % kPage * (kHeadDim * 2), k_off, k_off ^ 64u, k_off ^ 128u, k_off ^ 192u, ring_at + stage * kStageBytes);
    };
    const auto request_v = [&](int i, int stage) {
        request_4k((const char*)b.v_pool + page_at + (w.begin + i) * kTileKeys % kPage * 2, v_off, v_off1, v_off2, v_off3, ring_at + stage * kStageBytes + kKBytes);
    };
    const auto meet = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    request_k(0, 0);
    request_v(0, 0);
    // Q's rows come through LDS, whole, in the stage that the second tile will have.
    char* const q_stage = ring + kStageBytes + wave * (kWaveRows * 256);
    Rows q_row = first_row(base_row + (lane >> 4), b.q_stride);
    const int64_t q_last = first_row(packed - 1, b.q_stride).at;
#pragma unroll
    for (int x = 0; x < kWaveRows / 4; ++x) {
        const int r = x * 4 + (lane >> 4);
        const uint16_t* const from = b.q + (base_row + r < packed ? q_row.at : q_last) + ((lane & 15) ^ (r & 15)) * 8;
        next_row(q_row, b.q_stride);
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"((uint32_t)(uintptr_t)(lds_ptr_t)(q_stage + x * 1024)) : "memory", "m0");
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    X8 qreg[8];  // as the second operand of S^T = K Q^T: lane (qcol, hf) has dims 16 ks + 8 hf + [0, 8)
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qreg[ks] = *reinterpret_cast<const X8*>(q_stage + k_at(qcol, 2 * ks + hf));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    meet();
    if (n > 1) request_k(1, 1);

    f32x16 oacc[4], sacc[2];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[db][r] = 0.f;
    float m_ref = -INFINITY, l_run = 0.f;
    // Operand x of a tile's K (keys 32 (x % 2) + [0, 32), dims 16 (x / 2) + [0, 16)) and V (dims 32 (x % 4) + [0, 32), keys 16 (x / 4) + [0, 16)): the pieces' exchange
    // makes the step along a row an exclusive or.
    typedef __attribute__((address_space(3))) const X8* lds_x8_t;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_ptr_t)ring, k_base = lds_at + k_at(qcol, hf), v_base = lds_at + v_at(qcol, hf);
    const auto k_of = [&](int i) { return k_base + (i % kStages) * kStageBytes; };
    const auto v_of = [&](int i) { return v_base + (i % kStages) * kStageBytes; };
    const auto read_k = [&](uint32_t at, int x) { return *reinterpret_cast<lds_x8_t>((at ^ ((x >> 1) * 32)) + (x & 1) * 32 * 256); };
    const auto read_v = [&](uint32_t at, int x) { return *reinterpret_cast<lds_x8_t>((at ^ ((x >> 2) * 32)) + (x & 3) * 32 * 128); };
    const auto clear_scores = [&]() {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) sacc[kb][r] = 0.f;
    };
    const auto scores_of = [&](int i) {
        const uint32_t at = k_of(i);
        X8 kf[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) kf[x] = read_k(at, x);
        clear_scores();
#pragma unroll
        for (int x = 0; x < 16; ++x) sacc[x & 1] = Elem<E>::mfma_32x32x16(kf[x], qreg[x >> 1], sacc[x & 1]);
    };
    // P^T as the second operand of O^T = V^T P^T, rounded to the element type: step j has keys 16 j + {4 hf + [0, 4), 8 + 4 hf + [0, 4)}
    X8 pb[4];
    const auto refer = [&]() {  // to the tile's largest score (kLift below), where that is larger
        float tmax = sacc[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, sacc[kb][r]);
        // (the row's other keys are 32 lanes away)
        const float m_new = fmaxf(m_ref, fmaxf(tmax, __shfl_xor(tmax, 32)) * b.scale_log2 - Range<E>::kLift), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_new);
        m_ref = m_new;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
    };
    const auto probabilities = [&]() {
        float sum;
        for (int turn = 0;; ++turn) {
            // (no reference yet: hidden scores, minus infinity, are zeros; any other one is infinity here, so that the reference follows it)
            const float m_scaled = m_ref == -INFINITY ? -FLT_MAX : m_ref;
            const X2 ones = {(E)1.f, (E)1.f};
            float psum[2] = {0.f, 0.f};  // the sum of what the product will see, in 32 bits
            X2 pp[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float lo = __builtin_amdgcn_exp2f(sacc[x >> 3][2 * x & 15] * b.scale_log2 - m_scaled);
                const float hi = __builtin_amdgcn_exp2f(sacc[x >> 3][(2 * x & 15) + 1] * b.scale_log2 - m_scaled);
                pp[x] = X2{(E)lo, (E)hi};
                psum[x & 1] = Elem<E>::dot2_acc(pp[x], ones, psum[x & 1]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                struct Four {
                    X2 v[4];
                };
                pb[j] = __builtin_bit_cast(X8, Four{{pp[4 * j], pp[4 * j + 1], pp[4 * j + 2], pp[4 * j + 3]}});
            }
            sum = psum[0] + psum[1];
            if (turn > 0 || !__any(sum > Range<E>::kMostSum)) break;
            refer();
        }
        l_run += sum;
    };
    // sacc[kb][r] is the score of key c0 + 32 kb + 8 (r / 4) + 4 hf + r % 4 for the row of qcol.
    const auto hide = [&](int i) {
        const int seen = pos - (w.begin + i) * kTileKeys - 4 * hf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) sacc[kb][r] = kb * 32 + 8 * (r >> 2) + (r & 3) <= seen ? sacc[kb][r] : -INFINITY;
    };

    const int plain = wave_ok ? min(n - 1, (w.p0 + w.tile * kTileRows / b.group + 1) / kTileKeys - w.begin) : 0;
    if (wave_ok) {
        scores_of(0);
        if (plain <= 0) hide(0);
        refer();
    }
    // V(i + 1) and K(i + 2) are requested behind the meeting ahead of tile i's products, in place of V(i - 1) and K(i)
    const auto next = [&](int i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        meet();
        if (i + 1 < n) request_v(i + 1, (i + 1) % kStages);
        if (i + 2 < n) request_k(i + 2, i % kStages);
    };
    int i = 0;
    for (; i < plain; ++i) {
        const uint32_t v_now = v_of(i), k_next = k_of(i + 1);
        probabilities();
        next(i);
        __builtin_amdgcn_s_setprio(1);  // (the other workgroup's vector instructions would delay the products, 1 % in all)
        X8 vf[8], vg[8], kf[8], kg[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) vf[x] = read_v(v_now, x);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            oacc[x & 3] = Elem<E>::mfma_32x32x16(vf[x], pb[x >> 2], oacc[x & 3]);
            vg[x] = read_v(v_now, x + 8);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            oacc[x & 3] = Elem<E>::mfma_32x32x16(vg[x], pb[2 + (x >> 2)], oacc[x & 3]);
            kf[x] = read_k(k_next, x);
        }
        clear_scores();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            sacc[x & 1] = Elem<E>::mfma_32x32x16(kf[x], qreg[x >> 1], sacc[x & 1]);
            kg[x] = read_k(k_next, x + 8);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) sacc[x & 1] = Elem<E>::mfma_32x32x16(kg[x], qreg[4 + (x >> 1)], sacc[x & 1]);
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int x = 0; x < 24; ++x) {  // a product, a read
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
    }
    for (; i < n; ++i) {
        const int c0 = (w.begin + i) * kTileKeys;
        const bool active = wave_ok && c0 <= wave_last;
        if (active) {
            hide(i);
            probabilities();
        }
        next(i);
        if (active) {
            // A tile that not all rows see whole: a value that some row may not see must not reach its sum, not even as 0 times infinity.  (Behind the last row's
            // position lies what the page held before.)  0 times all of the values is 0 if they are finite; few tiles have others.
            int from = (i % kStages) * kStageBytes;
            uint32_t odd = 0;  // of this lane's keys, those that have such values: bit 8 j + e is key 16 j + 4 hf + e % 4 + 8 (e / 4)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                asm volatile("" : "+v"(from));  // (nothing is worked out ahead of the loop for this)
                X8 vf[8];
                float none[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < 8; ++x) vf[x] = read_v(v_base + from, 4 * j + x);
#pragma unroll
                for (int x = 0; x < 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) none[e] = Elem<E>::dot2_acc(X2{vf[x][2 * e], vf[x][2 * e + 1]}, X2{(E)0.f, (E)0.f}, none[e]);
                if (__any(none[0] + none[1] + none[2] + none[3] != 0.f)) {  // zeros for the product
#pragma unroll
                    for (int x = 0; x < 8; ++x)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (not_finite(vf[x][e])) {
                                odd |= 1u << (8 * (j + (x >> 2)) + e);
                                vf[x][e] = (E)0.f;
                            }
                }
#pragma unroll
                for (int x = 0; x < 8; ++x) oacc[x & 3] = Elem<E>::mfma_32x32x16(vf[x], pb[j + (x >> 2)], oacc[x & 3]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (__any(odd != 0)) {
                // What rows do see of such values is added by itself, one by one.
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) odd |= __shfl_xor((int)odd, d);
                for (int half = 0; half < 2; ++half) {
                    for (uint32_t rest = __builtin_amdgcn_readlane(odd, 32 * half); rest; rest &= rest - 1) {
                        const int bit = __builtin_ctz(rest), key = 16 * (bit >> 3) + 4 * half + (bit & 3) + 8 * (bit >> 2 & 1);
                        float pk = 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < 8; ++e) pk = 8 * j + e == bit ? (float)pb[j][e] : pk;
                        pk = __shfl(pk, (lane & 31) + 32 * half);
                        const bool sees = c0 + key <= pos;
                        const int slot = v_slot16(key);
                        int at = from + kKBytes + (slot & 7) * 2, rows = 4 * (lane >> 5);
#pragma unroll
                        for (int db = 0; db < 4; ++db)
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                asm volatile("" : "+v"(at), "+v"(rows));  // (64 addresses worked out ahead would take the loop's registers)
                                const int d = db * 32 + 8 * (r >> 2) + (r & 3) + rows;
                                const E v = *reinterpret_cast<const E*>(ring + at + d * 128 + (((slot >> 3) ^ ((d >> 1) & 7)) << 4));
                                if (sees && not_finite(v)) oacc[db][r] += pk * (float)v;
                            }
                    }
                }
            }
        }
        if (wave_ok && i + 1 < n) scores_of(i + 1);
    }
    if (!wave_ok) return;

    // oacc[db][r] is dim 32 db + 8 (r / 4) + 4 hf + r % 4 of the row of qcol
    const float l_all = l_run + __shfl_xor(l_run, 32);
    if (w.slot >= 0) {
        const size_t part = (size_t)w.slot * b.Hkv + g;
        float4* const to = p.parts + (part * kWaves + wave) * 16 * 64;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int rq = 0; rq < 4; ++rq)
                to[(db * 4 + rq) * 64 + lane] = make_float4(oacc[db][rq * 4], oacc[db][rq * 4 + 1], oacc[db][rq * 4 + 2], oacc[db][rq * 4 + 3]);
        if (hf == 0) p.stats[part * kTileRows + wave * kWaveRows + qcol] = make_float2(m_ref, l_all);
        return;
    }
    // Through LDS, so that memory gets whole rows: the wave's 32 rows take the place of a quarter of the stages' K, which everybody has read.
    const float inv = 1.f / l_all;
    char* const o_stage = ring + (wave >> 1) * kStageBytes + (wave & 1) * (kWaveRows * 256);
    static_assert(kWaves == 4 && kStages == 2 && kWaveRows * 256 * 2 == kKBytes, "two waves' rows in a stage's K");
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            X4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (E)(oacc[db][rq * 4 + e] * inv);
            *reinterpret_cast<X4*>(o_stage + k_at(qcol, db * 4 + rq) + hf * 8) = o;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    int at = lane;
    asm volatile("" : "+v"(at));  // (the rows' places of the beginning, kept, would take the loop's registers)
    Rows o_row = first_row(base_row + (at >> 4), b.out_stride);
#pragma unroll
    for (int x = 0; x < kWaveRows / 4; ++x) {
        const int r = x * 4 + (at >> 4);
        if (base_row + r < packed) *reinterpret_cast<X8*>(b.out + o_row.at + (at & 15) * 8) = *reinterpret_cast<const X8*>(o_stage + k_at(r, at & 15));
        next_row(o_row, b.out_stride);
    }
}

// The pieces of a tile: with M the largest of their references m, sum = sum_i l_i 2^(m_i - M), out = sum_i O_i 2^(m_i - M) / sum, in their order.  A workgroup takes 32 of
// the rows at a time, a wave 32 of their dims.
constexpr int kJoinWaves = kHeadDim / 32, kJoinGrid = 2048, kJoinAtOnce = 4;
template <typename E>
__global__ __launch_bounds__(64 * kJoinWaves) void prompt_join_kernel(PromptParams p) {
    typedef typename Elem<E>::x4 X4;
    const BatchRows& b = p.b;
    const int lane = threadIdx.x & 63, db = threadIdx.x >> 6, qcol = lane & 31, hf = lane >> 5;
    const int all = p.plan.listed->joins * b.Hkv * kWaves;
    for (int x = blockIdx.x; x < all; x += gridDim.x) {
        const int block = x % kWaves, g = x / kWaves % b.Hkv;
        const Join j = p.plan.joins[x / kWaves / b.Hkv];
        const int base_row = j.tile * kTileRows + block * kWaveRows, R = base_row + qcol;
        if (base_row >= j.rows * b.group) continue;
        float M = -INFINITY, L = 0.f;
        f32x4 sum[4];
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) sum[rq] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < j.pieces; i0 += kJoinAtOnce) {
            float2 st[kJoinAtOnce];
            f32x4 o[kJoinAtOnce][4];
#pragma unroll
            for (int u = 0; u < kJoinAtOnce; ++u) {
                st[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int rq = 0; rq < 4; ++rq) o[u][rq] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (i0 + u >= j.pieces) continue;
                const size_t part = (size_t)(j.slot + i0 + u) * b.Hkv + g;
                st[u] = p.stats[part * kTileRows + block * kWaveRows + qcol];
                const float4* const from = p.parts + ((part * kWaves + block) * 16 + db * 4) * 64 + lane;
#pragma unroll
                for (int rq = 0; rq < 4; ++rq) o[u][rq] = __builtin_bit_cast(f32x4, from[rq * 64]);
            }
            float m = M;
#pragma unroll
            for (int u = 0; u < kJoinAtOnce; ++u) m = fmaxf(m, st[u].x);
            const float m_scaled = m == -INFINITY ? 0.f : m, f = __builtin_amdgcn_exp2f(M - m_scaled);
            M = m;
            L *= f;
#pragma unroll
            for (int rq = 0; rq < 4; ++rq)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[rq][e] *= f;
#pragma unroll
            for (int u = 0; u < kJoinAtOnce; ++u) {
                // (a piece that the row sees nothing of has zeros)
                const float w = __builtin_amdgcn_exp2f(st[u].x - m_scaled);
                L = __builtin_fmaf(st[u].y, w, L);
#pragma unroll
                for (int rq = 0; rq < 4; ++rq)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[rq][e] = __builtin_fmaf(o[u][rq][e], w, sum[rq][e]);
            }
        }
        if (R >= j.rows * b.group) continue;
        const Quotient row = divide(R, b.group, b.group_inverse);
        const float inv = 1.f / L;
        E* const to = reinterpret_cast<E*>(b.out) + (int64_t)(j.row0 + row.q) * b.out_stride + (g * b.group + row.r) * kHeadDim + db * 32 + hf * 4;
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            X4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (E)(sum[rq][e] * inv);
            *reinterpret_cast<X4*>(to + rq * 8) = o;
        }
    }
}

// ---- sizes ----

struct Sizes {
    int64_t tiles, slots, works, joins;
    size_t works_at, joins_at, stats_at, parts_at, bytes;
};
Sizes sizes_of(int num_requests, int max_blocks, int n, int Hq, int Hkv) {
    Sizes s;
    // every request's last tile may be a part of one
    s.tiles = ((int64_t)n * (Hq / Hkv)) / kTileRows + std::min(num_requests, n);
    const int64_t keys = (int64_t)max_blocks * (kPage / kTileKeys), least = least_of(s.tiles, Hkv);
    s.slots = keys <= least ? 0 : std::min<int64_t>(2 * ((kParts + Hkv - 1) / Hkv), s.tiles * ((keys + least - 1) / least));
    s.joins = std::min(s.tiles, s.slots / 2);
    s.works = s.tiles + s.slots;
    s.works_at = sizeof(Listed);
    s.joins_at = s.works_at + sizeof(Work) * (s.works + 1);
    s.stats_at = align_up(s.joins_at + sizeof(Join) * (s.joins + 1), 256);
    s.parts_at = s.stats_at + sizeof(float2) * kTileRows * s.slots * Hkv;
    s.bytes = s.parts_at + sizeof(float) * kTileRows * kHeadDim * s.slots * Hkv;
    return s;
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" size_t cpmcu_batch_prompt_attention_workspace_bytes(int num_requests, int max_blocks, int n, int Hq, int Hkv) {
    if (num_requests < 1 || num_requests > kMostRequests || max_blocks < 1 || max_blocks > kMostBlocks || n < 0 || n >= 1 << 24 || Hkv < 1 || Hq < 1 || Hq > 1024 || Hq % Hkv) return 0;
    return sizes_of(num_requests, max_blocks, n, Hq, Hkv).bytes;
}

extern "C" int cpmcu_batch_prompt_attention(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, int num_pages, const int32_t* block_tables,
                                      int64_t table_stride, int max_blocks, const int32_t* row_offsets, const int32_t* positions, int num_requests, int n, int Hq, int Hkv,
                                      float scale, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    BatchRows b{(const uint16_t*)q, (uint16_t*)out, q_stride, out_stride, (const uint16_t*)k_pool, (const uint16_t*)v_pool, block_tables, row_offsets, positions,
                table_stride, num_requests, max_blocks, num_pages, n, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, 0, scale * 1.44269504088896341f};
    const int rc = check_batch_rows("prompt_attention", b, scale);
    if (rc != CPMCU_OK) return rc;
    if (n == 0) return CPMCU_OK;
    b.group_inverse = 0xffffffffu / (uint32_t)b.group;
    CPMCU_CHECK_ARG(row_offsets, "prompt_attention: null pointer argument");
    const Sizes s = sizes_of(num_requests, max_blocks, n, Hq, Hkv);
    CPMCU_CHECK_ARG(workspace && workspace_bytes >= s.bytes, "prompt_attention: workspace of %zu bytes, %zu needed", workspace_bytes, s.bytes);
    CPMCU_CHECK_ARG((uintptr_t)workspace % 16 == 0, "prompt_attention: the workspace has to lie on 16 bytes");
    const int64_t grid = s.works * Hkv;
    CPMCU_CHECK_ARG(grid * kThreads <= UINT32_MAX, "prompt_attention: %lld workgroups of %d threads are beyond a launch", (long long)grid, kThreads);
    char* const ws = static_cast<char*>(workspace);
    PlanParams plan{row_offsets, positions, num_requests, max_blocks, n, b.group, Hkv, (int)s.tiles, (int)s.slots, (Listed*)ws, (Work*)(ws + s.works_at), (Join*)(ws + s.joins_at)};
    PromptParams p{b, plan, (float4*)(ws + s.parts_at), (float2*)(ws + s.stats_at)};
    const hipStream_t st = resolve_stream(stream);
    const bool bf = options().dtype == 1;
    const bool listed = num_requests > kOwnThreads || s.tiles > kOwnThreads || s.tiles * Hkv > kOwnGrid || grid > 2 * kOwnGrid;
    if (listed) {
        if (num_requests <= 256 && s.tiles <= 512) hipLaunchKernelGGL((prompt_plan_kernel<256, 1>), dim3(1), dim3(256), 0, st, plan);
        else if (num_requests <= 1024) hipLaunchKernelGGL((prompt_plan_kernel<1024, 1>), dim3(1), dim3(1024), 0, st, plan);
        else hipLaunchKernelGGL((prompt_plan_kernel<1024, kMostRequests / 1024>), dim3(1), dim3(1024), 0, st, plan);
        CPMCU_LAUNCH_CHECK();
    }
    void (*kernel)(PromptParams) = bf ? prompt_attention_kernel<bf16, false> : prompt_attention_kernel<f16, false>;
    if (listed) kernel = bf ? prompt_attention_kernel<bf16, true> : prompt_attention_kernel<f16, true>;
    hipLaunchKernelGGL(kernel, dim3((int)grid), dim3(kThreads), 0, st, p);
    CPMCU_LAUNCH_CHECK();
    if (s.joins > 0) {
        hipLaunchKernelGGL(bf ? prompt_join_kernel<bf16> : prompt_join_kernel<f16>, dim3((int)std::min<int64_t>(s.joins * Hkv * kWaves, kJoinGrid)), dim3(64 * kJoinWaves), 0, st, p);
        CPMCU_LAUNCH_CHECK();
    }
    return CPMCU_OK;
}
