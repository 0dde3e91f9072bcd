// Attention of one new row of each request over its pages: a step of decoding for a batch.
//
//   out[t][h] = sum_x p_x v[x] / sum_x p_x,  p_x = exp(scale (q[t][h] . k[x] - max)),  x from 0 to the row's own position.
//
// Every key and value is read once and meets the heads on its KV head only, so the launch is bound by memory: 512 bytes a key and KV head.
// What decides its speed is that all of the card reads all of the time, whatever the requests' lengths are.  The tiles of 64 keys of all
// requests and KV heads are therefore one line, which the workgroups cut into equal parts, found on the device from the positions:
// a workgroup may end one request's keys, take others whole and begin the next one's.  What is not whole is left as sums that a
// second launch joins.
//
// A wave takes tiles of its own through LDS of its own, K and V in whole lines: straight into registers, as the matrix instructions want them, every
// instruction takes parts of 16 rows, at which a CU gets 45 GB/s -- enough where all CUs read (20 GB/s each), but 5 of the 10 us of a short context on two of them.
// No two waves read a tile, so nothing but the end of a request's keys makes them wait for each other.  S^T = K Q^T has the heads as its columns, in 16s; its
// results are the second operand of O^T = V^T P^T as they lie, with the order of tokens that the pages' V has.
#include "batch_attention.h"

#include <algorithm>

namespace cpmcu {
namespace {

constexpr int kHeads = 16;       // columns of the products: heads that a workgroup has at a time
constexpr int kWaves = 2;        // of a workgroup that has a part of the line: 64 KB of tiles, two a CU
constexpr int kGrid = 512;       // workgroups that share the line
// Where requests are short in the mean, a part of the line is a wave's; else it is a workgroup's, whose waves take a request's tiles in turn and meet in LDS (a tile a wave
// spares that, and leaves more for the second launch: 100 requests of up to 2000 on 8 heads 103 us, with parts of workgroups 118; one of 131000 55 more).
constexpr int kAloneMean = 16;  // tiles of a request
// Where no request has more tiles than this, and there are as many tiles as workgroups, a workgroup takes all of a request's on a KV head: no line, nothing to join.  Where the tables have no room
// for more it does so anyway, in one launch.  (200 requests of up to 900: 20 us in narrow tables, 25 in wide ones, 29 cut in parts; one of 500: 6, and in wide tables 12 whole, 10 in parts.)
constexpr int kWholeTiles = 16, kWideGrid = 256;
constexpr int kPartFloats = kHeads * kHeadDim;
constexpr int kKBytes = kTileKeys * kHeadDim * 2, kStageBytes = 2 * kKBytes;  // of a wave: a tile's K, then its V
// The second launch: a workgroup joins up to kFewParts parts of a unit, eight of them more (with 32 one request of 3000 takes 15.1 us instead of 13.6); a wave requests kAtOnce of them together.
constexpr int kJoinWaves = 16, kFewParts = 16, kAtOnce = 8;
// Probabilities are powers of two of a score less a reference, kLift below the largest: up to 4096 in fp16, which ends at 65504 and has fewer bits below 2^-14, so that a probability keeps all of its bits
// down to e^-18 of the largest (without, to e^-9.7: behind one key that has e^16.5 times the weight of each other, the others' sum was 2 % off).  bf16 has the range of 32 bits.
template <typename E>
constexpr float kLift = Elem<E>::kDtype == 0 ? 12.f : 0.f;
constexpr int kFewRequests = 1024;  // up to which the line's ends leave room for two workgroups a CU
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Line {
    int parts;  // that are cut
    int pad[3];
};
// A unit -- a request's keys for 16 heads on a KV head -- and the parts that have some of it.
struct Unit {
    int request, unit, from, to;
};

struct DecodeParams {
    BatchRows b;
    int units;  // of a request: KV heads times 16s of their heads
    int blocks; // 16s of the heads on a KV head
    Line* line;
    int* tiles;     // [requests]
    Unit* cut;      // [requests][units], where there are tiles
    Unit* owners;   // [parts]: whose tile each begins with
    float2* stats;  // [2 parts][16]: (reference in powers of two, sum)
    float4* sums;   // [2 parts][8 blocks of 16 dims][64 lanes]
};

// Quotients of whole numbers a < 2^53 (here 2^49 at most: 2^30 tiles on 2^10 units, 2^9 times) in 64-bit floats: one that is not whole is 1 / b or more below the next whole
// number, and its rounding moves it by at most a / b 2^-53, which is less.  (A division of 64-bit whole numbers is several times as long.)
__device__ inline int64_t quotient(int64_t a, int64_t b) { return (int64_t)((double)a / (double)b); }
// Part i of `parts` of `all` tiles begins here, and the part that has tile x.
__device__ inline int64_t part_begin(int64_t all, int parts, int i) { return quotient(all * i, parts); }
__device__ inline int part_of(int64_t all, int parts, int64_t x) { return (int)quotient((x + 1) * parts - 1, all); }

// A request's row and how many tiles of keys it sees; no tiles where it has no row to attend.
__device__ inline int tiles_of(const BatchRows& b, int r, int& row, int& pos) {
    row = r;
    pos = -1;
    if (b.row_offsets) {
        const int lo = b.row_offsets[r], hi = b.row_offsets[r + 1];
        row = lo;
        if (hi - lo != 1) return 0;
    }
    if ((unsigned)row >= (unsigned)b.n) return 0;
    pos = b.positions[row];
    if (pos < 0 || pos >= (int64_t)b.max_blocks * kPage) return 0;
    return pos / kTileKeys + 1;
}

// MOST: requests that the line may have (0: no line, a workgroup has a request's keys on a KV head).
template <typename E, int MOST, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void decode_attention_kernel(DecodeParams p) {
    constexpr bool WHOLE = MOST == 0;
    constexpr int kThreads = 64 * WAVES;
    typedef typename Elem<E>::x8 X8;
    typedef typename Elem<E>::x4 X4;
    __shared__ __attribute__((aligned(1024))) char stages[WAVES * kStageBytes];
    __shared__ int tile_end[WHOLE ? 1 : MOST];
    __shared__ int wave_total[WAVES];
    __shared__ float2 s_stat[WAVES][kHeads];
    const BatchRows& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int B = b.num_requests, col = lane & 15, lg = lane >> 4;
    char* const stage = stages + wave * kStageBytes;
    const uint32_t stage_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)stage);

    bool alone = false, all_whole = WHOLE;
    int parts = 0, part = 0;
    int64_t all = 0, at = WHOLE ? 0 : blockIdx.x, end = WHOLE ? 1 : (int64_t)B * p.units;
    if constexpr (!WHOLE) {
        // The line: each thread has a run of requests; their running totals.
        const int each = (B + kThreads - 1) / kThreads;
        int mine = 0, most = 0;
        for (int e = 0; e < each; ++e) {
            const int r = tid * each + e;
            int row, pos;
            const int tiles = r < B ? tiles_of(b, r, row, pos) : 0;
            mine += tiles;
            most = max(most, tiles);
            if (r < B) tile_end[r] = mine;
        }
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int from = __shfl_up(upto, d);
            if (lane >= d) upto += from;
        }
        if (lane == 63) wave_total[wave] = upto;
        all_whole = !__syncthreads_or(most > kWholeTiles);
        int before = upto - mine, total = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += wave_total[w];
            total += wave_total[w];
        }
        for (int e = 0; e < each; ++e) {
            const int r = tid * each + e;
            if (r < B) tile_end[r] += before;
        }
        __syncthreads();
        all = (int64_t)total * p.units;
        all_whole = all_whole && all >= gridDim.x;
        alone = !all_whole && total <= kAloneMean * B;
        parts = all_whole ? 0 : (int)min(alone ? (int64_t)WAVES * gridDim.x : (int64_t)gridDim.x, alone ? all : (all + WAVES - 1) / WAVES);
        if (blockIdx.x == 0) {
            if (tid == 0) *p.line = Line{parts, {0, 0, 0}};
            for (int r = tid; r < B; r += kThreads) p.tiles[r] = all_whole ? 0 : tile_end[r] - (r > 0 ? tile_end[r - 1] : 0);
        }
        if (!all_whole) {
            part = alone ? wave * gridDim.x + blockIdx.x : blockIdx.x;
            if (part >= parts) return;  // (whole workgroups where they share a part)
            at = part_begin(all, parts, part);
            end = part_begin(all, parts, part + 1);
        }
    }
    const int first_wave = alone ? 0 : wave, step = alone ? 1 : WAVES;
    for (bool begins = true; at < end; begins = false) {
        int r, unit, tiles, t0, t1, row, pos;
        if (all_whole) {
            const int x = WHOLE ? blockIdx.x : (int)at;
            r = x / p.units;
            unit = x % p.units;
            tiles = tiles_of(b, r, row, pos);
            if (tiles == 0) {
                if (WHOLE) return;
                at += gridDim.x;
                continue;
            }
            t0 = 0;
            t1 = tiles;
        } else {
            // the request: the first whose end, on all of its KV heads, lies behind
            int lo = 0, hi = B - 1;
            const int x = (int)quotient(at, p.units);
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (tile_end[mid] > x) hi = mid;
                else lo = mid + 1;
            }
            r = __builtin_amdgcn_readfirstlane(lo);
            const int start = __builtin_amdgcn_readfirstlane(r > 0 ? tile_end[r - 1] : 0);
            tiles = __builtin_amdgcn_readfirstlane(tile_end[r]) - start;
            const int64_t inside = at - (int64_t)start * p.units;
            unit = __builtin_amdgcn_readfirstlane((int)quotient(inside, tiles));
            t0 = __builtin_amdgcn_readfirstlane((int)(inside - (int64_t)unit * tiles));
            t1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)tiles, t0 + (end - at)));
            if (begins || t0 == 0) {  // (a workgroup's waves write the same)
                const int64_t first = (int64_t)start * p.units + (int64_t)unit * tiles;
                const Unit u{r, unit, part_of(all, parts, first), part_of(all, parts, first + tiles - 1)};
                if (begins && lane == 0) p.owners[part] = u;
                if (t0 == 0 && lane == 0) p.cut[r * p.units + unit] = u;
            }
            tiles_of(b, r, row, pos);
        }
        const int g = unit / p.blocks, h0 = unit % p.blocks * kHeads;  // of the heads on g
        const bool has = h0 + col < b.group;
        const int head = g * b.group + min(h0 + col, b.group - 1);

        // page numbers, 64 at a time, one a lane
        const int32_t* const table = b.block_tables + (size_t)r * b.table_stride;
        int pages_from = t0 * kTileKeys / kPage, pages = table[min(pages_from + lane, b.max_blocks - 1)];
        X8 q[4];  // second operand of S^T = K Q^T: lane (col, lg) has dims 32 kk + 8 lg + [0, 8) of its head
        {
            const E* const from = reinterpret_cast<const E*>(b.q) + (int64_t)row * b.q_stride + head * kHeadDim + 8 * lg;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) q[kk] = *reinterpret_cast<const X8*>(from + 32 * kk);
        }
        const auto place_of = [&](int t) {  // of a tile's first key: (page and KV head, place in the page)
            const int block = t * kTileKeys / kPage;
            if (block - pages_from >= 64) {
                pages_from = block;
                pages = table[min(block + lane, b.max_blocks - 1)];
            }
            return (size_t)page_within(__builtin_amdgcn_readlane(pages, block - pages_from), b.num_pages) * b.Hkv + g;
        };
        // In LDS: K a row of 256 bytes a key, its 16-byte pieces exchanged by the key's number; V a row of 128 bytes a dim, by half of the dim's.
        const uint32_t k_off = (lane >> 4) * 256 + ((lane & 15) ^ (lane >> 4)) * 16, v_off = (lane >> 3) * 512 + ((lane & 7) ^ (lane >> 4)) * 16;
        const auto request_k = [&](size_t page, int t) {
            const char* const from = reinterpret_cast<const char*>(b.k_pool + (page * kPage + t * kTileKeys % kPage) * kHeadDim);
#pragma unroll
            for (int i = 0; i < 4; ++i) request_4k(from + i * 4096, k_off, k_off ^ 64u, k_off ^ 128u, k_off ^ 192u, stage_at + i * 4096);
        };
        const auto request_v = [&](size_t page, int t) {
            const char* const from = reinterpret_cast<const char*>(b.v_pool + page * kHeadDim * kPage + t * kTileKeys % kPage);
#pragma unroll
            for (int i = 0; i < 4; ++i) request_4k(from + i * 16384, v_off, (v_off ^ 64u) + 3u * 1024u, v_off + 6u * 1024u, (v_off ^ 64u) + 9u * 1024u, stage_at + kKBytes + i * 4096);
        };
        f32x4 o[8];
#pragma unroll
        for (int db = 0; db < 8; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_ref = -INFINITY, l_run = 0.f;
        int t = t0 + first_wave;
        size_t page = 0;
        if (t < t1) {
            page = place_of(t);
            request_k(page, t);
            request_v(page, t);
        }
        // Row m of a product's 16 is key 32 sp + 16 (m / 8) + 4 (m / 4 % 2) + m % 4, + 8 in the second of a pair: the results of the two, four and four, are
        // then the eight tokens of a lane's piece of V.
        const int key = 16 * (col >> 3) + 4 * (col >> 2 & 1) + (col & 3);
        // While a tile's scores become probabilities the next one's keys are on their way, and its values while the scores are made.  (The first wait is for everything:
        // results of the segment before may be on their way too.)
        for (bool fresh = true; t < t1; t += step, fresh = false) {
            const int c0 = t * kTileKeys;
            if (fresh) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
            f32x4 s[2][2];
            {
                X8 k[2][2][4];
#pragma unroll
                for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                    for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const int row_of = 32 * sp + 8 * ab + key;
                            k[sp][ab][kk] = *reinterpret_cast<const X8*>(stage + row_of * 256 + (((4 * kk + lg) ^ (row_of & 15)) << 4));
                        }
#pragma unroll
                for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                    for (int ab = 0; ab < 2; ++ab) {
                        s[sp][ab] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) s[sp][ab] = Elem<E>::mfma_16x16x32(k[sp][ab][kk], q[kk], s[sp][ab]);
                    }
            }
            const bool more = t + step < t1;
            if (more) {
                page = place_of(t + step);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (K has been read)
                request_k(page, t + step);
                asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            X8 v[2][8];
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int db = 0; db < 8; ++db)
                    v[sp][db] = *reinterpret_cast<const X8*>(stage + kKBytes + (16 * db + col) * 128 + (((4 * sp + lg) ^ (col >> 1)) << 4));
            // lane (col, lg) has the scores of keys c0 + 32 sp + 16 (lg / 2) + 4 (lg % 2) + 8 ab + i
            if (c0 + kTileKeys - 1 > pos) {
                // behind the row's position lies what the page held before: no score, and no value, not even as 0 times infinity
                const int seen = pos - c0 - 16 * (lg >> 1) - 4 * (lg & 1);
#pragma unroll
                for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                    for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const int at = 32 * sp + 8 * ab + i;
                            const uint32_t keep = (at <= seen ? 0xffffu : 0u) | (at < seen ? 0xffff0000u : 0u);
                            s[sp][ab][i] = at <= seen ? s[sp][ab][i] : -INFINITY;
                            s[sp][ab][i + 1] = at < seen ? s[sp][ab][i + 1] : -INFINITY;
#pragma unroll
                            for (int db = 0; db < 8; ++db) {
                                u32x4 w = __builtin_bit_cast(u32x4, v[sp][db]);
                                w[2 * ab + i / 2] &= keep;
                                v[sp][db] = __builtin_bit_cast(X8, w);
                            }
                        }
            }
            float tmax = -INFINITY;
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, s[sp][ab][i]);
            tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32)) * b.scale_log2 - kLift<E>;
            const float m_new = fmaxf(m_ref, tmax);
            const float m_scaled = m_new == -INFINITY ? 0.f : m_new, alpha = __builtin_amdgcn_exp2f(m_ref - m_scaled);
            m_ref = m_new;
            l_run *= alpha;
            X8 pb[2];  // rounded to the element type; the sum is that of what the product will see
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pb[sp][4 * ab + i] = (E)__builtin_amdgcn_exp2f(s[sp][ab][i] * b.scale_log2 - m_scaled);
                        l_run += (float)pb[sp][4 * ab + i];
                    }
#pragma unroll
            for (int db = 0; db < 8; ++db) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[db][i] *= alpha;
#pragma unroll
                for (int sp = 0; sp < 2; ++sp) o[db] = Elem<E>::mfma_16x16x32(v[sp][db], pb[sp], o[db]);
            }
            if (more) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (V has been read)
                request_v(page, t + step);
            }
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
        // o[db][i] is dim 16 db + 4 lg + i of head col
        const bool whole = all_whole || (t0 == 0 && t1 == tiles);
        const int slot = 2 * part + (t0 == 0 ? 1 : 0);  // of a part that begins a unit's keys and of one that goes on with them
        const auto put = [&](int db, const f32x4& sum, float inv) {
            if (!whole) {
                p.sums[((size_t)slot * 8 + db) * 64 + lane] = __builtin_bit_cast(float4, sum);
            } else if (has) {
                X4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (E)(sum[i] * inv);
                *reinterpret_cast<X4*>(reinterpret_cast<E*>(b.out) + (int64_t)row * b.out_stride + head * kHeadDim + 16 * db + 4 * lg) = y;
            }
        };
        if (alone) {
            const float inv = 1.f / l_run;
#pragma unroll
            for (int db = 0; db < 8; ++db) put(db, o[db], inv);
            if (!whole && lg == 0) p.stats[slot * kHeads + col] = make_float2(m_ref, l_run);
        } else {
            // the waves' sums meet in LDS, each in place of its tiles; a share of the dims a wave
            float* const mine = reinterpret_cast<float*>(stage);
#pragma unroll
            for (int db = 0; db < 8; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[(db * 4 + i) * 64 + lane] = o[db][i];
            if (lg == 0) s_stat[wave][col] = make_float2(m_ref, l_run);
            __syncthreads();
            float M = -INFINITY, L = 0.f, f[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) M = fmaxf(M, s_stat[w][col].x);
            const float m_scaled = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                f[w] = __builtin_amdgcn_exp2f(s_stat[w][col].x - m_scaled);
                L = __builtin_fmaf(s_stat[w][col].y, f[w], L);
            }
            const float inv = 1.f / L;
#pragma unroll
            for (int d = 0; d < 8 / WAVES; ++d) {
                const int db = 8 / WAVES * wave + d;
                f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WAVES; ++w)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(reinterpret_cast<const float*>(stages + w * kStageBytes)[(db * 4 + i) * 64 + lane], f[w], sum[i]);
                put(db, sum, inv);
            }
            if (!whole && wave == 0 && lg == 0) p.stats[slot * kHeads + col] = make_float2(M, L);
            if (!WHOLE) __syncthreads();  // (the next segment's tiles may come)
        }
        at += WHOLE ? 1 : all_whole ? (int)gridDim.x : t1 - t0;
    }
}

// The parts of a unit: M the largest reference, sum_i l_i 2^(m_i - M), out = sum_i O_i 2^(m_i - M) over it.  A wave a block of 16 dims and every second of the
// parts; where there are many, every 16th.
template <typename E>
__global__ __launch_bounds__(64 * kJoinWaves, 8) void decode_join_kernel(DecodeParams p, int few) {
    typedef typename Elem<E>::x4 X4;
    __shared__ f32x4 s_sum[kJoinWaves][64];
    __shared__ float2 s_stat[kJoinWaves][kHeads];
    const BatchRows& b = p.b;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, lg = lane >> 4;
    // The first `few` workgroups have a unit each.  Behind them, eight for every kFewParts-th part: a unit of more has such a part, and the first one that begins
    // with its tiles counts.
    const bool many = (int)blockIdx.x >= few;
    const int mark = many ? ((int)blockIdx.x - few) / 8 * kFewParts : 0, request = many ? 0 : (int)blockIdx.x / p.units;
    const Unit u = many ? p.owners[mark] : p.cut[blockIdx.x];
    if (many ? mark >= p.line->parts : p.tiles[request] == 0) return;  // (what there is not has not been written)
    if (many) {
        // the first mark is the unit's first part only if that begins with it
        const Unit at_from = u.from % kFewParts == 0 ? p.owners[u.from] : Unit{-1, -1, 0, 0};
        const int first = at_from.request == u.request && at_from.unit == u.unit ? u.from : (u.from / kFewParts + 1) * kFewParts;
        if (u.to - u.from < kFewParts || mark != first) return;
    } else if (u.from == u.to || u.to - u.from >= kFewParts) {
        return;
    }
    const int row = b.row_offsets ? b.row_offsets[u.request] : u.request;
    const int groups = many ? kJoinWaves : kJoinWaves / 8, group = many ? wave : wave >> 3, db = many ? ((int)blockIdx.x - few) & 7 : wave & 7;
    float M = -INFINITY, L = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = u.from + group; i0 <= u.to; i0 += groups * kAtOnce) {
        float2 st[kAtOnce];
        f32x4 o[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int i = i0 + x * groups, slot = 2 * i + (i == u.from ? 1 : 0);
            st[x] = make_float2(-INFINITY, 0.f);
            o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i <= u.to) {
                st[x] = p.stats[slot * kHeads + col];
                o[x] = __builtin_bit_cast(f32x4, p.sums[((size_t)slot * 8 + db) * 64 + lane]);
            }
        }
        float m = M;
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) m = fmaxf(m, st[x].x);
        const float m_scaled = m == -INFINITY ? 0.f : m, f = __builtin_amdgcn_exp2f(M - m_scaled);
        M = m;
        L *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] *= f;
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const float w = __builtin_amdgcn_exp2f(st[x].x - m_scaled);
            L = __builtin_fmaf(st[x].y, w, L);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[x][i], w, sum[i]);
        }
    }
    s_sum[wave][lane] = sum;
    if (lg == 0) s_stat[wave][col] = make_float2(M, L);
    __syncthreads();
    if (group > 0) return;
    const int stride = many ? 1 : 8;
    M = -INFINITY;
    for (int w = 0; w < groups; ++w) M = fmaxf(M, s_stat[wave + w * stride][col].x);
    const float m_scaled = M == -INFINITY ? 0.f : M;
    L = 0.f;
    sum = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < groups; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_stat[wave + w * stride][col].x - m_scaled);
        L = __builtin_fmaf(s_stat[wave + w * stride][col].y, f, L);
        const f32x4 o = s_sum[wave + w * stride][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[i], f, sum[i]);
    }
    const int g = u.unit / p.blocks, h = u.unit % p.blocks * kHeads + col;
    if (h >= b.group) return;
    const float inv = 1.f / L;
    X4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (E)(sum[i] * inv);
    *reinterpret_cast<X4*>(reinterpret_cast<E*>(b.out) + (int64_t)row * b.out_stride + (g * b.group + h) * kHeadDim + 16 * db + 4 * lg) = y;
}

struct Sizes {
    int grid, parts;
    size_t tiles_at, cut_at, owners_at, stats_at, sums_at, bytes;
};
int units_of(int Hq, int Hkv) { return Hkv * ceil_div(Hq / Hkv, kHeads); }
Sizes sizes_of(int num_requests, int max_blocks, int Hq, int Hkv) {
    Sizes s;
    const int64_t tiles = (int64_t)num_requests * max_blocks * (kPage / kTileKeys) * units_of(Hq, Hkv);
    s.grid = (int)std::min<int64_t>(kGrid, tiles);
    s.parts = (int)std::min<int64_t>((int64_t)s.grid * kWaves, tiles);
    if (max_blocks * (kPage / kTileKeys) <= kWholeTiles) s.parts = 0;  // (nothing is cut: nothing of this is used)
    s.tiles_at = sizeof(Line);
    s.cut_at = align_up(s.tiles_at + sizeof(int) * num_requests, 16);
    s.owners_at = s.cut_at + sizeof(Unit) * num_requests * units_of(Hq, Hkv);
    s.stats_at = align_up(s.owners_at + sizeof(Unit) * s.parts, 256);
    s.sums_at = s.stats_at + sizeof(float2) * kHeads * 2 * s.parts;
    s.bytes = s.sums_at + sizeof(float) * kPartFloats * 2 * s.parts;
    return s;
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" size_t cpmcu_batch_decode_attention_workspace_bytes(int num_requests, int max_blocks, int Hq, int Hkv) {
    if (num_requests < 1 || num_requests > kMostRequests || max_blocks < 1 || max_blocks > kMostBlocks || Hkv < 1 || Hq < 1 || Hq > 1024 || Hq % Hkv) return 0;
    return sizes_of(num_requests, max_blocks, Hq, Hkv).bytes;
}

extern "C" int cpmcu_batch_decode_attention(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, int num_pages, const int32_t* block_tables,
                                      int64_t table_stride, int max_blocks, const int32_t* row_offsets, const int32_t* positions, int num_requests, int n, int Hq, int Hkv,
                                      float scale, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    BatchRows b{(const uint16_t*)q, (uint16_t*)out, q_stride, out_stride, (const uint16_t*)k_pool, (const uint16_t*)v_pool, block_tables, row_offsets, positions,
                table_stride, num_requests, max_blocks, num_pages, n, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, 0, scale * 1.44269504088896341f};
    const int rc = check_batch_rows("decode_attention", b, scale);
    if (rc != CPMCU_OK) return rc;
    if (n == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(row_offsets || n == num_requests, "decode_attention: %d rows of %d requests need row_offsets", n, num_requests);
    const Sizes s = sizes_of(num_requests, max_blocks, Hq, Hkv);
    CPMCU_CHECK_ARG(workspace && workspace_bytes >= s.bytes, "decode_attention: workspace of %zu bytes, %zu needed", workspace_bytes, s.bytes);
    CPMCU_CHECK_ARG((uintptr_t)workspace % 16 == 0, "decode_attention: the workspace has to lie on 16 bytes");
    const int64_t few = (int64_t)num_requests * units_of(Hq, Hkv), many = s.parts > kFewParts ? 8 * ceil_div(s.parts, kFewParts) : 0;
    CPMCU_CHECK_ARG((few + many) * 64 * kJoinWaves <= UINT32_MAX, "decode_attention: %lld workgroups of %d threads are beyond a launch", (long long)(few + many), 64 * kJoinWaves);
    char* const ws = static_cast<char*>(workspace);
    DecodeParams p{b, units_of(Hq, Hkv), ceil_div(b.group, kHeads), (Line*)ws, (int*)(ws + s.tiles_at), (Unit*)(ws + s.cut_at), (Unit*)(ws + s.owners_at), (float2*)(ws + s.stats_at), (float4*)(ws + s.sums_at)};
    const hipStream_t st = resolve_stream(stream);
    const bool bf = options().dtype == 1;
    if (s.parts == 0) {
        // four waves where a CU has one workgroup at most
        const int grid = num_requests * p.units;
        if (grid <= kWideGrid) hipLaunchKernelGGL((bf ? decode_attention_kernel<bf16, 0, 4> : decode_attention_kernel<f16, 0, 4>), dim3(grid), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((bf ? decode_attention_kernel<bf16, 0, 2> : decode_attention_kernel<f16, 0, 2>), dim3(grid), dim3(128), 0, st, p);
        CPMCU_LAUNCH_CHECK();
        return CPMCU_OK;
    }
    if (num_requests <= kFewRequests)
        hipLaunchKernelGGL((bf ? decode_attention_kernel<bf16, kFewRequests, kWaves> : decode_attention_kernel<f16, kFewRequests, kWaves>), dim3(s.grid), dim3(64 * kWaves), 0, st, p);
    else
        hipLaunchKernelGGL((bf ? decode_attention_kernel<bf16, kMostRequests, kWaves> : decode_attention_kernel<f16, kMostRequests, kWaves>), dim3(s.grid), dim3(64 * kWaves), 0, st, p);
    CPMCU_LAUNCH_CHECK();
    // (one part is the whole line: nothing is cut)
    if (s.parts > 1) {
        hipLaunchKernelGGL(bf ? decode_join_kernel<bf16> : decode_join_kernel<f16>, dim3((int)(few + many)), dim3(64 * kJoinWaves), 0, st, p, (int)few);
        CPMCU_LAUNCH_CHECK();
    }
    return CPMCU_OK;
}
