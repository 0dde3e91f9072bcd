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
// A wave takes a tile of its own straight into registers, K and V as the matrix instructions want them (no tile is read by two waves, so
// LDS would add a trip and save none): 32 KB in flight a wave, eight waves a CU.  S^T = K Q^T has the heads as its columns, in 16s; its results are the
// second operand of O^T = V^T P^T as they lie, with the order of tokens that the pages' V has.
#include "batch_attention.h"

#include <algorithm>

namespace cpmcu {
namespace {

constexpr int kHeads = 16;       // columns of the products: heads that a workgroup has at a time
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMostParts = 512;  // workgroups that share the line: two a CU
constexpr int kLeastTiles = kWaves;  // tiles of a part, unless all of the line is less
constexpr int kPartFloats = kHeads * kHeadDim;
constexpr int kJoinWaves = 8;

// Where the second launch finds what belongs together.  Request r's tiles are [start, start + tiles) of each KV head's line.
struct Line {
    int parts;   // that are cut
    int total;   // tiles of one KV head, all requests
    int pad[2];
};
struct Span {
    int start, tiles;
};

struct DecodeParams {
    BatchRows b;
    int units;  // of a request: KV heads times 16s of their heads
    int blocks; // 16s of the heads on a KV head
    Line* line;
    Span* spans;
    float2* stats;  // [2 parts][16]: (reference in powers of two, sum)
    float4* sums;   // [2 parts][8 blocks of 16 dims][64 lanes]
};

// Part i of `parts` of `all` tiles begins here.
__device__ inline int64_t part_begin(int64_t all, int parts, int i) { return all * i / parts; }
// ... and the part that has tile x.
__device__ inline int part_of(int64_t all, int parts, int64_t x) { return (int)(((x + 1) * parts - 1) / all); }

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

template <typename E>
__global__ __launch_bounds__(kThreads, 2) void decode_attention_kernel(DecodeParams p) {
    typedef typename Elem<E>::x8 X8;
    typedef typename Elem<E>::x4 X4;
    __shared__ int tile_end[kMostRequests];
    __shared__ int wave_total[kWaves];
    __shared__ float s_sum[kWaves][32][64];
    __shared__ float2 s_stat[kWaves][kHeads];
    const BatchRows& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int B = b.num_requests, col = lane & 15, lg = lane >> 4;

    // The line: each thread has a run of requests; their running totals.
    const int each = (B + kThreads - 1) / kThreads;
    int mine = 0;
    for (int e = 0; e < each; ++e) {
        const int r = tid * each + e;
        int row, pos;
        const int tiles = r < B ? tiles_of(b, r, row, pos) : 0;
        mine += tiles;
        if (r < B) tile_end[r] = mine;
    }
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int from = __shfl_up(upto, d);
        if (lane >= d) upto += from;
    }
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    int before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += wave_total[w];
        total += wave_total[w];
    }
    for (int e = 0; e < each; ++e) {
        const int r = tid * each + e;
        if (r >= B) break;
        tile_end[r] += before;
    }
    __syncthreads();
    const int64_t all = (int64_t)total * p.units;
    const int parts = (int)min((int64_t)gridDim.x, (all + kLeastTiles - 1) / kLeastTiles);
    if (blockIdx.x == 0) {
        if (tid == 0) *p.line = Line{parts, total, {0, 0}};
        for (int r = tid; r < B; r += kThreads) {
            const int start = r > 0 ? tile_end[r - 1] : 0;
            p.spans[r] = Span{start, tile_end[r] - start};
        }
    }
    if ((int)blockIdx.x >= parts) return;
    int64_t at = part_begin(all, parts, blockIdx.x);
    const int64_t end = part_begin(all, parts, blockIdx.x + 1);
    while (at < end) {
        // the request: the first whose end, on all of its KV heads, lies behind
        int lo = 0, hi = B - 1;
        const int64_t x = at / p.units;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (tile_end[mid] > x) hi = mid;
            else lo = mid + 1;
        }
        const int r = __builtin_amdgcn_readfirstlane(lo);
        const int start = __builtin_amdgcn_readfirstlane(r > 0 ? tile_end[r - 1] : 0), tiles = __builtin_amdgcn_readfirstlane(tile_end[r]) - start;
        const int64_t inside = at - (int64_t)start * p.units;
        const int unit = (int)(inside / tiles), t0 = (int)(inside % tiles), t1 = (int)min((int64_t)tiles, t0 + (end - at));
        const int g = unit / p.blocks, h0 = unit % p.blocks * kHeads;  // of the heads on g
        int row, pos;
        tiles_of(b, r, row, pos);
        const bool has = h0 + col < b.group;
        const int head = g * b.group + min(h0 + col, b.group - 1);

        X8 q[4];  // second operand of S^T = K Q^T: lane (col, lg) has dims 32 kk + 8 lg + [0, 8) of its head
        {
            const E* const from = reinterpret_cast<const E*>(b.q) + (int64_t)row * b.q_stride + head * kHeadDim + 8 * lg;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) q[kk] = *reinterpret_cast<const X8*>(from + 32 * kk);
        }
        const int32_t* const table = b.block_tables + (size_t)r * b.max_blocks;
        f32x4 o[8];
#pragma unroll
        for (int db = 0; db < 8; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_ref = -INFINITY, l_run = 0.f;
        for (int t = t0 + wave; t < t1; t += kWaves) {
            const int c0 = t * kTileKeys, slot0 = c0 % kPage;
            const size_t page = (size_t)page_within(table[c0 / kPage], b.num_pages) * b.Hkv + g;
            const E* const kt = reinterpret_cast<const E*>(b.k_pool) + (page * kPage + slot0) * kHeadDim;
            const E* const vt = reinterpret_cast<const E*>(b.v_pool) + page * kHeadDim * kPage + slot0;
            // Row m of a product's 16 is key 32 sp + 16 (m / 8) + 4 (m / 4 % 2) + m % 4, + 8 in the second of a pair: the results of the two, four and four, are
            // then the eight tokens of a lane's piece of V.
            X8 k[2][2][4], v[2][8];
            const int key = 16 * (col >> 3) + 4 * (col >> 2 & 1) + (col & 3);
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) k[sp][ab][kk] = *reinterpret_cast<const X8*>(kt + (32 * sp + 8 * ab + key) * kHeadDim + 32 * kk + 8 * lg);
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int db = 0; db < 8; ++db) v[sp][db] = *reinterpret_cast<const X8*>(vt + (16 * db + col) * kPage + 32 * sp + 8 * lg);
            f32x4 s[2][2];
#pragma unroll
            for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                for (int ab = 0; ab < 2; ++ab) {
                    s[sp][ab] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) s[sp][ab] = Elem<E>::mfma_16x16x32(k[sp][ab][kk], q[kk], s[sp][ab]);
                }
            // lane (col, lg) has the scores of keys c0 + 32 sp + 16 (lg / 2) + 4 (lg % 2) + 8 ab + i
            const int first = 16 * (lg >> 1) + 4 * (lg & 1);
            if (c0 + kTileKeys - 1 > pos) {
                // behind the row's position lies what the page held before: no score, and no value, not even as 0 times infinity
                const int seen = pos - c0 - first;
#pragma unroll
                for (int sp = 0; sp < 2; ++sp)
#pragma unroll
                    for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool sees = 32 * sp + 8 * ab + i <= seen;
                            s[sp][ab][i] = sees ? s[sp][ab][i] : -INFINITY;
#pragma unroll
                            for (int db = 0; db < 8; ++db) v[sp][db][4 * ab + i] = sees ? v[sp][db][4 * ab + i] : (E)0.f;
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
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32)) * b.scale_log2;
            const float m_new = fmaxf(m_ref, tmax);
            const float m_scaled = m_new == -INFINITY ? 0.f : m_new, alpha = __builtin_amdgcn_exp2f(m_ref - m_scaled);
            m_ref = m_new;
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < 8; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[db][i] *= alpha;
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                X8 pb;  // rounded to the element type; the sum is that of what the product will see
#pragma unroll
                for (int ab = 0; ab < 2; ++ab)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pb[4 * ab + i] = (E)__builtin_amdgcn_exp2f(s[sp][ab][i] * b.scale_log2 - m_scaled);
                        l_run += (float)pb[4 * ab + i];
                    }
#pragma unroll
                for (int db = 0; db < 8; ++db) o[db] = Elem<E>::mfma_16x16x32(v[sp][db], pb, o[db]);
            }
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
        // o[db][i] is dim 16 db + 4 lg + i of head col.  The waves' sums meet in LDS, a quarter of the dims a wave.
        __syncthreads();  // (the last segment's have been read)
#pragma unroll
        for (int db = 0; db < 8; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[wave][db * 4 + i][lane] = o[db][i];
        if (lg == 0) s_stat[wave][col] = make_float2(m_ref, l_run);
        __syncthreads();
        float M = -INFINITY, L = 0.f, f[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_stat[w][col].x);
        const float m_scaled = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            f[w] = __builtin_amdgcn_exp2f(s_stat[w][col].x - m_scaled);
            L = __builtin_fmaf(s_stat[w][col].y, f[w], L);
        }
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);  // of a part that begins a unit's keys and of one that goes on with them
        const float inv = 1.f / L;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int db = 2 * wave + x;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(s_sum[w][db * 4 + i][lane], f[w], sum[i]);
            if (!whole) {
                p.sums[((size_t)slot * 8 + db) * 64 + lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
            } else if (has) {
                X4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (E)(sum[i] * inv);
                *reinterpret_cast<X4*>(reinterpret_cast<E*>(b.out) + (int64_t)row * b.out_stride + head * kHeadDim + 16 * db + 4 * lg) = y;
            }
        }
        if (!whole && wave == 0 && lg == 0) p.stats[slot * kHeads + col] = make_float2(M, L);
        at += t1 - t0;
    }
}

// The parts of a request's keys on a KV head, in their order: M the largest reference, sum_i l_i 2^(m_i - M), out = sum_i O_i 2^(m_i - M) over it.  A workgroup a block
// of 16 dims, its waves every eighth part each.
template <typename E>
__global__ __launch_bounds__(64 * kJoinWaves) void decode_join_kernel(DecodeParams p) {
    typedef typename Elem<E>::x4 X4;
    __shared__ f32x4 s_sum[kJoinWaves][64];
    __shared__ float2 s_stat[kJoinWaves][kHeads];
    const BatchRows& b = p.b;
    const int db = blockIdx.x % 8, unit = blockIdx.x / 8 % p.units, r = blockIdx.x / 8 / p.units;
    const Span span = p.spans[r];
    const Line line = *p.line;
    if (span.tiles == 0) return;
    const int64_t all = (int64_t)line.total * p.units, begin = (int64_t)span.start * p.units + (int64_t)unit * span.tiles;
    const int from = part_of(all, line.parts, begin), to = part_of(all, line.parts, begin + span.tiles - 1);
    if (from == to) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, lg = lane >> 4;
    int row, pos;
    tiles_of(b, r, row, pos);
    constexpr int kAtOnce = 8;
    float M = -INFINITY, L = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = from + wave; i0 <= to; i0 += kJoinWaves * kAtOnce) {
        float2 st[kAtOnce];
        f32x4 o[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int i = min(i0 + u * kJoinWaves, to);
            const int slot = 2 * i + (i == from ? 1 : 0);
            st[u] = p.stats[slot * kHeads + col];
            o[u] = __builtin_bit_cast(f32x4, p.sums[((size_t)slot * 8 + db) * 64 + lane]);
        }
        float m = M;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            if (i0 + u * kJoinWaves <= to) m = fmaxf(m, st[u].x);
        const float m_scaled = m == -INFINITY ? 0.f : m, f = __builtin_amdgcn_exp2f(M - m_scaled);
        M = m;
        L *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] *= f;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if (i0 + u * kJoinWaves > to) break;
            const float w = __builtin_amdgcn_exp2f(st[u].x - m_scaled);
            L = __builtin_fmaf(st[u].y, w, L);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[u][i], w, sum[i]);
        }
    }
    s_sum[wave][lane] = sum;
    if (lg == 0) s_stat[wave][col] = make_float2(M, L);
    __syncthreads();
    if (wave > 0) return;
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) M = fmaxf(M, s_stat[w][col].x);
    const float m_scaled = M == -INFINITY ? 0.f : M;
    L = 0.f;
    sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_stat[w][col].x - m_scaled);
        L = __builtin_fmaf(s_stat[w][col].y, f, L);
        const f32x4 o = s_sum[w][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[i], f, sum[i]);
    }
    const int g = unit / p.blocks, h = unit % p.blocks * kHeads + col;
    if (h >= b.group) return;
    const float inv = 1.f / L;
    X4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (E)(sum[i] * inv);
    *reinterpret_cast<X4*>(reinterpret_cast<E*>(b.out) + (int64_t)row * b.out_stride + (g * b.group + h) * kHeadDim + 16 * db + 4 * lg) = y;
}

struct Sizes {
    int grid;
    size_t spans_at, stats_at, sums_at, bytes;
};
int units_of(int Hq, int Hkv) { return Hkv * ceil_div(Hq / Hkv, kHeads); }
Sizes sizes_of(int num_requests, int max_blocks, int Hq, int Hkv) {
    Sizes s;
    const int64_t tiles = (int64_t)num_requests * max_blocks * (kPage / kTileKeys) * units_of(Hq, Hkv);
    s.grid = (int)std::min<int64_t>(kMostParts, (tiles + kLeastTiles - 1) / kLeastTiles);
    s.spans_at = sizeof(Line);
    s.stats_at = align_up(s.spans_at + sizeof(Span) * num_requests, 256);
    s.sums_at = s.stats_at + sizeof(float2) * kHeads * 2 * s.grid;
    s.bytes = s.sums_at + sizeof(float) * kPartFloats * 2 * s.grid;
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
                                      int max_blocks, const int32_t* row_offsets, const int32_t* positions, int num_requests, int n, int Hq, int Hkv,
                                      float scale, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    BatchRows b{(const uint16_t*)q, (uint16_t*)out, q_stride, out_stride, (const uint16_t*)k_pool, (const uint16_t*)v_pool, block_tables, row_offsets, positions,
                num_requests, max_blocks, num_pages, n, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, scale * 1.44269504088896341f};
    const int rc = check_batch_rows("decode_attention", b, scale);
    if (rc != CPMCU_OK) return rc;
    if (n == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(row_offsets || n == num_requests, "decode_attention: %d rows of %d requests need row_offsets", n, num_requests);
    const Sizes s = sizes_of(num_requests, max_blocks, Hq, Hkv);
    CPMCU_CHECK_ARG(workspace && workspace_bytes >= s.bytes, "decode_attention: workspace of %zu bytes, %zu needed", workspace_bytes, s.bytes);
    CPMCU_CHECK_ARG((uintptr_t)workspace % 16 == 0, "decode_attention: the workspace has to lie on 16 bytes");
    char* const ws = static_cast<char*>(workspace);
    DecodeParams p{b, units_of(Hq, Hkv), ceil_div(b.group, kHeads), (Line*)ws, (Span*)(ws + s.spans_at), (float2*)(ws + s.stats_at), (float4*)(ws + s.sums_at)};
    const hipStream_t st = resolve_stream(stream);
    const bool bf = options().dtype == 1;
    hipLaunchKernelGGL(bf ? decode_attention_kernel<bf16> : decode_attention_kernel<f16>, dim3(s.grid), dim3(kThreads), 0, st, p);
    CPMCU_LAUNCH_CHECK();
    // (one workgroup has the line to itself: nothing is cut)
    if (s.grid > 1) {
        hipLaunchKernelGGL(bf ? decode_join_kernel<bf16> : decode_join_kernel<f16>, dim3(num_requests * p.units * 8), dim3(64 * kJoinWaves), 0, st, p);
        CPMCU_LAUNCH_CHECK();
    }
    return CPMCU_OK;
}
