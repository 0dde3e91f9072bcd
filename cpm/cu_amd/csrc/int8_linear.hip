// Products of 8-bit rows and 8-bit weights with a scale for each row and each channel, and the quantisation of 16-bit rows.
//
//   rows:     s = amax / 127,  q = rint(127 x / amax), ties to even       (amax the row's largest |x|; an empty row has s = 0, q = 0)
//   product:  y[t][c] = (sum over k of q[t][k] w[c][k]) * (s[t] * sw[c])
// The sums are 32-bit integers and exact (16384 * 131071 < 2^31): their order, and with it the split of K, does not show in the
// result, which is rounded to 24 bits, multiplied and rounded once to the element type.
#include "internal.h"

#include <algorithm>
#include <cmath>

namespace cpmcu {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

typedef uint32_t Piece __attribute__((ext_vector_type(4), aligned(2)));  // moved as 16 bytes at any even address

constexpr int kMaxColumns = 131071;
constexpr int kMaxChannels = 1 << 30, kMaxRows = 1 << 30;
constexpr int kCus = 256;             // of an MI355X
constexpr int kStep = 64;             // columns of a matrix instruction; rows and weights are padded to whole steps
constexpr int kBlock = 16;            // channels of a weight block
constexpr int kTile = kBlock * kStep; // bytes of a weight tile: lane l holds channel l & 15, columns (l >> 4) * 16 ..

// ---- rows ----

constexpr int kQuantThreads = 256;
constexpr int kQuantPieces = 8;   // pieces of eight values that a thread keeps between the two passes
constexpr int kQuantRows = 1024;  // as many rows get a wave each

__device__ inline u16x8 max_bits(u16x8 a, u16x8 b) { return __builtin_elementwise_max(a, b); }

// A workgroup a row, which reads rows of up to 16384 values once; a wave a row where there are many rows of up to 4096 values, which spares
// the meeting of the waves and fills the card with loads: 8192 rows of 4096 values 19.3 us (5.2 TB/s, a copy's rate) and 24 by workgroups,
// 8192 of 1024 9.0 and 17.7, 1024 of 4096 4.4 and 5.1, but 512 4.0 and 3.5 and a single one 3.4 and 2.7.  Rows start at any even address:
// 16-byte loads may, and only a row's last values are loaded one by one (8192 rows of 4099: 28 us, 48 with every value by itself).
// |x| is ordered as its bits are, so the maximum is taken on packed 16-bit integers, and an infinity or NaN is a
// maximum from the infinity's pattern on: such a row gets scale NaN and zeros, and its products are NaN.  127 x is exact in 32 bits, and
// the quotient's error is mended by one Newton step, which is exact where the quotient is: rint sees a tie where there is one, and a
// quotient that is none is at least 2^-19 of itself away from the next one.
template <typename E, int THREADS, bool WHOLE>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const E* x, long stride, int n, int K, int padded, int8_t* xq, float* scales) {
    __shared__ uint32_t wave_max[kQuantThreads / 64];
    const int tid = threadIdx.x % THREADS, at = blockIdx.x * (kQuantThreads / THREADS) + threadIdx.x / THREADS;
    if (at >= n) return;  // (only whole waves, and only where no barrier follows)
    const E* row = x + at * stride;
    const auto load = [&](int i) {
        u16x8 v = {};
        if (WHOLE ? 8 * i < K : 8 * i + 8 <= K) {
            v = __builtin_bit_cast(u16x8, *reinterpret_cast<const Piece*>(row + 8 * i));
        } else if (8 * i < K) {
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (8 * i + j < K) v[j] = __builtin_bit_cast(uint16_t, row[8 * i + j]);
        }
        return v;
    };
    const int pieces = padded / 8;
    u16x8 kept[kQuantPieces], m = {};
#pragma unroll
    for (int u = 0; u < kQuantPieces; ++u) {
        kept[u] = load(tid + u * THREADS);
        m = max_bits(m, kept[u] & (uint16_t)0x7FFF);
    }
    for (int i = tid + kQuantPieces * THREADS; i < pieces; i += THREADS) m = max_bits(m, load(i) & (uint16_t)0x7FFF);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, (uint32_t)m[j]);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) wave_max[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) top = max(top, wave_max[w]);
    }
    const float amax = Elem<E>::from_bits((uint16_t)top);
    const bool finite = amax <= Elem<E>::kMaxFinite;
    // (bfloat16 reaches as far as 32 bits do: 127 x and 1 / amax stay in range by a power of two on both)
    const float pre = amax > 0x1p100f ? 0x1p-30f : amax < 0x1p-100f ? 0x1p30f : 1.f;
    const float a = amax * pre, inverse = finite && amax > 0.f ? 1.f / a : 0.f, to127 = 127.f * pre;
    if (tid == 0) scales[at] = finite ? amax / 127.f : __builtin_nanf("");
    uint2* out = reinterpret_cast<uint2*>(xq + (size_t)at * padded);
    const auto put = [&](int i, u16x8 v) {
        uint32_t w[2] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = Elem<E>::from_bits(v[j]) * to127;
            float q = t * inverse;
            q = fmaf(fmaf(-q, a, t), inverse, q);
            const int n = finite ? (int)rintf(q) : 0;
            w[j >> 2] |= (uint32_t)(n & 0xFF) << (8 * (j & 3));
        }
        out[i] = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int u = 0; u < kQuantPieces; ++u)
        if (tid + u * THREADS < pieces) put(tid + u * THREADS, kept[u]);
    for (int i = tid + kQuantPieces * THREADS; i < pieces; i += THREADS) put(i, load(i));
}

// ---- weights ----

// w [V][K] row-major to [ceil(V/16)][ceil(K/64)][64 lanes][16 bytes], zeros where there is no channel or column.
template <bool WIDE>
__global__ __launch_bounds__(256) void int8_weight_tile_kernel(const int8_t* w, int V, int K, int steps, int8_t* tiled) {
    const int lane = threadIdx.x & 63, step = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (step >= steps) return;
    for (int block = blockIdx.x; block < (V + kBlock - 1) / kBlock; block += gridDim.x) {
        const int c = block * kBlock + (lane & 15), k = step * kStep + (lane >> 4) * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < V) {
            const int8_t* from = w + (size_t)c * K + k;
            if constexpr (WIDE) {
                if (k < K) v = *reinterpret_cast<const uint4*>(from);
            } else {
                uint32_t p[4] = {};
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (k + j < K) p[j >> 2] |= (uint32_t)(uint8_t)from[j] << (8 * (j & 3));
                v = make_uint4(p[0], p[1], p[2], p[3]);
            }
        }
        *reinterpret_cast<uint4*>(tiled + ((size_t)block * steps + step) * kTile + lane * 16) = v;
    }
}

// ---- product ----

struct LinearParams {
    const int8_t *xq, *w;
    const float *x_scales, *w_scales;
    void* out;
    int n, V, steps, blocks;  // (blocks of channels)
    int row_tiles, channel_tiles;
    bool quads;  // four channels' results are stored at once
};

// The tile of a workgroup.  Workgroups of equal number modulo 8 share an XCD and its L2: each XCD takes a run of tiles, in columns of up to
// eight row tiles, so that those that run at the same time use few rows and weights.
constexpr int kXcds = 8;
constexpr int kColumn = 8;
__device__ inline void tile_of(const LinearParams& p, int block, int* tx, int* tv) {
    const int total = p.row_tiles * p.channel_tiles, each = total / kXcds, more = total % kXcds, xcd = block % kXcds;
    const int i = xcd * each + min(xcd, more) + block / kXcds;
    const int band = i / (kColumn * p.channel_tiles), rows = min(kColumn, p.row_tiles - band * kColumn), in_band = i - band * kColumn * p.channel_tiles;
    *tx = band * kColumn + in_band % rows;
    *tv = in_band / rows;
}

// Rows are requested so that four lanes take 64 neighbouring bytes: requests whose neighbouring lanes are in different rows, as the operands are, reach
// 38 to 51 GB/s a CU from L2, and 110 to 150 this way.  LDS puts the operands together: row r of a block has piece c of a step's four in place c ^ turned(r), which
// keeps the lanes that are served at once in different banks (no conflicts are counted; with the places in another order 40 % of LDS's cycles).
__device__ inline int turned(int r) { return r >> 3 << 1; }
__device__ inline int operand_place(int lane) { return (lane & 15) * 4 + ((lane >> 4) ^ turned(lane & 15)); }  // in 16-byte places

// Channels c .. c + 3 of row t.
template <typename E>
__device__ inline void store_quad(const LinearParams& p, int t, int c, i32x4 sum) {
    if (t >= p.n || c >= p.V) return;
    const float s = p.x_scales[t];
    uint16_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = c + j < p.V ? Elem<E>::to_bits((float)sum[j] * (s * p.w_scales[c + j])) : 0;
    uint16_t* to = (uint16_t*)p.out + (size_t)t * p.V + c;
    if (p.quads) {
        *reinterpret_cast<uint2*>(to) = make_uint2(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < p.V) to[j] = y[j];
    }
}

// NX blocks of rows and NV blocks of channels per workgroup, for few rows: the weights are the bytes, each is read by one workgroup, and the
// waves take K's steps in turn, so that a workgroup's requests are whole kilobytes one behind the other.  A wave requests U steps at once
// while it works on the U before them; rows go through LDS for the operands' order (which spares 1.8 of 9.5 us at 17 rows of
// 4096 columns to 4608 channels); the waves' sums meet in LDS, where a wave adds up each block's (0.4 us less than halving the waves).  One row: 5.6 us.
constexpr int kSplit = 8;

template <typename E, int NX, int NV, int U>
__global__ __launch_bounds__(64 * kSplit) void int8_linear_split_kernel(LinearParams p) {
    constexpr int kQuads = NX * NV;
    __shared__ union {
        i32x4 part[kSplit][kQuads][64];
        i32x4 rows[kSplit][U][NX][64];
    } lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tx, tv;
    tile_of(p, blockIdx.x, &tx, &tv);
    const int t0 = tx * NX * 16, b0 = tv * NV, last = p.steps - 1;
    const int8_t *x[NX], *w[NV];
#pragma unroll
    for (int b = 0; b < NX; ++b) x[b] = p.xq + (size_t)min(t0 + b * 16 + (lane >> 2), p.n - 1) * p.steps * kStep + ((lane & 3) ^ turned(lane >> 2)) * 16;
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = p.w + (size_t)min(b0 + v, p.blocks - 1) * p.steps * kTile + lane * 16;
    struct Group {
        i32x4 a[U][NV], x[U][NX];
    };
    const auto load = [&](int s, Group& g) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t at = min(s + u * kSplit, last);
#pragma unroll
            for (int v = 0; v < NV; ++v) g.a[u][v] = *reinterpret_cast<const i32x4*>(w[v] + at * kTile);
#pragma unroll
            for (int b = 0; b < NX; ++b) g.x[u][b] = *reinterpret_cast<const i32x4*>(x[b] + at * kStep);
        }
    };
    // Lanes read what other lanes of their wave wrote: LDS serves a wave in the order of its requests, which the fences keep (they cost no instruction).
    const auto fence = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    i32x4 acc[NX][NV] = {};
    const auto multiply = [&](int s, const Group& g) {
        i32x4(&rows)[U][NX][64] = lds.rows[wave];  // (one wave's own: no barrier)
        fence();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int b = 0; b < NX; ++b) rows[u][b][lane] = g.x[u][b];
        fence();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u * kSplit > last) break;  // (the same for the whole wave)
#pragma unroll
            for (int b = 0; b < NX; ++b) {
                const i32x4 r = rows[u][b][operand_place(lane)];
#pragma unroll
                for (int v = 0; v < NV; ++v) acc[b][v] = __builtin_amdgcn_mfma_i32_16x16x64_i8(g.a[u][v], r, acc[b][v], 0, 0, 0);
            }
        }
    };
    constexpr int kTurn = U * kSplit;
    Group g0, g1;
    load(wave, g0);
    for (int s = wave; s <= last; s += 2 * kTurn) {
        if (s + kTurn <= last) load(s + kTurn, g1);
        multiply(s, g0);
        if (s + kTurn > last) break;
        if (s + 2 * kTurn <= last) load(s + 2 * kTurn, g0);
        multiply(s + kTurn, g1);
    }
    __syncthreads();  // (the sums lie where rows were)
#pragma unroll
    for (int b = 0; b < NX; ++b)
#pragma unroll
        for (int v = 0; v < NV; ++v) lds.part[wave][b * NV + v][lane] = acc[b][v];
    __syncthreads();
    static_assert(kQuads <= kSplit, "a wave for each block of sums");
    if (wave >= kQuads) return;
    i32x4 sum = {};
#pragma unroll
    for (int u = 0; u < kSplit; ++u) sum += lds.part[u][wave][lane];
    store_quad<E>(p, t0 + wave / NV * 16 + (lane & 15), (b0 + wave % NV) * kBlock + (lane >> 4) * 4, sum);
}

// A wave's tile: NX blocks of rows from t0 on, NV blocks of channels from c0 on.  The results go through LDS, as many blocks of rows at a time
// as ROOM bytes of the wave's own hold, so that a row's are stored as one run of NV * 32 bytes (as they lie in the accumulators a row has 8);
// rows of an uneven V start anywhere, which 16-byte stores may.  They go past the L2 (8192 rows of 4096 columns to 16384 channels with the
// rows' quantisation 495 us, 505 through it).
template <typename E, int NX, int NV, int ROOM>
__device__ inline void store_tile(const LinearParams& p, int t0, int c0, i32x4 (&acc)[NX][NV], int8_t* part) {
    constexpr int kRoom = ROOM / (512 * NV), kPieces = 2 * NV, kPass = NX <= kRoom ? NX : kRoom < 4 ? 2 : kRoom < 8 ? 4 : 8;
    static_assert(kRoom >= 2 && NX % kPass == 0, "passes of whole blocks");
    const int lane = threadIdx.x & 63;
    float sw[NV][4];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) sw[v][j] = p.w_scales[min(c0 + v * kBlock + (lane >> 4) * 4 + j, p.V - 1)];
#pragma unroll
    for (int b1 = 0; b1 < NX; b1 += kPass) {
        const int t1 = t0 + b1 * 16;
#pragma unroll
        for (int b = 0; b < kPass; ++b) {
            const int r = b * 16 + (lane & 15);
            const float sx = p.x_scales[min(t1 + r, p.n - 1)];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const i32x4 sum = acc[b1 + b][v];
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = Elem<E>::to_bits((float)sum[j] * (sx * sw[v][j]));
                const int piece = (v * 2 + (lane >> 5)) ^ (r & (kPieces - 1));
                *reinterpret_cast<uint2*>(part + r * (kPieces * 16) + piece * 16 + ((lane >> 4) & 1) * 8) = make_uint2(y[0] | y[1] << 16, y[2] | y[3] << 16);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // (one wave's own: no barrier)
#pragma unroll
        for (int i = 0; i < (kPass * 16 * kPieces + 63) / 64; ++i) {
            const int r = i * (64 / kPieces) + lane / kPieces, piece = lane % kPieces, t = t1 + r, c = c0 + piece * 8;
            const uint4 y = *reinterpret_cast<const uint4*>(part + r * (kPieces * 16) + (piece ^ (r & (kPieces - 1))) * 16);
            if (r >= kPass * 16 || t >= p.n || c >= p.V) continue;
            uint16_t* to = (uint16_t*)p.out + (size_t)t * p.V + c;
            if (c + 8 <= p.V) {
                __builtin_nontemporal_store(Piece{y.x, y.y, y.z, y.w}, reinterpret_cast<Piece*>(to));
            } else {
                const uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (c + j < p.V) to[j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
}

// Tiles of (WX NX) x (WV NV) blocks for more rows: WX x WV waves, each with NX x NV of the blocks in its accumulators, and KS such groups, each with
// a share of K: a second group hides the first one's waits where a CU has one tile (256 rows of 4096 columns to 4608 channels 12.6 us, 14.9 with one
// group, 17.7 with one and requests in the operands' order).
// Rows go to LDS by direct loads, two steps at a time, eight rows of whole 128-byte lines a request; row r has piece c of a line's eight in place
// c ^ (r % 8), so that the operands are read back without bank conflicts.  Weights lie
// in operand order already and go straight into registers, AHEAD pairs of steps in advance, so that LDS is read for the rows alone.
// Half of a step's rows are read from LDS while the other half is multiplied, so the next pair's have to be there a pair early: its
// rows are requested in front of the weights of two pairs before.  Requests return in order, and the wait for the weights of pair j, which the
// compiler puts in front of their first use, is one for the rows of pair j + 2 as well; the one in front of the barrier says so.
template <typename E, int NX, int NV, int WX, int WV, int AHEAD, int KS>
__global__ __launch_bounds__(64 * WX * WV * KS, WX * WV * KS / 4) void int8_linear_tile_kernel(LinearParams p) {
    constexpr int kWaves = WX * WV, kBlocks = WX * NX, kLoads = 2 * kBlocks / kWaves, kStages = AHEAD + 3, kHalf = NX / 2, kSets = 2 * (AHEAD + 1);
    static_assert(KS == 1 || (KS == 2 && kHalf * NV * 1024 <= kStages * kLoads * kTile), "the groups' sums have room in the ring");
    static_assert(2 * kBlocks % kWaves == 0 && NX % 2 == 0, "every wave requests as many kilobytes of rows");
    constexpr int kStageBytes = kBlocks * 2 * kTile;
    __shared__ __attribute__((aligned(16))) int8_t ring[KS * kStages * kStageBytes];
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = all / kWaves, wave = all % kWaves, wx = wave / WV, wv = wave % WV;
    int tx, tv;
    tile_of(p, blockIdx.x, &tx, &tv);
    const int t0 = tx * kBlocks * 16, b0 = (tv * WV + wv) * NV, last_pair = (p.steps - 1) / 2;
    // this group's pairs of steps: [first, end), of which `pairs` are whole
    const int per = last_pair / KS + 1, first = min(group * per, last_pair), end = min(group * per + per, last_pair + 1), pairs = max(min(end, p.steps / 2) - group * per, 0);
    const bool odd = (p.steps & 1) && group * per <= last_pair && end == last_pair + 1;
    // (an uneven last step: its pair takes the columns of the one step twice, and only the first is multiplied)
    const uint32_t piece = (lane & 7) ^ (lane >> 3), no_second = (p.steps & 1) && piece >= 4 ? kStep : 0;
    const int8_t* x_tile = p.xq + (size_t)t0 * p.steps * kStep;
    uint32_t row[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) row[j] = (uint32_t)(min((wave * kLoads + j) * 8 + (lane >> 3), p.n - 1 - t0) * p.steps * kStep) + piece * 16;
    const int8_t* w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = p.w + (size_t)min(b0 + v, p.blocks - 1) * p.steps * kTile;
    const uint32_t lane16 = lane * 16, ring_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)ring + group * (kStages * kStageBytes) + wave * (kLoads * kTile);
    const auto request = [&](int pair, int stage) {
        const int at = min(first + pair, max(end - 1, first));
        const int8_t* from = x_tile + (size_t)at * (2 * kStep);
        const uint32_t back = at == last_pair ? no_second : 0;
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(row[j] - back), "s"(from), "s"(ring_at + stage * kStageBytes + j * kTile) : "memory", "m0");
    };
    const auto weights = [&](int s, i32x4* a) {
#pragma unroll
        for (int v = 0; v < NV; ++v) a[v] = *reinterpret_cast<const i32x4*>(w[v] + (size_t)min(2 * first + s, min(max(2 * end, 2 * first + 1), p.steps) - 1) * kTile + lane16);
    };
    i32x4 acc[NX][NV] = {}, x0[kHalf], x1[kHalf];
    const int8_t* mine = ring + group * (kStages * kStageBytes) + wx * (NX * 2 * kTile) + ((lane & 15) >> 3) * kTile + (lane & 7) * 128;
    const int at[2] = {((lane >> 4) ^ (lane & 7)) * 16, ((4 + (lane >> 4)) ^ (lane & 7)) * 16};
    // The order below is kept: what is read comes ahead of the products that hide its way.
    const auto read = [&](int stage, int second, int half, i32x4* x) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < kHalf; ++b) x[b] = *reinterpret_cast<const i32x4*>(mine + stage * kStageBytes + (half * kHalf + b) * (2 * kTile) + at[second]);
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](const i32x4* a, const i32x4* x, int half) {
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int v = 0; v < NV; ++v) acc[half * kHalf + b][v] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[v], x[b], acc[half * kHalf + b][v], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto after = [](int stage, int n) { return stage + n >= kStages ? stage + n - kStages : stage + n; };
    i32x4 a[kSets][NV];
    request(0, 0);
    request(1, 1);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        request(j + 2, j + 2);
        weights(2 * j, a[2 * j]);
        weights(2 * j + 1, a[2 * j + 1]);
    }
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(AHEAD * (kLoads + 2 * NV)) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    int stage = 0;
    read(0, 0, 0, x0);
    for (int j0 = 0; j0 < pairs; j0 += AHEAD + 1) {
#pragma unroll
        for (int u = 0; u <= AHEAD; ++u) {
            const int j = j0 + u;
            if (j < pairs) {
                read(stage, 0, 1, x1);
                request(j + AHEAD + 2, after(stage, AHEAD + 2));
                weights(2 * (j + AHEAD), a[2 * (u + AHEAD) % kSets]);
                multiply(a[2 * u], x0, 0);
                read(stage, 1, 0, x0);
                multiply(a[2 * u], x1, 1);
                read(stage, 1, 1, x1);
                weights(2 * (j + AHEAD) + 1, a[(2 * (u + AHEAD) + 1) % kSets]);
                multiply(a[2 * u + 1], x0, 0);
                stage = after(stage, 1);
                read(stage, 0, 0, x0);
                multiply(a[2 * u + 1], x1, 1);
                // the rows read so far are in registers, those of pair j + 2 in LDS: behind them AHEAD pairs' requests at most
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(AHEAD * (kLoads + 2 * NV)) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" : : : "memory");
            }
        }
    }
    if constexpr (KS > 1) {  // (a barrier for every pair of the group that has most)
        for (int j = pairs; j < min(per, p.steps / 2); ++j) __builtin_amdgcn_s_barrier();
    }
    if (odd) {
        read(stage, 0, 1, x1);
#pragma unroll
        for (int u = 0; u <= AHEAD; ++u)
            if (pairs % (AHEAD + 1) == u) {
                multiply(a[2 * u], x0, 0);
                multiply(a[2 * u], x1, 1);
            }
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (requests beyond the last pair write to LDS, too)
    __syncthreads();
    if constexpr (KS == 1) {
        store_tile<E, NX, NV, kStages * kLoads * kTile>(p, t0 + wx * NX * 16, b0 * kBlock, acc, ring + wave * (kStages * kLoads * kTile));
    } else {  // each group takes half of the rows, and gives the sums of the others
        i32x4 half[kHalf][NV];
        i32x4* given = reinterpret_cast<i32x4*>(ring) + all * (kHalf * NV * 64) + lane;
        const i32x4* taken = reinterpret_cast<const i32x4*>(ring) + ((1 - group) * kWaves + wave) * (kHalf * NV * 64) + lane;
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                given[(b * NV + v) * 64] = group == 0 ? acc[kHalf + b][v] : acc[b][v];
                half[b][v] = group == 0 ? acc[b][v] : acc[kHalf + b][v];
            }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int v = 0; v < NV; ++v) half[b][v] += taken[(b * NV + v) * 64];
        __syncthreads();
        store_tile<E, kHalf, NV, kStages * kLoads * kTile>(p, t0 + (wx * NX + group * kHalf) * 16, b0 * kBlock, half, ring + all * (kStages * kLoads * kTile));
    }
}

// Larger tiles for many rows.  With waves that share channels each weight crosses from L2 once for every one of them; here rows and weights are both in
// LDS and a CU takes each once.  A step is requested three in advance and has to be there one early, as above.  A CU with 256 x 256 to do takes
// 0.6 us a step where few CUs run and 0.8 to 0.9 where all do, of which the matrix cores need 0.43 at their peak: 2260 TOP/s at 8192 x 4096 x 16384 (rows,
// columns, channels), 2510 at 8192 x 16384 x 4096, 10 % more on zeros, which draw less power; deeper rings and other orders of the tiles change nothing.
// LDS needs as long as the matrix cores: eight waves read 12 KiB a step and 32 KiB are written, 1024 cycles at 128 bytes each, so the two have to run side by side whole.
template <typename E, int NX, int NV, int WX, int WV>
__global__ __launch_bounds__(64 * WX * WV, WX * WV / 4) void int8_linear_wide_kernel(LinearParams p) {
    constexpr int kWaves = WX * WV, kRows = WX * NX, kChannels = WV * NV, kStages = 4, kStageBytes = (kRows + kChannels) * kTile, kHalf = NX / 2;
    constexpr int kX = kRows / kWaves, kW = kChannels / kWaves, kRoom = kStages * kStageBytes / kWaves;
    __shared__ __attribute__((aligned(16))) int8_t ring[kStages * kStageBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wx = wave / WV, wv = wave % WV;
    int tx, tv;
    tile_of(p, blockIdx.x, &tx, &tv);
    const int t0 = tx * kRows * 16, last = p.steps - 1;
    const int8_t* x_tile = p.xq + (size_t)t0 * p.steps * kStep;
    uint32_t row[kX];
    const int8_t* w[kW];
#pragma unroll
    for (int j = 0; j < kX; ++j) row[j] = (uint32_t)(min((wave * kX + j) * 16 + (lane >> 2), p.n - 1 - t0) * p.steps * kStep) + ((lane & 3) ^ turned(lane >> 2)) * 16;
#pragma unroll
    for (int j = 0; j < kW; ++j) w[j] = p.w + (size_t)min(tv * kChannels + wave * kW + j, p.blocks - 1) * p.steps * kTile;
    const uint32_t lane16 = lane * 16, ring_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)ring;
    const auto request = [&](int s, int stage) {
        const size_t at = min(s, last);
        const uint32_t to = ring_at + stage * kStageBytes;
#pragma unroll
        for (int j = 0; j < kX; ++j)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(row[j]), "s"(x_tile + at * kStep), "s"(to + (wave * kX + j) * kTile) : "memory", "m0");
#pragma unroll
        for (int j = 0; j < kW; ++j)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane16), "s"(w[j] + at * kTile), "s"(to + (kRows + wave * kW + j) * kTile) : "memory", "m0");
    };
    i32x4 acc[NX][NV] = {}, x0[kHalf], x1[kHalf], a0[NV], a1[NV];
    const int8_t* x_at = ring + wx * (NX * kTile) + operand_place(lane) * 16;
    const int8_t* w_at = ring + (kRows + wv * NV) * kTile + lane16;
    const auto read_x = [&](int stage, int half, i32x4* x) {
#pragma unroll
        for (int b = 0; b < kHalf; ++b) x[b] = *reinterpret_cast<const i32x4*>(x_at + stage * kStageBytes + (half * kHalf + b) * kTile);
    };
    const auto read_w = [&](int stage, i32x4* a) {
#pragma unroll
        for (int v = 0; v < NV; ++v) a[v] = *reinterpret_cast<const i32x4*>(w_at + stage * kStageBytes + v * kTile);
    };
    // The order is kept: what is read comes ahead of the products that hide its way.
    const auto multiply = [&](const i32x4* a, const i32x4* x, int half) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int v = 0; v < NV; ++v) acc[half * kHalf + b][v] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[v], x[b], acc[half * kHalf + b][v], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto step = [&](int s, const i32x4* a, i32x4* next) {
        const int now = s % kStages, then = (s + 1) % kStages;
        read_x(now, 1, x1);
        request(s + 3, (s + 3) % kStages);
        multiply(a, x0, 0);
        read_w(then, next);
        read_x(then, 0, x0);
        multiply(a, x1, 1);
        // what was read is in registers, step s + 2 in LDS: behind it the requests of step s + 3
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(kX + kW) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
    };
    request(0, 0);
    request(1, 1);
    request(2, 2);
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kX + kW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read_w(0, a0);
    read_x(0, 0, x0);
    for (int s = 0; s < p.steps; s += 2) {
        step(s, a0, a1);
        if (s + 1 < p.steps) step(s + 1, a1, a0);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (requests beyond the last step write to LDS, too)
    __syncthreads();
    store_tile<E, NX, NV, kRoom>(p, t0 + wx * NX * 16, (tv * kChannels + wv * NV) * kBlock, acc, ring + wave * kRoom);
}

// The shapes, and what they cost, fitted to 448 sizes of 1 to 8192 rows, 512 to 73448 channels and 512 to 16384 columns: `start` us of a launch; for a
// round (a tile on every CU) `round` us and `step` more for every 64 columns, `busy` more of them where all CUs work; and `whole` says how much of a
// last round that is not full counts as a full one.  The choice is the shape with the least cost: against the best of the eight, timed again, 0.8 % more in
// the mean of those sizes and 12 % at most (0.3 us), and 1.8 % and 52 % (600 rows of 64 columns to 4096 channels: 7.4 us, 4.9) over 182 sizes that
// were no part of the fit, 64 to 500 channels or columns among them (profiles/int8_linear_shapes.txt; `python -m cpm.cu_amd.sweep int8` times them).
// In us, rows x columns x channels: 1 x 4096 x 4608 16 x 32 split 5.7, 16 x 16 6.0, 32 x 64 7.7; 64 x 4096 x 4608 32 x 64 8.4, 16 x 64 split 9.6, 64 x 128
// 12.1; 64 x 4096 x 4096 16 x 64 split 6.8, 32 x 64 8.3; 256 x 4096 x 4608 64 x 128 12.3, 32 x 64 15.5, 64 x 256 19.1; 333 x 4099 x 12289 128 x 256 26.8,
// 64 x 128 33.0, 64 x 256 33.9, 256 x 256 46.1; 2048 x 4096 x 16384: 256 x 256 115, 128 x 256 127, 64 x 256 135.
struct Variant {
    const char* name;
    void (*f16_kernel)(LinearParams);
    void (*bf16_kernel)(LinearParams);
    int rows, channels, threads;
    float start, round, step, busy, whole;
};
#define CPMCU_SPLIT(nx, nv, u) "int8_linear_split_kernel<" #nx "," #nv ">", int8_linear_split_kernel<f16, nx, nv, u>, int8_linear_split_kernel<bf16, nx, nv, u>, 16 * nx, kBlock* nv, 64 * kSplit
#define CPMCU_TILE(nx, nv, wx, wv, ahead, ks)                                                                                                                   \
    "int8_linear_tile_kernel<" #nx "," #nv "," #wx "," #wv "," #ks ">", int8_linear_tile_kernel<f16, nx, nv, wx, wv, ahead, ks>, \
        int8_linear_tile_kernel<bf16, nx, nv, wx, wv, ahead, ks>, 16 * nx * wx, kBlock* nv* wv, 64 * wx * wv * ks
#define CPMCU_WIDE(nx, nv, wx, wv)                                                                                                                     \
    "int8_linear_wide_kernel<" #nx "," #nv "," #wx "," #wv ">", int8_linear_wide_kernel<f16, nx, nv, wx, wv>, int8_linear_wide_kernel<bf16, nx, nv, wx, wv>, \
        16 * nx * wx, kBlock* nv* wv, 64 * wx * wv
const Variant kVariants[kInt8LinearShapes] = {
    {CPMCU_SPLIT(1, 1, 4), 2.7f, 0.51f, 0.0027f, 0.02f, 0.6f},        {CPMCU_SPLIT(1, 2, 4), 2.5f, 0.33f, 0.0245f, 0.011f, 0.4f},
    {CPMCU_SPLIT(1, 4, 2), 2.4f, 0.33f, 0.0437f, 0.0095f, 0.4f},      {CPMCU_TILE(2, 1, 1, 4, 3, 2), 2.4f, 0.44f, 0.0754f, 0.f, 0.4f},
    {CPMCU_TILE(4, 2, 1, 4, 2, 2), 2.7f, 1.48f, 0.116f, 0.043f, 0.5f}, {CPMCU_TILE(4, 4, 1, 4, 2, 1), 3.5f, 1.16f, 0.229f, 0.037f, 0.6f},
    {CPMCU_WIDE(4, 4, 2, 4), 1.5f, 3.46f, 0.279f, 0.16f, 1.f},        {CPMCU_WIDE(8, 4, 2, 4), 4.3f, 4.f, 0.457f, 0.37f, 0.6f}};
#undef CPMCU_SPLIT
#undef CPMCU_TILE
#undef CPMCU_WIDE

int choose_variant(int n, int V, int K) {
    if (options().int8_linear_shape >= 0) return options().int8_linear_shape;
    const int steps = ceil_div(K, kStep);
    int best = 0;
    float least = 0.f;
    for (int i = 0; i < kInt8LinearShapes; ++i) {
        const Variant& v = kVariants[i];
        const float tiles = (float)ceil_div(n, v.rows) * (float)ceil_div(V, v.channels) / kCus;
        const float rounds = tiles <= 1.f ? 1.f : v.whole * std::ceil(tiles) + (1.f - v.whole) * tiles;
        const float cost = v.start + rounds * (v.round + (float)steps * (v.step + v.busy * std::min(tiles, 1.f)));
        const float floor = (float)V * (float)K / 6e6f;  // (weights at 6 TB/s)
        const float total = std::max(cost, floor) + 0.1f * cost;
        if (i == 0 || total < least) {
            best = i;
            least = total;
        }
    }
    return best;
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" int cpmcu_quantize_rows(const void* x, int64_t x_stride, int n, int K, int8_t* xq, float* scales, void* stream) {
    CPMCU_CHECK_ARG(n >= 0 && K >= 1 && K <= kMaxColumns, "quantize_rows: n=%d, K=%d outside [1, %d]", n, K, kMaxColumns);
    if (n == 0) return CPMCU_OK;  // (rows that are not there may have no memory)
    CPMCU_CHECK_ARG(x && xq && scales, "quantize_rows: null pointer argument");
    CPMCU_CHECK_ARG(n < 1 << 24, "quantize_rows: n=%d, more rows than a launch has workgroups", n);
    CPMCU_CHECK_ARG(x_stride >= K, "quantize_rows: rows closer than their %d values", K);
    const int padded = ceil_div(K, kStep) * kStep;
    const size_t x_bytes = 2 * ((size_t)(n - 1) * (size_t)x_stride + K), q_bytes = (size_t)n * padded, s_bytes = 4 * (size_t)n;
    CPMCU_CHECK_ARG(!overlap(xq, q_bytes, x, x_bytes) && !overlap(scales, s_bytes, x, x_bytes) && !overlap(xq, q_bytes, scales, s_bytes), "quantize_rows: the results lie in the rows' memory or in each other's");
    CPMCU_CHECK_ARG((uintptr_t)xq % 16 == 0, "quantize_rows: xq has to lie on 16 bytes");
    hipStream_t st = resolve_stream(stream);
    const bool whole = K % 8 == 0, waves = n >= kQuantRows && padded <= 64 * 8 * kQuantPieces;
#define CPMCU_QUANT(E)                                                                                                                              \
    hipLaunchKernelGGL((waves ? whole ? quantize_rows_kernel<E, 64, true> : quantize_rows_kernel<E, 64, false>                                      \
                              : whole ? quantize_rows_kernel<E, kQuantThreads, true> : quantize_rows_kernel<E, kQuantThreads, false>),              \
                       dim3(waves ? ceil_div(n, kQuantThreads / 64) : n), dim3(kQuantThreads), 0, st, (const E*)x, (long)x_stride, n, K, padded, xq, scales)
    if (options().dtype == 1) CPMCU_QUANT(bf16);
    else CPMCU_QUANT(f16);
#undef CPMCU_QUANT
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}

extern "C" size_t cpmcu_int8_weight_bytes(int V, int K) {
    if (V < 1 || V > kMaxChannels || K < 1 || K > kMaxColumns) return 0;
    return (size_t)ceil_div(V, kBlock) * ceil_div(K, kStep) * kTile;
}

extern "C" int cpmcu_int8_weight_tile(const int8_t* w, int V, int K, int8_t* w_tiled, void* stream) {
    CPMCU_CHECK_ARG(w && w_tiled && (const void*)w != (const void*)w_tiled, "int8_weight_tile: null or aliased pointer argument");
    CPMCU_CHECK_ARG(V >= 1 && V <= kMaxChannels && K >= 1 && K <= kMaxColumns, "int8_weight_tile: V=%d outside [1, %d] or K=%d outside [1, %d]", V, kMaxChannels, K, kMaxColumns);
    CPMCU_CHECK_ARG((uintptr_t)w_tiled % 16 == 0, "int8_weight_tile: w_tiled has to lie on 16 bytes");
    const bool wide = (uintptr_t)w % 16 == 0 && K % 16 == 0;
    const int steps = ceil_div(K, kStep);
    const dim3 grid(std::min(ceil_div(V, kBlock), 1 << 20), ceil_div(steps, 4));
    hipLaunchKernelGGL(wide ? int8_weight_tile_kernel<true> : int8_weight_tile_kernel<false>, grid, dim3(256), 0, resolve_stream(stream), w, V, K, steps, w_tiled);
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}

extern "C" int cpmcu_int8_linear_plan(int n, int V, int K, char* kernel_name, size_t kernel_name_bytes, int* num_workgroups) {
    CPMCU_CHECK_ARG(n >= 1 && n <= kMaxRows && V >= 1 && V <= kMaxChannels && K >= 1 && K <= kMaxColumns, "int8_linear_plan: n=%d, V=%d, K=%d outside [1, %d]", n, V, K, kMaxColumns);
    const Variant& v = kVariants[choose_variant(n, V, K)];
    if (kernel_name && kernel_name_bytes) snprintf(kernel_name, kernel_name_bytes, "%s", v.name);
    if (num_workgroups) *num_workgroups = (int)std::min<int64_t>((int64_t)ceil_div(n, v.rows) * ceil_div(V, v.channels), INT32_MAX);
    return CPMCU_OK;
}

extern "C" int cpmcu_int8_linear(const int8_t* xq, const float* x_scales, const int8_t* w_tiled, const float* w_scales, int n, int V, int K, void* out,
                                 void* stream) {
    CPMCU_CHECK_ARG(n >= 0 && n <= kMaxRows && V >= 1 && V <= kMaxChannels && K >= 1 && K <= kMaxColumns, "int8_linear: n=%d, V=%d, K=%d outside [1, %d]", n, V, K, kMaxColumns);
    if (n == 0) return CPMCU_OK;
    CPMCU_CHECK_ARG(xq && x_scales && w_tiled && w_scales && out, "int8_linear: null pointer argument");
    CPMCU_CHECK_ARG(((uintptr_t)xq | (uintptr_t)w_tiled) % 16 == 0, "int8_linear: xq and w_tiled have to lie on 16 bytes");
    LinearParams p{xq, w_tiled, x_scales, w_scales, out, n, V, ceil_div(K, kStep), ceil_div(V, kBlock), 0, 0, V % 4 == 0 && (uintptr_t)out % 8 == 0};
    const Variant v = kVariants[choose_variant(n, V, K)];
    p.row_tiles = ceil_div(n, v.rows);
    p.channel_tiles = ceil_div(V, v.channels);
    CPMCU_CHECK_ARG((int64_t)p.row_tiles * p.channel_tiles * v.threads <= UINT32_MAX, "int8_linear: n=%d rows of V=%d channels are more than a launch has threads", n, V);
    const size_t bytes = 2 * (size_t)n * V;
    CPMCU_CHECK_ARG(!overlap(out, bytes, xq, (size_t)n * p.steps * kStep) && !overlap(out, bytes, x_scales, 4 * (size_t)n) && !overlap(out, bytes, w_tiled, cpmcu_int8_weight_bytes(V, K)) &&
                        !overlap(out, bytes, w_scales, 4 * (size_t)V),
                    "int8_linear: out is the memory of an input");
    const dim3 grid(p.row_tiles * p.channel_tiles);
    hipLaunchKernelGGL(options().dtype == 1 ? v.bf16_kernel : v.f16_kernel, grid, dim3(v.threads), 0, resolve_stream(stream), p);
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
