// Products of 8-bit rows and 8-bit weights with a scale for each row and each channel, and the quantisation of 16-bit rows.
//
//   rows:     s = amax / 127,  q = rint(127 x / amax), ties to even       (amax the row's largest |x|; an empty row has s = 0, q = 0)
//   product:  y[t][c] = (sum over k of q[t][k] w[c][k]) * (s[t] * sw[c])
// The sums are 32-bit integers and exact (16384 * 131071 < 2^31): their order, and with it the split of K, does not show in the
// result, which is rounded to 24 bits, multiplied and rounded once to the element type.
#include "internal.h"

#include <algorithm>

namespace cpmcu {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxColumns = 131071;
constexpr int kStep = 64;             // columns of a matrix instruction; rows and weights are padded to whole steps
constexpr int kBlock = 16;            // channels of a weight block
constexpr int kTile = kBlock * kStep; // bytes of a weight tile: lane l holds channel l & 15, columns (l >> 4) * 16 ..

// ---- rows ----

constexpr int kQuantThreads = 256;
constexpr int kQuantPieces = 8;  // pieces of eight values that a thread keeps between the two passes: rows of up to 16384 values are read once

__device__ inline u16x8 max_bits(u16x8 a, u16x8 b) { return __builtin_elementwise_max(a, b); }

// One workgroup a row.  |x| is ordered as its bits are, so the maximum is taken on packed 16-bit integers, and an infinity or NaN is a
// maximum from the infinity's pattern on: such a row gets scale NaN and zeros, and its products are NaN.  127 x is exact in 32 bits, and
// the quotient's error is mended by one Newton step, which is exact where the quotient is: rint sees a tie where there is one, and a
// quotient that is none is at least 2^-19 of itself away from the next one.
template <typename E, bool WIDE>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const E* x, long stride, int K, int padded, int8_t* xq, float* scales) {
    __shared__ uint32_t wave_max[kQuantThreads / 64];
    const int tid = threadIdx.x;
    const E* row = x + blockIdx.x * stride;
    const auto load = [&](int i) {
        u16x8 v = {};
        if constexpr (WIDE) {
            if (8 * i < K) v = *reinterpret_cast<const u16x8*>(row + 8 * i);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * i + j < K) v[j] = __builtin_bit_cast(uint16_t, row[8 * i + j]);
        }
        return v;
    };
    const int pieces = padded / 8;
    u16x8 kept[kQuantPieces], m = {};
#pragma unroll
    for (int u = 0; u < kQuantPieces; ++u) {
        kept[u] = load(tid + u * kQuantThreads);
        m = max_bits(m, kept[u] & (uint16_t)0x7FFF);
    }
    for (int i = tid + kQuantPieces * kQuantThreads; i < pieces; i += kQuantThreads) m = max_bits(m, load(i) & (uint16_t)0x7FFF);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, (uint32_t)m[j]);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if ((tid & 63) == 0) wave_max[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantThreads / 64; ++w) top = max(top, wave_max[w]);
    const float amax = Elem<E>::from_bits((uint16_t)top);
    const bool finite = amax <= Elem<E>::kMaxFinite;
    // (bfloat16 reaches as far as 32 bits do: 127 x and 1 / amax stay in range by a power of two on both)
    const float pre = amax > 0x1p100f ? 0x1p-30f : amax < 0x1p-100f ? 0x1p30f : 1.f;
    const float a = amax * pre, inverse = finite && amax > 0.f ? 1.f / a : 0.f, to127 = 127.f * pre;
    if (tid == 0) scales[blockIdx.x] = finite ? amax / 127.f : __builtin_nanf("");
    uint2* out = reinterpret_cast<uint2*>(xq + (size_t)blockIdx.x * padded);
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
        if (tid + u * kQuantThreads < pieces) put(tid + u * kQuantThreads, kept[u]);
    for (int i = tid + kQuantPieces * kQuantThreads; i < pieces; i += kQuantThreads) put(i, load(i));
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

// A block of channels and NX blocks of rows per workgroup; the waves take K's steps in turn.
template <typename E, int NX>
__global__ __launch_bounds__(512) void int8_linear_kernel(LinearParams p) {
    __shared__ i32x4 part[8][NX][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t0 = blockIdx.y * NX * 16;
    const int8_t* w = p.w + (size_t)blockIdx.x * p.steps * kTile + lane * 16;
    const int8_t* x[NX];
#pragma unroll
    for (int b = 0; b < NX; ++b) x[b] = p.xq + (size_t)min(t0 + b * 16 + (lane & 15), p.n - 1) * p.steps * kStep + (lane >> 4) * 16;
    i32x4 acc[NX] = {};
    for (int s = wave; s < p.steps; s += 8) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(w + (size_t)s * kTile);
#pragma unroll
        for (int b = 0; b < NX; ++b)
            acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *reinterpret_cast<const i32x4*>(x[b] + (size_t)s * kStep), acc[b], 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < NX; ++b) part[wave][b][lane] = acc[b];
    __syncthreads();
    for (int b = wave; b < NX; b += 8) {
        i32x4 sum = part[0][b][lane];
#pragma unroll
        for (int k = 1; k < 8; ++k) sum += part[k][b][lane];
        store_quad<E>(p, t0 + b * 16 + (lane & 15), blockIdx.x * kBlock + (lane >> 4) * 4, sum);
    }
}

// Tiles of (WX NX) x (WV NV) blocks for more rows: WX x WV waves, each with NX x NV of the blocks in its accumulators.
// Rows go to LDS by direct loads, in operand order (a block's step is 1 KB, read back without bank conflicts), kAhead steps in advance
// in a ring of kStages; weights lie in operand order already and go straight into registers, two steps in advance, so that LDS
// is read for the rows alone.  The loads are numbered as they return: waiting for the weights of step s (which the compiler does, in front of their
// first use) waits for every request in front of them, among them the rows of step s + 1; the wait in front of the barrier says so.
constexpr int kStages = 4;
constexpr int kAhead = kStages - 1;

template <typename E, int NX, int NV, int WX, int WV>
__global__ __launch_bounds__(64 * WX * WV, 2) void int8_linear_tile_kernel(LinearParams p) {
    constexpr int kWaves = WX * WV, kBlocks = WX * NX, kLoads = kBlocks / kWaves;
    static_assert(kBlocks % kWaves == 0, "every wave requests as many blocks of rows");
    __shared__ __attribute__((aligned(16))) int8_t ring[kStages][kBlocks][kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wx = wave / WV, wv = wave % WV;
    int tx, tv;
    tile_of(p, blockIdx.x, &tx, &tv);
    const int t0 = tx * kBlocks * 16, b0 = (tv * WV + wv) * NV, last = p.steps - 1;
    const int8_t* row[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) row[j] = p.xq + (size_t)min(t0 + (wave * kLoads + j) * 16 + (lane & 15), p.n - 1) * p.steps * kStep + (lane >> 4) * 16;
    const int8_t* w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = p.w + (size_t)min(b0 + v, p.blocks - 1) * p.steps * kTile + lane * 16;
    const auto request = [&](int s) {
        const size_t at = (size_t)min(s, last) * kStep;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&ring[s % kStages][wave * kLoads + j][0]);
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(row[j] + at), "s"(dst) : "memory", "m0");
        }
    };
    const auto weights = [&](int s, i32x4* a) {
#pragma unroll
        for (int v = 0; v < NV; ++v) a[v] = *reinterpret_cast<const i32x4*>(w[v] + (size_t)min(s, last) * kTile);
    };
    i32x4 acc[NX][NV] = {};
    const auto step = [&](int s, const i32x4* now, i32x4* next) {
        request(s + kAhead);
        weights(s + 2, next);
        const int8_t* x = &ring[s % kStages][wx * NX][0] + lane * 16;
#pragma unroll
        for (int b = 0; b < NX; ++b) {
            const i32x4 rows = *reinterpret_cast<const i32x4*>(x + b * kTile);
#pragma unroll
            for (int v = 0; v < NV; ++v) acc[b][v] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[v], rows, acc[b][v], 0, 0, 0);
        }
        // this step's rows are read, the next one's are there: behind them two steps' requests at most
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(2 * (kLoads + NV)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
    };
    i32x4 a0[NV], a1[NV], a2[NV];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) request(s);
    weights(0, a0);
    weights(1, a1);
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    for (int s = 0; s < p.steps; s += 3) {
        step(s, a0, a2);
        if (s + 1 < p.steps) step(s + 1, a1, a0);
        if (s + 2 < p.steps) step(s + 2, a2, a1);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (requests beyond the last step write to LDS, too)
#pragma unroll
    for (int b = 0; b < NX; ++b)
#pragma unroll
        for (int v = 0; v < NV; ++v) store_quad<E>(p, t0 + (wx * NX + b) * 16 + (lane & 15), (b0 + v) * kBlock + (lane >> 4) * 4, acc[b][v]);
}

}  // namespace
}  // namespace cpmcu

using namespace cpmcu;

extern "C" int cpmcu_quantize_rows(const void* x, int64_t x_stride, int n, int K, int8_t* xq, float* scales, void* stream) {
    CPMCU_CHECK_ARG(x && xq && scales, "quantize_rows: null pointer argument");
    CPMCU_CHECK_ARG(n >= 0 && K >= 1 && K <= kMaxColumns, "quantize_rows: n=%d, K=%d outside [1, %d]", n, K, kMaxColumns);
    CPMCU_CHECK_ARG(x_stride >= K, "quantize_rows: rows closer than their %d values", K);
    CPMCU_CHECK_ARG((uintptr_t)xq % 16 == 0, "quantize_rows: xq has to lie on 16 bytes");
    if (n == 0) return CPMCU_OK;
    const bool wide = (uintptr_t)x % 16 == 0 && x_stride % 8 == 0 && K % 8 == 0;
    const int padded = ceil_div(K, kStep) * kStep;
    hipStream_t st = resolve_stream(stream);
#define CPMCU_QUANT(E) hipLaunchKernelGGL((wide ? quantize_rows_kernel<E, true> : quantize_rows_kernel<E, false>), dim3(n), dim3(kQuantThreads), 0, st, (const E*)x, (long)x_stride, K, padded, xq, scales)
    if (options().dtype == 1) CPMCU_QUANT(bf16);
    else CPMCU_QUANT(f16);
#undef CPMCU_QUANT
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}

extern "C" size_t cpmcu_int8_weight_bytes(int V, int K) {
    if (V < 1 || K < 1) return 0;
    return (size_t)ceil_div(V, kBlock) * ceil_div(K, kStep) * kTile;
}

extern "C" int cpmcu_int8_weight_tile(const int8_t* w, int V, int K, int8_t* w_tiled, void* stream) {
    CPMCU_CHECK_ARG(w && w_tiled && (const void*)w != (const void*)w_tiled, "int8_weight_tile: null or aliased pointer argument");
    CPMCU_CHECK_ARG(V >= 1 && K >= 1 && K <= kMaxColumns, "int8_weight_tile: V=%d, K=%d outside [1, %d]", V, K, kMaxColumns);
    CPMCU_CHECK_ARG((uintptr_t)w_tiled % 16 == 0, "int8_weight_tile: w_tiled has to lie on 16 bytes");
    const bool wide = (uintptr_t)w % 16 == 0 && K % 16 == 0;
    const int steps = ceil_div(K, kStep);
    const dim3 grid(std::min(ceil_div(V, kBlock), 1 << 20), ceil_div(steps, 4));
    hipLaunchKernelGGL(wide ? int8_weight_tile_kernel<true> : int8_weight_tile_kernel<false>, grid, dim3(256), 0, resolve_stream(stream), w, V, K, steps, w_tiled);
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}

extern "C" int cpmcu_int8_linear(const int8_t* xq, const float* x_scales, const int8_t* w_tiled, const float* w_scales, int n, int V, int K, void* out,
                                 void* stream) {
    CPMCU_CHECK_ARG(xq && x_scales && w_tiled && w_scales && out, "int8_linear: null pointer argument");
    CPMCU_CHECK_ARG(n >= 0 && V >= 1 && K >= 1 && K <= kMaxColumns, "int8_linear: n=%d, V=%d, K=%d outside [1, %d]", n, V, K, kMaxColumns);
    CPMCU_CHECK_ARG(((uintptr_t)xq | (uintptr_t)w_tiled) % 16 == 0, "int8_linear: xq and w_tiled have to lie on 16 bytes");
    if (n == 0) return CPMCU_OK;
    LinearParams p{xq, w_tiled, x_scales, w_scales, out, n, V, ceil_div(K, kStep), ceil_div(V, kBlock), 0, 0, V % 4 == 0 && (uintptr_t)out % 8 == 0};
    hipStream_t st = resolve_stream(stream);
    const bool is_bf16 = options().dtype == 1;
    if (n > 64) {
#define CPMCU_TILE(E, NX, NV, WX, WV)                                                                                                   \
    do {                                                                                                                                \
        p.row_tiles = ceil_div(n, 16 * NX * WX);                                                                                        \
        p.channel_tiles = ceil_div(p.blocks, NV * WV);                                                                                  \
        hipLaunchKernelGGL((int8_linear_tile_kernel<E, NX, NV, WX, WV>), dim3(p.row_tiles * p.channel_tiles), dim3(64 * WX * WV), 0, st, p); \
    } while (0)
        if (n > 512) {
            if (is_bf16) CPMCU_TILE(bf16, 8, 4, 2, 4);
            else CPMCU_TILE(f16, 8, 4, 2, 4);
        } else {
            if (is_bf16) CPMCU_TILE(bf16, 8, 2, 1, 4);
            else CPMCU_TILE(f16, 8, 2, 1, 4);
        }
#undef CPMCU_TILE
        CPMCU_LAUNCH_CHECK();
        return CPMCU_OK;
    }
    const int nx = n <= 16 ? 1 : n <= 32 ? 2 : 4;
    const dim3 grid(p.blocks, 1);
#define CPMCU_LINEAR(E) (nx == 1 ? int8_linear_kernel<E, 1> : nx == 2 ? int8_linear_kernel<E, 2> : int8_linear_kernel<E, 4>)
    hipLaunchKernelGGL(is_bf16 ? CPMCU_LINEAR(bf16) : CPMCU_LINEAR(f16), grid, dim3(512), 0, st, p);
#undef CPMCU_LINEAR
    CPMCU_LAUNCH_CHECK();
    return CPMCU_OK;
}
