// w4.hip -- fully connected layers on 4-bit weights with a scale for every group of 32, 64 or 128 neighbours of a
// row, on MI355X (gfx950): out[b][m] = act(sum_g scale[m][g] sum_{k in g} code[m][k] x[b][k] + bias[m]), act = identity or
// GPT-2's tanh GELU, INT4 or FP4 (E2M1) codes, bf16 scales.
//
// A weight is half a byte, so at the memory's rate a CU has 40 of them for every nanosecond: the products go to the
// matrix cores (16x16x32 bf16, codes and x exact in it, float sums), also for one vector, which leaves the
// vector units half an instruction a weight to make operands of the codes.  Scales are no operand's (their product with
// a code is not exact in bf16): a group's sum is multiplied in float and added to the row's.
//
// Weights are laid out once, in the order in which lanes need them: 16 rows x 128 columns are one block of 1 KB,
// lane 16 g + r's 16 bytes of which are columns 32 j + 8 g .. + 7 of row r in dword j, so that product j is columns 32 j ..
// 32 j + 31, a group or a part of one, and a load of the block is contiguous.  (INT4: in the order from which operand()
// makes columns in theirs.)  Weights are the products' right operand, so that of a result lane 16 g + r has weight row r
// for vectors 4 g .. 4 g + 3: one scale a lane, and INT4's -8 times the vectors' sums as four neighbouring floats.  (As
// the left one: 64 vectors x 50304 x 768 15.4 us.)
//
// Vectors go through LDS: loaded directly in the operands' order, neighbouring lanes would be in different rows, and
// a load takes 64 cycles in place of 16.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fc.hpp"
#include "matrix.hpp"

namespace {

constexpr int kRows = 16, kCols = 128;         // of a block
constexpr int kBlockBytes = kRows * kCols / 2;
constexpr int kW4Waves = 8;
constexpr int kTallGroups = 256;               // workgroups: one a CU
constexpr size_t kTallLds = 152 * 1024;
constexpr int kMostRows = (1 << 28) - 32;      // workgroups of two row tiles: 2^32 threads are too many
constexpr int kMostCols = 65535;               // the grid's second side
// Where a matrix's blocks and scales lie.
struct W4Shape {
    int M, K, group, tiles, steps, groups;     // row tiles, blocks of a row tile, groups of a block
    __host__ __device__ size_t scale_bytes() const { return (size_t)32 * groups; }     // of a block
    __host__ __device__ size_t scales_at() const { return (size_t)tiles * steps * kBlockBytes; }
    __host__ __device__ size_t bytes() const { return scales_at() + (size_t)tiles * steps * scale_bytes(); }
};

bool shape_of(int M, int K, int group, W4Shape& s) {
    if (group != 32 && group != 64 && group != 128) return false;
    if (M < 1 || K < group || K % group != 0 || M > kRowMask || K > (1 << 20) || (long long)M * K >= (1ll << 40)) return false;
    s = W4Shape{M, K, group, (M + kRows - 1) / kRows, (K + kCols - 1) / kCols, kCols / group};
    return true;
}

struct W4Args {
    void* out;
    void* pre_gelu;
    const uint8_t* w;
    const uint8_t* scales;
    const uint16_t* x;
    const uint16_t* bias;
    int B, M, K, steps, gelu;
};

// A lane's scales of a block.
template <int kGroups> struct Scales {
    uint32_t w[kGroups == 4 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (kGroups == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x;
            w[1] = v.y;
        } else if constexpr (kGroups == 2) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ float of(int q) const { return q & 1 ? bf16_hi(w[q / 2]) : bf16_lo(w[q / 2]); }
};

// A block's vectors in LDS: 256 bytes a vector, 16-byte chunks turned by the vector's number, so that the lanes that read one
// chunk of 16 vectors find them in different banks.
__device__ __forceinline__ int x_at(int vec, int chunk) { return vec * 256 + ((chunk ^ (vec & 15)) << 4); }

// The products of a block, 16 rows x 16 kNT vectors, added to acc.  x(j, q): vectors' operand of product q.  INT4: the
// operand's codes are 8 too large, so -8 times the vectors goes into a group's sum too; start(j, q), if given, has it.
// kRT row tiles share the vectors' operands.
struct NoStart {};
template <bool kFp4, int kGroups, int kNT, int kRT, typename X, typename S = NoStart>
__device__ __forceinline__ void block_products(const uint4 (&w)[kRT], const Scales<kGroups> (&sc)[kRT], X&& x,
                                               F32x4 (&acc)[kRT][kNT], S start = {}) {
    constexpr int kPer = 4 / kGroups;          // products of a group
    constexpr bool kMinus = !kFp4 && std::is_same<S, NoStart>::value;
    const Bf16x8 minus8 = (Bf16x8)(__bf16)(-8.0f);
    // A product's vectors are asked for while the product before it runs (of 64 vectors the registers are missing: 16.4 us
    // in place of 14.7; 1 vector x 50304 x 768 6.7 in place of 7.5).
    constexpr bool kAhead = kNT <= 2;
    Bf16x8 v[2][kNT];
#pragma unroll
    for (int j = 0; j < (kAhead ? kNT : 0); ++j) v[0][j] = x(j, 0);
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
        F32x4 d[kRT][kNT];
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
            F32x4 d0 = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (!kFp4 && !kMinus) d0 = start(j, q);
#pragma unroll
            for (int i = 0; i < kRT; ++i) d[i][j] = d0;
        }
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
            constexpr int kLast = 3;
            const int at = q * kPer + p;
            if (kAhead && at < kLast) {
#pragma unroll
                for (int j = 0; j < kNT; ++j) v[(at + 1) & 1][j] = x(j, at + 1);
            }
            Bf16x8 op[kRT];
#pragma unroll
            for (int i = 0; i < kRT; ++i) {
                const uint32_t c[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                op[i] = operand<kFp4>(c[at]);
            }
            if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
                const Bf16x8 vec = kAhead ? v[at & 1][j] : x(j, at);
#pragma unroll
                for (int i = 0; i < kRT; ++i) {
                    if constexpr (kMinus) d[i][j] = mfma(vec, minus8, d[i][j]);
                    d[i][j] = mfma(vec, op[i], d[i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kRT; ++i) {
            const float f = sc[i].of(q);
#pragma unroll
            for (int j = 0; j < kNT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[i][j][e], f, acc[i][j][e]);
        }
    }
}

// One output through the epilogue.
template <bool kOutF32>
__device__ __forceinline__ void finish(const W4Args& a, int b, int m, float pre) {
    const size_t o = (size_t)b * a.M + m;
    if (a.pre_gelu) store_res<kOutF32>(a.pre_gelu, o, pre);
    if (a.gelu) pre = gelu_tanh(pre);
    store_res<kOutF32>(a.out, o, pre);
}

// Waves of a workgroup split the columns of kRT row tiles, for kNT tiles of 16 vectors, of which 4 kQ are there at most: four
// vectors a load, 16 lanes each, past the last one that one again.  (A load that only some calls need, behind a branch, is
// waited for before the next: 64 vectors 49 us in place of 10.)  kGroups: groups of a block.
template <bool kFp4, int kGroups, int kRT, int kNT, int kQ, bool kOutF32>
__global__ __launch_bounds__(kW4Waves * kWave) void gemv_w4_kernel(W4Args a) {
    constexpr int kPitch = kRT * kRows + 4;    // floats; spreads the banks
    constexpr int kXBytes = kNT * 16 * 256, kWaveLds = std::max(kXBytes, kNT * 16 * kPitch * 4);
    extern __shared__ __align__(16) uint8_t lds[];     // a wave's vectors of a block, then [waves][kNT * 16][kPitch] sums
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int tiles = (a.M + kRows - 1) / kRows;
    const int tile0 = blockIdx.x * kRT, b0 = blockIdx.y * 16 * kNT;
    const int s0 = (int)((long long)a.steps * wave / kW4Waves), s1 = (int)((long long)a.steps * (wave + 1) / kW4Waves);
    constexpr int kScaleBytes = 32 * kGroups;
    const uint8_t* wp[kRT];
    const uint8_t* sp[kRT];
#pragma unroll
    for (int i = 0; i < kRT; ++i) {
        const size_t block = (size_t)min(tile0 + i, tiles - 1) * a.steps;
        wp[i] = a.w + block * kBlockBytes + lane * 16;
        sp[i] = a.scales + block * kScaleBytes + col * 2 * kGroups;
    }
    struct Block {
        uint4 w[kRT];
        Scales<kGroups> sc[kRT];
        uint4 x[kQ];
    };
    auto load = [&](Block& t, int s) {
#pragma unroll
        for (int i = 0; i < kRT; ++i) {
            t.w[i] = load16(wp[i] + (size_t)s * kBlockBytes);
            t.sc[i].load(sp[i] + (size_t)s * kScaleBytes);
        }
        const int k = min(s * kCols + 8 * col, a.K - 8);
#pragma unroll
        for (int q = 0; q < kQ; ++q) t.x[q] = *reinterpret_cast<const uint4*>(a.x + (size_t)min(b0 + 4 * q + g, a.B - 1) * a.K + k);
    };
    uint8_t* const xs = lds + wave * kWaveLds;
    F32x4 acc[kRT][kNT] = {};
    Block t;
    if (s0 < s1) load(t, s0);
    for (int s = s0; s < s1; ++s) {
        const bool in = s * kCols + 8 * col < a.K;     // what is past the row's end is zero
        lds_order();
#pragma unroll
        for (int q = 0; q < kQ; ++q) *reinterpret_cast<uint4*>(xs + x_at(4 * q + g, col)) = in ? t.x[q] : make_uint4(0, 0, 0, 0);
        lds_order();
        uint4 w[kRT];
        Scales<kGroups> sc[kRT];
#pragma unroll
        for (int i = 0; i < kRT; ++i) {
            w[i] = t.w[i];
            sc[i] = t.sc[i];
        }
        if (s + 1 < s1) load(t, s + 1);
        auto x_of = [&](int j, int q) { return *reinterpret_cast<const Bf16x8*>(xs + x_at(16 * j + col, 4 * q + g)); };
        block_products<kFp4, kGroups, kNT, kRT>(w, sc, x_of, acc);
        lds_order();
    }
    // Lane 16 g + c holds weight row c for vectors 4 g .. 4 g + 3.
    lds_order();
#pragma unroll
    for (int i = 0; i < kRT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<float*>(xs)[(16 * j + 4 * g + e) * kPitch + 16 * i + col] = acc[i][j][e];
    __syncthreads();
    for (int e = threadIdx.x; e < kRT * kRows * kNT * 16; e += kW4Waves * kWave) {
        const int mm = e % (kRT * kRows), bb = e / (kRT * kRows), m = tile0 * kRows + mm, b = b0 + bb;
        if (m >= a.M || b >= a.B) continue;
        float v[kW4Waves];
#pragma unroll
        for (int w = 0; w < kW4Waves; ++w) v[w] = reinterpret_cast<const float*>(lds + w * kWaveLds)[bb * kPitch + mm];
#pragma unroll
        for (int d = 1; d < kW4Waves; d *= 2)
#pragma unroll
            for (int w = 0; w + d < kW4Waves; w += 2 * d) v[w] += v[w + d];
        finish<kOutF32>(a, b, m, v[0] + (a.bias ? bf16_to_f32(a.bias[m]) : 0.0f));
    }
}

// Tall matrices: a workgroup, one a CU, keeps its 16 kNT vectors in LDS for their whole length, and each of its waves takes
// whole row tiles, with no sum across waves.  INT4: -8 times the vectors' sums over every group are made once, too.
// (Two row tiles a wave, of half as many waves: the same time.)
constexpr int kTallW4Waves = 16, kTallW4Steps = 3;     // blocks of a load, two of which are in flight
template <bool kFp4, int kGroups, int kNT, bool kOutF32>
__global__ __launch_bounds__(kTallW4Waves * kWave) void gemv_w4_tall_kernel(W4Args a, int groups) {
    constexpr int kT = kTallW4Steps, kWaves = kTallW4Waves, kScaleBytes = 32 * kGroups;
    extern __shared__ __align__(16) uint8_t lds[];     // [steps][kNT * 16][256], then [steps * kGroups][kNT * 16] floats
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int tiles = (a.M + kRows - 1) / kRows;
    const int grp = blockIdx.x, b0 = blockIdx.y * 16 * kNT;
    const int tile0 = (int)((long long)tiles * grp / groups), tile1 = (int)((long long)tiles * (grp + 1) / groups);
    float* const sums = reinterpret_cast<float*>(lds + (size_t)a.steps * kNT * 16 * 256);
    struct Block {
        uint4 w[kT][1];
        Scales<kGroups> sc[kT][1];
    };
    const int chunks = (a.steps + kT - 1) / kT;
    int ltile = tile0 + wave, lchunk = 0;              // what is loaded next
    auto next = [&](Block& t) {
        if (ltile >= tile1) return false;
#pragma unroll
        for (int u = 0; u < kT; ++u) {
            const int s = min(lchunk * kT + u, a.steps - 1);
            const size_t block = (size_t)ltile * a.steps + s;
            t.w[u][0] = load16(a.w + block * kBlockBytes + lane * 16);
            t.sc[u][0].load(a.scales + block * kScaleBytes + col * 2 * kGroups);
        }
        if (++lchunk == chunks) {
            lchunk = 0;
            ltile += kWaves;
        }
        return true;
    };
    Block t0, t1;
    const bool busy = next(t0);
    bool more = next(t1);
    // Vectors to LDS, four a load.
    const int quads = min(4 * kNT, (min(a.B - b0, 16 * kNT) + 3) / 4), pieces = a.steps * quads;
    constexpr int kAhead = 6;
    for (int i0 = wave; i0 < pieces; i0 += kWaves * kAhead) {
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = min(i0 + k * kWaves, pieces - 1), s = i / quads, q = i - s * quads;
            v[k] = *reinterpret_cast<const uint4*>(a.x + (size_t)min(b0 + 4 * q + g, a.B - 1) * a.K + min(s * kCols + 8 * col, a.K - 8));
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kWaves;
            if (i >= pieces) break;
            const int s = i / quads, q = i - s * quads;
            *reinterpret_cast<uint4*>(lds + (size_t)s * kNT * 16 * 256 + x_at(4 * q + g, col)) =
                s * kCols + 8 * col < a.K ? v[k] : make_uint4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    auto x_of = [&](int s, int j, int q) {
        return *reinterpret_cast<const Bf16x8*>(lds + (size_t)s * kNT * 16 * 256 + x_at(16 * j + col, 4 * q + g));
    };
    if constexpr (!kFp4) {
        const F32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        const Bf16x8 minus8 = (Bf16x8)(__bf16)(-8.0f);
        for (int i = wave; i < a.steps * kNT; i += kWaves) {
            const int s = i / kNT, j = i - s * kNT;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                F32x4 d = zero;
#pragma unroll
                for (int p = 0; p < 4 / kGroups; ++p) d = mfma(x_of(s, j, q * (4 / kGroups) + p), minus8, d);
                if (col == 0) *reinterpret_cast<F32x4*>(sums + ((s * kGroups + q) * kNT + j) * 16 + 4 * g) = d;
            }
        }
        __syncthreads();
    }
    if (!busy) return;
    int tile = tile0 + wave, chunk = 0;                // what is worked on
    F32x4 acc[1][kNT] = {};
    auto consume = [&](const Block& t) {
#pragma unroll
        for (int u = 0; u < kT; ++u) {
            const int s = chunk * kT + u;
            if (s >= a.steps) break;
            block_products<kFp4, kGroups, kNT, 1>(t.w[u], t.sc[u], [&](int j, int q) { return x_of(s, j, q); }, acc, [&](int j, int q) {
                return *reinterpret_cast<const F32x4*>(sums + ((s * kGroups + q) * kNT + j) * 16 + 4 * g);
            });
        }
        if (++chunk < chunks) return;
        const int m = tile * kRows + col;
        const float bias = a.bias ? bf16_to_f32(a.bias[min(m, a.M - 1)]) : 0.0f;
        const int left = m < a.M ? a.B - b0 - 4 * g : 0;       // vectors from this lane's first on
        if (a.gelu || a.pre_gelu) {
#pragma unroll
            for (int j = 0; j < kNT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * j + e < left) finish<kOutF32>(a, b0 + 16 * j + 4 * g + e, m, acc[0][j][e] + bias);
        } else {
            size_t o = (size_t)(b0 + 4 * g) * a.M + m;
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * j + e < left) store_res<kOutF32>(a.out, o + (size_t)e * a.M, acc[0][j][e] + bias);
                o += (size_t)16 * a.M;
            }
        }
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[0][j] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
        chunk = 0;
        tile += kWaves;
    };
    while (true) {
        consume(t0);
        if (!more) break;
        more = next(t0);
        consume(t1);
        if (!more) break;
        more = next(t1);
    }
}

template <bool kFp4, int kGroups, int kNT, bool kOutF32>
const void* kernel_for(int row_tiles, int B) {
    if (row_tiles == 0) return (const void*)&gemv_w4_tall_kernel<kFp4, kGroups, kNT, kOutF32>;
    if (kNT == 1 && B <= 4) {
        return row_tiles == 1 ? (const void*)&gemv_w4_kernel<kFp4, kGroups, 1, kNT, 1, kOutF32>
                              : (const void*)&gemv_w4_kernel<kFp4, kGroups, 2, kNT, 1, kOutF32>;
    }
    return row_tiles == 1 ? (const void*)&gemv_w4_kernel<kFp4, kGroups, 1, kNT, 4 * kNT, kOutF32>
                          : (const void*)&gemv_w4_kernel<kFp4, kGroups, 2, kNT, 4 * kNT, kOutF32>;
}
template <bool kFp4, int kGroups, int kNT>
const void* kernel_for(int row_tiles, int B, bool out_f32) {
    return out_f32 ? kernel_for<kFp4, kGroups, kNT, true>(row_tiles, B) : kernel_for<kFp4, kGroups, kNT, false>(row_tiles, B);
}
template <int kNT>
const void* kernel_for(bool fp4, int groups, int row_tiles, int B, bool out_f32) {
    if (fp4)
        return groups == 4 ? kernel_for<true, 4, kNT>(row_tiles, B, out_f32)
                           : groups == 2 ? kernel_for<true, 2, kNT>(row_tiles, B, out_f32) : kernel_for<true, 1, kNT>(row_tiles, B, out_f32);
    return groups == 4 ? kernel_for<false, 4, kNT>(row_tiles, B, out_f32)
                       : groups == 2 ? kernel_for<false, 2, kNT>(row_tiles, B, out_f32) : kernel_for<false, 1, kNT>(row_tiles, B, out_f32);
}

// ------------------------------------------------------------------------------------
// Laying weights out.
// ------------------------------------------------------------------------------------
// The dword of row m's columns k .. k + 7, and the scale of its group, in the layout.
__device__ __forceinline__ size_t dword_at(const W4Shape& s, int m, int k) {
    const size_t block = (size_t)(m / kRows) * s.steps + k / kCols;
    const int in = k % kCols, j = in / 32, g = in % 32 / 8;
    return block * (kBlockBytes / 4) + (16 * g + m % kRows) * 4 + j;
}
__device__ __forceinline__ size_t scale_at(const W4Shape& s, int m, int k) {
    const size_t block = (size_t)(m / kRows) * s.steps + k / kCols;
    return block * (kRows * s.groups) + (m % kRows) * s.groups + k % kCols / s.group;
}

// Eight codes, the first in the lowest half byte, in the order that operand() takes.
__device__ __forceinline__ uint32_t in_layout(uint32_t w, bool int4) {
    if (!int4) return w;
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o |= ((w >> (4 * i)) & 15u) << (8 * i) | ((w >> (16 + 4 * i)) & 15u) << (8 * i + 4);
    return o;
}

// A thread for every dword of the layout; what is behind the matrix's end is zero.
__global__ __launch_bounds__(256) void pack_w4_kernel(uint32_t* w4, uint16_t* out_scales, const uint32_t* codes, const uint16_t* scales,
                                                      W4Shape s, int int4) {
    const long long words = (long long)s.tiles * kRows * s.steps * (kCols / 8);
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < words; e += (long long)gridDim.x * 256) {
        const int per = s.steps * (kCols / 8), m = (int)(e / per), k = (int)(e - (long long)m * per) * 8;
        const bool in = m < s.M && k < s.K;
        w4[dword_at(s, m, k)] = in_layout(in ? codes[((size_t)m * s.K + k) / 8] : int4 ? 0x88888888u : 0u, int4);
        if (k % s.group == 0) out_scales[scale_at(s, m, k)] = in ? scales[(size_t)m * (s.K / s.group) + k / s.group] : 0;
    }
}

// A thread for every group: its scale from its largest magnitude, then its codes.
template <bool kSrcF32, bool kFp4>
__global__ __launch_bounds__(256) void quantize_w4_kernel(uint32_t* w4, uint16_t* out_scales, const void* W, W4Shape s) {
    const int per = s.steps * s.groups;
    const long long all = (long long)s.tiles * kRows * per;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
        const int m = (int)(e / per), k0 = (int)(e - (long long)m * per) * s.group;
        const bool in = m < s.M && k0 < s.K;
        const size_t from = (size_t)m * s.K + k0;
        auto value = [&](int i) {
            if constexpr (kSrcF32) return reinterpret_cast<const float*>(W)[from + i];
            else return bf16_to_f32(reinterpret_cast<const uint16_t*>(W)[from + i]);
        };
        float amax = 0.0f;
        for (int i = 0; i < (in ? s.group : 0); ++i) amax = fmaxf(amax, fabsf(value(i)));
        const uint16_t bits = f32_to_bf16(amax / (kFp4 ? 6.0f : 7.0f));
        const float scale = bf16_to_f32(bits);
        out_scales[scale_at(s, m, k0)] = bits;
        for (int i0 = 0; i0 < s.group; i0 += 8) {
            uint32_t w = 0;
            for (int i = 0; i < 8; ++i) {
                float y = in && scale > 0.0f ? value(i0 + i) / scale : 0.0f;
                y = y == y ? y : 0.0f;
                uint32_t c;
                if constexpr (kFp4) {
                    const float v = fabsf(y);              // to nearest, ties to the even code
                    c = (v > 0.25f) + (v >= 0.75f) + (v > 1.25f) + (v >= 1.75f) + (v > 2.5f) + (v >= 3.5f) + (v > 5.0f);
                    c |= (__float_as_uint(y) >> 28) & 8u;
                } else {
                    c = (uint32_t)((int)fminf(fmaxf(rintf(y), -7.0f), 7.0f) + 8);
                }
                w |= c << (4 * i);
            }
            w4[dword_at(s, m, k0 + i0)] = in_layout(w, !kFp4);
        }
    }
}

int hip_status(hipError_t e) {
    if (e == hipSuccess) return KVATTN_OK;
    kvattn_internal::set_last_hip_error((int)e);
    return KVATTN_ERR_HIP;
}

bool is_4bit(int dt) { return dt == KVATTN_KV_INT4 || dt == KVATTN_KV_FP4_E2M1; }

}  // namespace

extern "C" {

size_t kvattn_w4_bytes(int M, int K, int group) {
    W4Shape s;
    return shape_of(M, K, group, s) ? s.bytes() : 0;
}

int kvattn_w4_pack(void* w4, const void* codes, const void* scales, int M, int K, int group, int w_dtype, void* stream) {
    W4Shape s;
    if (!is_4bit(w_dtype)) return KVATTN_ERR_DTYPE;
    if (!shape_of(M, K, group, s)) return KVATTN_ERR_SHAPE;
    if (!w4 || !codes || !scales) return KVATTN_ERR_NULL_POINTER;
    if (((uintptr_t)w4 & 15u) || ((uintptr_t)codes & 15u) || ((uintptr_t)scales & 1u)) return KVATTN_ERR_MISALIGNED;
    int int4 = w_dtype == KVATTN_KV_INT4;
    uint8_t* sc = (uint8_t*)w4 + s.scales_at();
    const long long words = (long long)s.tiles * kRows * s.steps * (kCols / 8);
    void* params[] = {&w4, &sc, &codes, &scales, &s, &int4};
    return hip_status(hipLaunchKernel((const void*)&pack_w4_kernel, dim3((unsigned)std::min<long long>((words + 255) / 256, 1 << 20)),
                                      dim3(256), params, 0, (hipStream_t)stream));
}

int kvattn_w4_quantize(void* w4, const void* W, int M, int K, int group, int src_dtype, int w_dtype, void* stream) {
    W4Shape s;
    if (!is_4bit(w_dtype) || (src_dtype != KVATTN_KV_F32 && src_dtype != KVATTN_KV_BF16)) return KVATTN_ERR_DTYPE;
    if (!shape_of(M, K, group, s)) return KVATTN_ERR_SHAPE;
    if (!w4 || !W) return KVATTN_ERR_NULL_POINTER;
    if (((uintptr_t)w4 & 15u) || ((uintptr_t)W % (src_dtype == KVATTN_KV_F32 ? 4 : 2))) return KVATTN_ERR_MISALIGNED;
    uint8_t* sc = (uint8_t*)w4 + s.scales_at();
    const bool fp4 = w_dtype == KVATTN_KV_FP4_E2M1;
    const void* fn = src_dtype == KVATTN_KV_F32 ? (fp4 ? (const void*)&quantize_w4_kernel<true, true> : (const void*)&quantize_w4_kernel<true, false>)
                                                : (fp4 ? (const void*)&quantize_w4_kernel<false, true> : (const void*)&quantize_w4_kernel<false, false>);
    const long long all = (long long)s.tiles * kRows * s.steps * s.groups;
    void* params[] = {&w4, &sc, &W, &s};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)std::min<long long>((all + 255) / 256, 1 << 20)), dim3(256), params, 0, (hipStream_t)stream));
}

int kvattn_gemv_w4(void* out, void* pre_gelu, const void* w4, const void* x, const void* bias, int B, int M, int K, int group,
                   int w_dtype, int out_dtype, int gelu, void* stream) {
    W4Shape s;
    if (!is_4bit(w_dtype) || (out_dtype != KVATTN_KV_F32 && out_dtype != KVATTN_KV_BF16)) return KVATTN_ERR_DTYPE;
    if (!shape_of(M, K, group, s)) return KVATTN_ERR_SHAPE;
    if (B < 1 || M > kMostRows || (long long)B * M >= (1ll << 31) || (long long)B * K >= (1ll << 31)) return KVATTN_ERR_SHAPE;
    if (!out || !w4 || !x) return KVATTN_ERR_NULL_POINTER;
    const size_t osz = out_dtype == KVATTN_KV_F32 ? 4 : 2;
    if (((uintptr_t)w4 & 15u) || ((uintptr_t)x & 15u) || ((uintptr_t)out % osz) || ((uintptr_t)pre_gelu % osz) || ((uintptr_t)bias & 1u))
        return KVATTN_ERR_MISALIGNED;
    W4Args a{out, pre_gelu, (const uint8_t*)w4, (const uint8_t*)w4 + s.scales_at(), (const uint16_t*)x, (const uint16_t*)bias,
             B, M, K, s.steps, gelu ? 1 : 0};
    const bool fp4 = w_dtype == KVATTN_KV_FP4_E2M1, f32 = out_dtype == KVATTN_KV_F32;
    int nt = B <= 16 ? 1 : B <= 32 ? 2 : 4;
    auto x_lds = [&](int n) { return (size_t)s.steps * n * 16 * (256 + 4 * s.groups); };
    // us per call (graph), INT4, groups of 64, one / two row tiles a workgroup / vectors in LDS for their whole length:
    //   vectors       6400 x 1600         12000 x 768        20000 x 1600         32000 x 1600         50304 x 768         50304 x 1600
    //    1         3.7 / 3.8 / 7.5    3.6 / 3.7 / 5.0     5.8 / 6.0 / 9.2     8.2 / 7.2 / 9.5    7.8 / 8.1 / 7.1    11.9 / 11.3 / 12.1
    //   16         4.2 / 4.1 / 8.1    4.8 / 4.1 / 6.1     8.2 / 7.0 / 9.8    12.6 / 9.5 / 10.2  11.5 / 9.4 / 8.1    19.1 / 15.0 / 13.1
    //   32         5.7 / 5.4 / 10.5   5.8 / 7.0 / 7.2    11.9 / 12.9 / 12.3  19.1 / 17.9 / 12.9 19.1 / 21.1 / 10.1  29.5 / 29.9 / 16.4
    //   64        12.0 / 8.8          12.1 / 11.2 / 10.7  30.1 / 24.1         49.6 / 32.7        50.7 / 36.4 / 14.0  81.0 / 56.0
    // Two row tiles halve the vectors' loads, where workgroups for the GPU are left.  Of 32 vectors 512 row tiles run at once
    // either way, and a last round that is less than half full is shorter with one; of 64 vectors 256 and 512 run at once.
    // Vectors in LDS pay where a matrix is tall, the more the vectors (their filling: one vector over long rows never);
    // 64 that do not fit go in two halves (64 x 32000 x 1600 23.7 us).  FP4 and groups of 32 go by the same borders: at these
    // sizes within 5 % of the fastest of the three, but for INT4 in groups of 32 at 1 x 50304 x 768 (7.7, two row tiles 6.8) and
    // 32 x 20000 x 1600 (13.8, one row tile 12.2).
    const long long work = (long long)s.tiles * ((B + 16 * nt - 1) / (16 * nt)), last = work % 512;
    int row_tiles = 1;
    if (nt == 1) row_tiles = work >= (B <= 4 ? 512 : 320) ? 2 : 1;
    else if (nt == 2) row_tiles = work >= 320 && (last == 0 || last >= 320) ? 2 : 1;
    else row_tiles = work > 256 ? 2 : 1;
    const int tall = nt == 1 ? (B <= 4 && K > 1024 ? kRowMask : 2400) : nt == 2 ? 1250 : B <= 64 ? 513 : 1024;
    if (s.tiles >= tall && x_lds(nt) <= kTallLds) {
        row_tiles = 0;
    } else if (nt == 4 && s.tiles >= 1536 && x_lds(2) <= kTallLds) {
        nt = 2;
        row_tiles = 0;
    }
    const void* fn = nt == 1 ? kernel_for<1>(fp4, s.groups, row_tiles, B, f32)
                             : nt == 2 ? kernel_for<2>(fp4, s.groups, row_tiles, B, f32) : kernel_for<4>(fp4, s.groups, row_tiles, B, f32);
    int groups = kTallGroups;
    const int grid = row_tiles ? (s.tiles + row_tiles - 1) / row_tiles : groups, waves = row_tiles ? kW4Waves : kTallW4Waves;
    const size_t lds = row_tiles ? (size_t)kW4Waves * nt * 16 * std::max(256, (row_tiles * kRows + 4) * 4) : x_lds(nt);
    if (lds > 64 * 1024) {
        const int st = hip_status(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (st != KVATTN_OK) return st;
    }
    void* params[] = {&a, &groups};
    // More vectors than a grid has columns for go in several launches.
    for (int b0 = 0; b0 < B; b0 += kMostCols * 16 * nt) {
        a.B = std::min(B - b0, kMostCols * 16 * nt);
        a.x = (const uint16_t*)x + (size_t)b0 * K;
        a.out = (uint8_t*)out + (size_t)b0 * M * osz;
        if (pre_gelu) a.pre_gelu = (uint8_t*)pre_gelu + (size_t)b0 * M * osz;
        const int cols = (a.B + 16 * nt - 1) / (16 * nt);
        const int st = hip_status(hipLaunchKernel(fn, dim3((unsigned)grid, (unsigned)cols), dim3(waves * kWave), params, lds, (hipStream_t)stream));
        if (st != KVATTN_OK) return st;
    }
    return KVATTN_OK;
}

}  // extern "C"
