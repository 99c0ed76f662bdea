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
// 32 j + 31, a group or a part of one, and a load of the block is contiguous.  Scales of a block lie in the order in
// which results have rows (lane 16 g + r: rows 4 g .. 4 g + 3).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fc.hpp"
#include "matrix.hpp"

namespace {

constexpr int kRows = 16, kCols = 128;         // of a block
constexpr int kBlockBytes = kRows * kCols / 2;
constexpr int kW4Waves = 8;

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

// kGroups: groups of a block; kRT, kNT: row tiles and tiles of 16 vectors of a workgroup, whose waves split the columns.
template <bool kFp4, int kGroups, int kRT, int kNT, bool kOutF32>
__global__ __launch_bounds__(kW4Waves * kWave) void gemv_w4_kernel(W4Args a) {
    constexpr int kPitch = kRT * kRows + 4;    // floats; keeps 16-byte stores aligned and spreads the banks
    extern __shared__ float red[];             // [waves][kNT * 16][kPitch]
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
        sp[i] = a.scales + block * kScaleBytes + g * 8 * kGroups;
    }
    const uint16_t* xp[kNT];
#pragma unroll
    for (int j = 0; j < kNT; ++j) xp[j] = a.x + (size_t)min(b0 + 16 * j + col, a.B - 1) * a.K + 8 * g;

    F32x4 acc[kRT][kNT] = {};
    const F32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const Bf16x8 minus8 = (Bf16x8)(__bf16)(-8.0f);
    for (int s = s0; s < s1; ++s) {
        uint4 w[kRT];
        uint2 sc[kRT][kGroups];
#pragma unroll
        for (int i = 0; i < kRT; ++i) {
            w[i] = load16(wp[i] + (size_t)s * kBlockBytes);
#pragma unroll
            for (int q = 0; q < kGroups; ++q) sc[i][q] = *reinterpret_cast<const uint2*>(sp[i] + (size_t)s * kScaleBytes + 8 * q);
        }
        Bf16x8 x[kNT][4];
        F32x4 init[kNT][kGroups];
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = s * kCols + 32 * q + 8 * g;
                uint4 v = *reinterpret_cast<const uint4*>(xp[j] + min(s * kCols + 32 * q, a.K - 32));
                if (k >= a.K) v = make_uint4(0, 0, 0, 0);
                x[j][q] = in_order<kFp4>(v);
            }
            // INT4: the operand's codes are 8 too large, so a group's sum starts at -8 times that of x.
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                init[j][q] = zero;
                if constexpr (!kFp4) {
#pragma unroll
                    for (int p = 0; p < 4 / kGroups; ++p) init[j][q] = mfma(minus8, x[j][q * (4 / kGroups) + p], init[j][q]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kRT; ++i) {
            const uint32_t c[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                F32x4 d[kNT];
#pragma unroll
                for (int j = 0; j < kNT; ++j) d[j] = init[j][q];
#pragma unroll
                for (int p = 0; p < 4 / kGroups; ++p) {
                    const int at = q * (4 / kGroups) + p;
                    const Bf16x8 op = operand<kFp4>(c[at]);
#pragma unroll
                    for (int j = 0; j < kNT; ++j) d[j] = mfma(op, x[j][at], d[j]);
                }
                const float f[4] = {bf16_lo(sc[i][q].x), bf16_hi(sc[i][q].x), bf16_lo(sc[i][q].y), bf16_hi(sc[i][q].y)};
#pragma unroll
                for (int j = 0; j < kNT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[j][e], f[e], acc[i][j][e]);
            }
        }
    }
    // Lane 16 g + c holds rows 4 g .. 4 g + 3 of vector c.
#pragma unroll
    for (int i = 0; i < kRT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j)
            *reinterpret_cast<F32x4*>(red + (size_t)((wave * kNT + j) * 16 + col) * kPitch + 16 * i + 4 * g) = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < kRT * kRows * kNT * 16; e += kW4Waves * kWave) {
        const int mm = e % (kRT * kRows), bb = e / (kRT * kRows), m = tile0 * kRows + mm, b = b0 + bb;
        if (m >= a.M || b >= a.B) continue;
        float v[kW4Waves];
#pragma unroll
        for (int w = 0; w < kW4Waves; ++w) v[w] = red[(size_t)(w * kNT * 16 + bb) * kPitch + mm];
#pragma unroll
        for (int d = 1; d < kW4Waves; d *= 2)
#pragma unroll
            for (int w = 0; w + d < kW4Waves; w += 2 * d) v[w] += v[w + d];
        float pre = v[0] + (a.bias ? bf16_to_f32(a.bias[m]) : 0.0f);
        const size_t o = (size_t)b * a.M + m;
        if (a.pre_gelu) store_res<kOutF32>(a.pre_gelu, o, pre);
        if (a.gelu) pre = gelu_tanh(pre);
        store_res<kOutF32>(a.out, o, pre);
    }
}

template <bool kFp4, int kGroups, int kRT, int kNT>
const void* kernel_for(bool out_f32) {
    return out_f32 ? (const void*)&gemv_w4_kernel<kFp4, kGroups, kRT, kNT, true> : (const void*)&gemv_w4_kernel<kFp4, kGroups, kRT, kNT, false>;
}
template <int kRT, int kNT>
const void* kernel_for(bool fp4, int groups, bool out_f32) {
    if (fp4) return groups == 4 ? kernel_for<true, 4, kRT, kNT>(out_f32) : groups == 2 ? kernel_for<true, 2, kRT, kNT>(out_f32) : kernel_for<true, 1, kRT, kNT>(out_f32);
    return groups == 4 ? kernel_for<false, 4, kRT, kNT>(out_f32) : groups == 2 ? kernel_for<false, 2, kRT, kNT>(out_f32) : kernel_for<false, 1, kRT, kNT>(out_f32);
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
    const int r = m % kRows;
    return block * (16 * s.groups) + (r / 4) * 4 * s.groups + (k % kCols / s.group) * 4 + r % 4;
}

// A thread for every dword of the layout; what is behind the matrix's end is zero.
__global__ __launch_bounds__(256) void pack_w4_kernel(uint32_t* w4, uint16_t* out_scales, const uint32_t* codes, const uint16_t* scales,
                                                      W4Shape s, uint32_t none) {
    const long long words = (long long)s.tiles * kRows * s.steps * (kCols / 8);
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < words; e += (long long)gridDim.x * 256) {
        const int per = s.steps * (kCols / 8), m = (int)(e / per), k = (int)(e - (long long)m * per) * 8;
        const bool in = m < s.M && k < s.K;
        w4[dword_at(s, m, k)] = in ? codes[((size_t)m * s.K + k) / 8] : none;
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
            w4[dword_at(s, m, k0 + i0)] = w;
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
    uint32_t none = w_dtype == KVATTN_KV_INT4 ? 0x88888888u : 0u;
    uint8_t* sc = (uint8_t*)w4 + s.scales_at();
    const long long words = (long long)s.tiles * kRows * s.steps * (kCols / 8);
    void* params[] = {&w4, &sc, &codes, &scales, &s, &none};
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
    if (B < 1 || (long long)B * M >= (1ll << 31) || (long long)B * K >= (1ll << 31)) return KVATTN_ERR_SHAPE;
    if (!out || !w4 || !x) return KVATTN_ERR_NULL_POINTER;
    const size_t osz = out_dtype == KVATTN_KV_F32 ? 4 : 2;
    if (((uintptr_t)w4 & 15u) || ((uintptr_t)x & 15u) || ((uintptr_t)out % osz) || ((uintptr_t)pre_gelu % osz) || ((uintptr_t)bias & 1u))
        return KVATTN_ERR_MISALIGNED;
    W4Args a{out, pre_gelu, (const uint8_t*)w4, (const uint8_t*)w4 + s.scales_at(), (const uint16_t*)x, (const uint16_t*)bias,
             B, M, K, s.steps, gelu ? 1 : 0};
    const bool fp4 = w_dtype == KVATTN_KV_FP4_E2M1, f32 = out_dtype == KVATTN_KV_F32;
    const int nt = B <= 16 ? 1 : B <= 32 ? 2 : 4;
    const void* fn = nt == 1 ? kernel_for<1, 1>(fp4, s.groups, f32) : nt == 2 ? kernel_for<1, 2>(fp4, s.groups, f32) : kernel_for<1, 4>(fp4, s.groups, f32);
    const long long cols = (B + 16 * nt - 1) / (16 * nt);
    if (cols > 65535) return KVATTN_ERR_SHAPE;
    const size_t lds = (size_t)kW4Waves * nt * 16 * (kRows + 4) * sizeof(float);
    void* params[] = {&a};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)s.tiles, (unsigned)cols), dim3(kW4Waves * kWave), params, lds, (hipStream_t)stream));
}

}  // extern "C"
