// Products of a few rows with 4-bit weights: C[M][N] = x[M][K] . W[N][K]^T, W[n][k] = scale[n][g] * (q[n][k] - zero[n][g]), g = k / group.
// A lane's 16 bytes are 32 weights of one output column: four MFMA A fragments (16 columns x 32 k each).  A nibble q is, as an
// 8-bit float (e4m3), exactly q * 2^-9 -- the subnormals and the first binade are one linear ramp -- so one conversion with a
// scale of 512 makes two exact bf16 whole numbers.  The MFMA adds up x . q of one group in fp32, another one with an all-ones
// fragment the sum of the group's x, and the accumulator takes scale * (x.q - zero * sum x) in fp32: no weight is ever rounded.
// Bound: N K / 2 bytes of weights (plus scales and zeros) while the rows are few.
//
// Layout (the packer writes it once): k blocks of 128, columns in tiles of 16:
//   wq   [N/16][K/128][64 lanes][16 bytes]: lane l = fq * 16 + fr holds column nt * 16 + fr; its word j (0 .. 3) the weights
//        k = kb * 128 + j * 32 + fq * 8 + i, i = 0 .. 7: byte i % 4, low nibble for i < 4, high nibble for i >= 4
//   scales [N/16][groups][16] in dtype, zeros [N/16][groups][16] bytes (NULL: 8 everywhere); groups = (K/128) * (128/group)
// N and K are rounded up to whole tiles with scale 0.
#include "common.h"

struct W4Args {
    const void* x; const uint4* wq; const void* scales; const uint8_t* zeros; const void* bias; const void* resid; void* out;
    long x_rs;
    int M, N, K, KB, ldc, epi;
};

__device__ __forceinline__ bf16x8 w4_fragment(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
__device__ __forceinline__ void w4_store(const W4Args& a, int m, int n, const f32x4& v) {          // columns n .. n + 3 of row m
    if (m >= a.M) return;
    if (a.epi == VALLE_EPI_GEGLU) {
        T* c = (T*)a.out + (long)m * a.ldc;
#pragma unroll
        for (int r = 0; r < 4; r += 2)
            if (n + r < a.N) c[(n + r) >> 1] = from_f32<T>(gelu_act<T>(v[r]) * v[r + 1]);           // N is even
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= a.N) continue;
        const long at = (long)m * a.ldc + n + r;
        float y = v[r];
        if (a.epi == VALLE_EPI_F32OUT) {
            if (a.bias) y += ((const float*)a.bias)[n + r];
            ((float*)a.out)[at] = y;
        } else {
            if (a.bias) y += to_f32<T>(((const T*)a.bias)[n + r]);
            if (a.epi == VALLE_EPI_RESID) y += to_f32<T>(((const T*)a.resid)[at]);
            ((T*)a.out)[at] = from_f32<T>(y);
        }
    }
}

// One workgroup: 16 output columns x up to 16 * MT rows; its waves split the k blocks, partial sums meet in LDS in wave order.
template <typename T, int G, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void linear_w4_kernel(W4Args a) {
    constexpr int GPB = 128 / G, FPG = G / 32;                           // groups per k block, fragments per group
    const int nt = blockIdx.x, m0 = blockIdx.y * 16 * MT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const uint4* wp = a.wq + (long)nt * a.KB * 64 + lane;
    const T* sp = (const T*)a.scales + (long)nt * a.KB * GPB * 16 + fq * 4;
    const uint8_t* zp = a.zeros ? a.zeros + (long)nt * a.KB * GPB * 16 + fq * 4 : nullptr;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < a.KB; kb += NW) {
        const uint4 w4 = wp[(long)kb * 64];
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            typedef T vec4 __attribute__((ext_vector_type(4)));
            const vec4 sv = *reinterpret_cast<const vec4*>(sp + (long)(kb * GPB + g) * 16);
            const uint32_t zv = zp ? *reinterpret_cast<const uint32_t*>(zp + (long)(kb * GPB + g) * 16) : 0x08080808u;
            f32x4 xq[MT], xs[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) xq[t] = xs[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < FPG; ++f) {
                const int j = g * FPG + f, k = kb * 128 + j * 32 + fq * 8;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int m = m0 + t * 16 + fr;
                    const bool in = m < a.M && k < a.K;                  // K % 32 == 0: a lane's 8 are in or out together
                    const T* xp = (const T*)a.x + (long)m * a.x_rs + k;
                    if constexpr (sizeof(T) == 2) {
                        bf16x8 xv = {};
                        if (in) xv = *reinterpret_cast<const bf16x8*>(xp);
                        const bf16 one = (bf16)1.0f;
                        xq[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w4_fragment(w[j]), xv, xq[t], 0, 0, 0);
                        xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16x8{one, one, one, one, one, one, one, one}, xv, xs[t], 0, 0, 0);
                    } else {
                        f32x4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
                        if (in) { x0 = *reinterpret_cast<const f32x4*>(xp); x1 = *reinterpret_cast<const f32x4*>(xp + 4); }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float qv = (float)((w[j] >> ((i & 3) * 8 + (i >> 2) * 4)) & 15u), xv = i < 4 ? x0[i & 3] : x1[i & 3];
                            xq[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(qv, xv, xq[t], 0, 0, 0);
                            xs[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.0f, xv, xs[t], 0, 0, 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[t][r] += to_f32<T>(sv[r]) * (xq[t][r] - (float)((zv >> (8 * r)) & 255u) * xs[t][r]);
        }
    }
    __shared__ f32x4 part[NW][MT][64];
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 64; i += NW * 64) {
        const int t = i >> 6, l = i & 63;
        f32x4 s = part[0][t][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const f32x4 p = part[w][t][l];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] += p[r];
        }
        w4_store<T>(a, m0 + t * 16 + (l & 15), nt * 16 + (l >> 4) * 4, s);
    }
}

template <typename T, int G>
static void w4_launch(const W4Args& a, hipStream_t s) {
    const int nt = ceil_div(a.N, 16);
    if (a.M <= 16) linear_w4_kernel<T, G, 1, 8><<<dim3(nt, 1), 512, 0, s>>>(a);
    else linear_w4_kernel<T, G, 4, 8><<<dim3(nt, ceil_div(a.M, 64)), 512, 0, s>>>(a);
}
template <typename T>
static void w4_launch_group(const W4Args& a, int group, hipStream_t s) {
    if (group == 32) w4_launch<T, 32>(a, s);
    else if (group == 64) w4_launch<T, 64>(a, s);
    else w4_launch<T, 128>(a, s);
}

extern "C" int valle_linear_w4(const void* x, int64_t x_row_stride, const void* wq, const void* scales, const uint8_t* zeros, const void* bias,
                               const void* resid, void* C, int M, int N, int K, int group, int ldc, int epilogue, int dtype, void* stream) {
    VALLE_REQUIRE(x && wq && scales && C, VALLE_E_ARG, "valle_linear_w4: null pointer");
    VALLE_REQUIRE(dtype == VALLE_BF16 || dtype == VALLE_F32, VALLE_E_ARG, "valle_linear_w4: unknown dtype %d", dtype);
    VALLE_REQUIRE(group == 32 || group == 64 || group == 128, VALLE_E_UNSUPPORTED, "valle_linear_w4: group %d (32, 64 and 128 are built)", group);
    VALLE_REQUIRE(M >= 0 && N > 0 && K > 0 && K % group == 0, VALLE_E_ARG, "valle_linear_w4: M=%d N=%d K=%d (K must be a multiple of the group, %d)", M, N, K, group);
    VALLE_REQUIRE(epilogue == VALLE_EPI_STORE || epilogue == VALLE_EPI_RESID || epilogue == VALLE_EPI_GEGLU || epilogue == VALLE_EPI_F32OUT, VALLE_E_ARG,
                  "valle_linear_w4: epilogue %d is not built", epilogue);
    VALLE_REQUIRE(epilogue != VALLE_EPI_RESID || resid, VALLE_E_ARG, "valle_linear_w4: residual missing");
    VALLE_REQUIRE(epilogue != VALLE_EPI_GEGLU || (N % 2 == 0 && !bias), VALLE_E_ARG, "valle_linear_w4: EPI_GEGLU takes an even N and no bias");
    VALLE_REQUIRE(ldc >= (epilogue == VALLE_EPI_GEGLU ? N / 2 : N), VALLE_E_ARG, "valle_linear_w4: ldc %d too small", ldc);
    VALLE_REQUIRE((((uintptr_t)x | (uintptr_t)wq | (uintptr_t)scales | (uintptr_t)zeros) & 15) == 0, VALLE_E_ARG, "valle_linear_w4: operands must be 16-byte aligned");
    VALLE_REQUIRE(x_row_stride >= 0 && x_row_stride % (16 / (int)dtype_size(dtype)) == 0, VALLE_E_ARG, "valle_linear_w4: rows of x must stay 16-byte aligned");
    VALLE_REQUIRE(M <= 65535 * 64, VALLE_E_ARG, "valle_linear_w4: %d rows", M);
    if (M == 0) return VALLE_OK;
    W4Args a{x, (const uint4*)wq, scales, zeros, bias, resid, C, x_row_stride, M, N, K, ceil_div(K, 128), ldc, epilogue};
    if (dtype == VALLE_BF16) w4_launch_group<bf16>(a, group, (hipStream_t)stream);
    else w4_launch_group<float>(a, group, (hipStream_t)stream);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}
