// Products of a few rows with 4-bit weights: C[M][N] = x[M][K] . W[N][K]^T, W[n][k] = scale[n][g] * (q[n][k] - zero[n][g]), g = k / group.
// A lane's 16 bytes are 32 weights of one output column: four MFMA A fragments (16 columns x 32 k each).  A nibble q is, as an
// 8-bit float (e4m3), exactly q * 2^-9 -- the subnormals and the first binade are one linear ramp -- so one conversion with a
// scale of 512 makes two exact bf16 whole numbers.  The MFMA adds up x . q of one group in fp32, another one with an all-ones
// fragment the sum of the group's x, and the accumulator takes scale * (x.q - zero * sum x) in fp32: no weight is ever rounded.
// Bound: N K / 2 bytes of weights (plus scales and zeros) while the rows are few: 8192 -> 8192, group 128 (36 MB), 1 / 16 rows 9.5 / 9.9 us
// = 3.7 TB/s; every row tile of 16 more costs 4 us (32 rows 13.5, 40 rows 16.5, 64 rows 21.4): x passes through every CU whole and the row sums
// are computed by every workgroup (40 rows took 16.9 when they took 11.0 without x and 14.9 without the sums).  There the vector unit issues in
// 0.41 of a busy CU's cycles, the matrix unit works in 0.26, waves wait in 0.32 of theirs.  Small layers are a launch and two round trips:
// 1024 -> 1024 3.1, 1024 -> 8192 3.5.  (us here and at the choices below: graph replays on the same inputs, both sides in one run.)
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

__device__ __forceinline__ uint32_t w4_word(const uint4& w, int j) { return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w; }
__device__ __forceinline__ float w4_value(uint32_t w, int i) {           // weight i of a word: v_cvt_f32_ubyte of one byte
    return (float)((((i < 4 ? w : w >> 4) & 0x0f0f0f0fu) >> ((i & 3) * 8)) & 255u);
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

// ---- the bf16 form.  A wave owns NT column tiles x MT row tiles and every NW-th k block.  x goes from L2 straight into the wave's own
// LDS (no registers, no writes on the way; through registers 18.0 instead of 16.4 us at 8192 -> 8192, 40 rows), a ring of NS stages: a whole
// k block up to two row tiles, half of one beyond (a fragment at a time, more of them under way: 18.2 us; every stage costs its reads' latency).
// NS - 1 stages are always under way, and the next block's weights (two blocks' weights: 16.8 us, and 9.9 for 9.4 at one row).  A
// load is 16 rows x 64 bytes, four lanes to a row (a row per lane, as the fragments have it, runs at a quarter of the rate), and lands as it
// comes, lane after lane; the 16-byte pieces of a row are asked for in the order c ^ (row / 2 mod 4), so that a fragment's read (eight
// rows of one piece at a time) meets no bank twice.  Partial sums of the waves meet in LDS, in wave order.
template <int GPB, int NT> struct W4Stage { uint4 w[NT]; uint2 s[GPB][NT]; uint32_t z[GPB][NT]; };

// the fragments of a stage, MT row tiles each (the compiler would wait for every load into LDS first)
__device__ __forceinline__ void w4_read(uint32_t at, bf16x8 (&x)[4][1]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[1][0]), "=&v"(x[2][0]), "=&v"(x[3][0]) : "v"(at), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10) : "memory");
}
__device__ __forceinline__ void w4_read(uint32_t at, bf16x8 (&x)[4][2]) {
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:%9\n\tds_read_b128 %2, %8 offset:%10\n\tds_read_b128 %3, %8 offset:%11\n\t"
                 "ds_read_b128 %4, %8 offset:%12\n\tds_read_b128 %5, %8 offset:%13\n\tds_read_b128 %6, %8 offset:%14\n\tds_read_b128 %7, %8 offset:%15\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[2][0]), "=&v"(x[2][1]), "=&v"(x[3][0]), "=&v"(x[3][1])
                 : "v"(at), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10), "n"(4 << 10), "n"(5 << 10), "n"(6 << 10), "n"(7 << 10) : "memory");
}
__device__ __forceinline__ void w4_read(uint32_t at, bf16x8 (&x)[2][3]) {
    asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:%7\n\tds_read_b128 %2, %6 offset:%8\n\tds_read_b128 %3, %6 offset:%9\n\t"
                 "ds_read_b128 %4, %6 offset:%10\n\tds_read_b128 %5, %6 offset:%11\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[1][2])
                 : "v"(at), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10), "n"(4 << 10), "n"(5 << 10) : "memory");
}

__device__ __forceinline__ void w4_read(uint32_t at, bf16x8 (&x)[2][4]) {
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:%9\n\tds_read_b128 %2, %8 offset:%10\n\tds_read_b128 %3, %8 offset:%11\n\t"
                 "ds_read_b128 %4, %8 offset:%12\n\tds_read_b128 %5, %8 offset:%13\n\tds_read_b128 %6, %8 offset:%14\n\tds_read_b128 %7, %8 offset:%15\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[1][2]), "=&v"(x[1][3])
                 : "v"(at), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10), "n"(4 << 10), "n"(5 << 10), "n"(6 << 10), "n"(7 << 10) : "memory");
}

template <int G, int NT, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void linear_w4_kernel(W4Args a) {
    constexpr int GPB = 128 / G, FPG = G / 32;                           // groups per k block, fragments per group
    constexpr int SF = MT <= 2 ? 4 : 2, STEPS = 4 / SF;                  // fragments per stage, stages per block
    constexpr int NS = MT == 3 ? 3 : 2, STAGE = SF * MT * 1024;          // bytes of a stage
    // Loads younger than a stage's own, which may be under way while it is multiplied: NS - 1 stages, and the next block's weights unless
    // the stage was asked for behind them (they are asked for with a block's first stage)
    constexpr int AHEAD = (NS - 1) * SF * MT, WEIGHTS = NT * (1 + 2 * GPB);
    const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT, tiles = (a.N + 15) >> 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    __shared__ f32x4 lds[NW * NS * STAGE / 16];                          // x of the waves, then their partial sums
    char* xl = reinterpret_cast<char*>(lds) + wave * NS * STAGE;
    const uint32_t xr = (uint32_t)(uintptr_t)(buf_lds*)xl + fr * 64 + ((fq ^ (fr >> 1)) & 3) * 16;
    const int rows = min(a.M - m0, 16 * MT), xrow = lane >> 2, xc = (lane ^ (xrow >> 1)) & 3;
    const __amdgpu_buffer_rsrc_t xb = buf_rsrc((const bf16*)a.x + (long)m0 * a.x_rs, (uint32_t)(((rows - 1) * a.x_rs + a.K) * 2));
    uint32_t xo[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xo[t] = (uint32_t)(min(t * 16 + xrow, rows - 1) * a.x_rs + xc * 8) * 2;   // rows behind the last: never stored
    __amdgpu_buffer_rsrc_t wb[NT], sb[NT], zb[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {                                       // tiles behind the last one read zeros
        const long nt = nt0 + n;
        const bool on = nt < tiles;
        wb[n] = buf_rsrc(a.wq + nt * a.KB * 64, on ? a.KB * 1024 : 0);
        sb[n] = buf_rsrc((const bf16*)a.scales + nt * a.KB * GPB * 16, on ? a.KB * GPB * 32 : 0);
        zb[n] = buf_rsrc(a.zeros + nt * a.KB * GPB * 16, on && a.zeros ? a.KB * GPB * 16 : 0);
    }
    const bool has_z = a.zeros != nullptr;
    typedef W4Stage<GPB, NT> Stage;
    auto load_w = [&](Stage& st, int kb) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            st.w[n] = buf_load16(wb[n], kb * 1024 + lane * 16);
#pragma unroll
            for (int g = 0; g < GPB; ++g) {
                st.s[g][n] = buf_load8(sb[n], (kb * GPB + g) * 32 + fq * 8);
                st.z[g][n] = buf_load4(zb[n], (kb * GPB + g) * 16 + fq * 4);
            }
        }
    };
    // Stage i of this wave: part i % STEPS of block wave + NW (i / STEPS).  Behind the last block nothing moves; behind K (scales 0 there) the last
    // fragment once more, which is a number wherever the row is.
    auto load_x = [&](int i, int slot) {
        const int kb = wave + NW * (i / STEPS);
#pragma unroll
        for (int f = 0; f < SF; ++f) {
            const int k = min(kb * 128 + (i % STEPS * SF + f) * 32, a.K - 32);
#pragma unroll
            for (int t = 0; t < MT; ++t)
                buf_load16_lds(xb, xl + slot * STAGE + (f * MT + t) * 1024, kb < a.KB ? xo[t] + k * 2 : BUF_OFF);
        }
    };
    f32x4 acc[NT][MT], xq[NT][MT], xs[MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto use = [&](const Stage& st, int part, int slot) {
        bf16x8 x[SF][MT];
        w4_read(xr + slot * STAGE, x);
#pragma unroll
        for (int f = 0; f < SF; ++f) {
            const int j = part * SF + f, g = j / FPG;
            const bf16 one = (bf16)1.0f;
            const bf16x8 ones = bf16x8{one, one, one, one, one, one, one, one};
            const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < MT; ++t) xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[f][t], j % FPG ? xs[t] : none, 0, 0, 0);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bf16x8 q = w4_fragment(w4_word(st.w[n], j));
#pragma unroll
                for (int t = 0; t < MT; ++t) xq[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, x[f][t], j % FPG ? xq[n][t] : none, 0, 0, 0);
            }
            if (j % FPG == FPG - 1) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const bf16x4 sv = __builtin_bit_cast(bf16x4, st.s[g][n]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float s = (float)sv[r], z = has_z ? (float)((st.z[g][n] >> (8 * r)) & 255u) : 8.0f;
#pragma unroll
                        for (int t = 0; t < MT; ++t) acc[n][t][r] = fmaf(s, fmaf(-z, xs[t][r], xq[n][t][r]), acc[n][t][r]);
                    }
                }
            }
        }
    };
    if (a.KB <= NW) {                                                    // one block per wave: nothing to request ahead (1024 -> 8192: 3.5 against 4.0 us)
        Stage A;
        if (wave < a.KB) {
            load_w(A, wave);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) load_x(i, i);
            if constexpr (STEPS == 2) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(SF * MT) : "memory");
                use(A, 0, 0);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            use(A, STEPS - 1, STEPS - 1);
        }
    } else {
        Stage A, B;
        load_w(A, wave);
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) load_x(i, i);
        int slot = 0, i = 0;
        auto step = [&](const Stage& st, int part, bool on) {            // asks for stage i + NS - 1, multiplies stage i
            load_x(i + NS - 1, slot == 0 ? NS - 1 : slot - 1);
            if (on) {
                if (part >= NS - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(AHEAD) : "memory");
                else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(AHEAD + WEIGHTS) : "memory");
                use(st, part, slot);
            }
            slot = slot == NS - 1 ? 0 : slot + 1;
            ++i;
        };
        // (one way out, behind all loads: from any other the compiler carries loads that are not under way into the loop's head and
        // waits for those that are)
        for (int kb = wave; kb < a.KB; kb += 2 * NW) {
            load_w(B, kb + NW);
#pragma unroll
            for (int p = 0; p < STEPS; ++p) step(A, p, true);
            load_w(A, kb + 2 * NW);
#pragma unroll
            for (int p = 0; p < STEPS; ++p) step(B, p, kb + NW < a.KB);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                 // nothing more lands in LDS
    }
    typedef f32x4 part_t[NT * MT][64];
    part_t* part = reinterpret_cast<part_t*>(lds);
    __syncthreads();                                                     // every wave is done with its x
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[wave][n * MT + t][lane] = acc[n][t];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * MT * 64; i += NW * 64) {
        const int p = i >> 6, l = i & 63, n = p / MT, t = p % MT;
        f32x4 s = part[0][p][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const f32x4 v = part[w][p][l];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] += v[r];
        }
        w4_store<bf16>(a, m0 + t * 16 + (l & 15), (nt0 + n) * 16 + (l >> 4) * 4, s);
    }
}

// Place (in 16 bytes) of piece c of row r in the wave's x: 8 consecutive lanes, the unit of a 16-byte LDS access, touch 8 different places
// mod 8 whether they hold two rows x four pieces (the writes) or eight rows of one piece (the reads).  (With a rotation by 4 places per
// piece the writes met in pairs: 9,200 of 39,000 cycles per CU at 8192 -> 8192, 40 rows.)
__device__ __forceinline__ int w4_place(int r, int c) { return c * 16 + (((r & 7) | (((r >> 3) ^ (r >> 1)) & 1) << 3) ^ ((c & 3) << 1)); }

// ---- the fp32 form: weights become (q - zero) * scale in fp32 (one rounding), the group structure ends there; an MFMA takes 4 inputs, the
// k slots of a fragment are dealt so that a lane's 8 weights of a word meet its 8 values of x.  Two accumulators, for the dependent chain.
template <int GPB> struct W4Stage32 { uint4 w; float s[GPB]; uint32_t z[GPB]; uint4 x[8]; };

template <int G, int NW>
__global__ __launch_bounds__(NW * 64) void linear_w4_f32_kernel(W4Args a) {
    constexpr int GPB = 128 / G;
    const int m0 = blockIdx.y * 16;
    const long nt = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    __shared__ f32x4 lds[NW * 8 * 64];                                   // x of the waves, then their partial sums
    uint4* xl = reinterpret_cast<uint4*>(lds) + wave * 8 * 64;
    const int pc = lane & 3, rw = lane >> 2;                             // this lane loads pieces pc and pc + 4 (of 8 per fragment) of row rw
    const int rows = min(a.M - m0, 16);
    const __amdgpu_buffer_rsrc_t xb = buf_rsrc((const float*)a.x + (long)m0 * a.x_rs, (uint32_t)(((rows - 1) * a.x_rs + a.K) * 4));
    const uint32_t xo = (uint32_t)(min(rw, rows - 1) * a.x_rs + pc * 4) * 4;
    const __amdgpu_buffer_rsrc_t wb = buf_rsrc(a.wq + nt * a.KB * 64, a.KB * 1024);
    const __amdgpu_buffer_rsrc_t sb = buf_rsrc((const float*)a.scales + nt * a.KB * GPB * 16, a.KB * GPB * 64);
    const __amdgpu_buffer_rsrc_t zb = buf_rsrc(a.zeros + nt * a.KB * GPB * 16, a.zeros ? a.KB * GPB * 16 : 0);
    const bool has_z = a.zeros != nullptr;
    typedef W4Stage32<GPB> Stage;
    auto load = [&](Stage& st, int kb) {
        st.w = buf_load16(wb, kb * 1024 + lane * 16);
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            st.s[g] = __builtin_bit_cast(float, buf_load4(sb, (kb * GPB + g) * 64 + fr * 4));
            st.z[g] = buf_load4(zb, (kb * GPB + g) * 16 + (fr & 12));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = kb * 128 + (j >> 1) * 32;
            st.x[j] = buf_load16(xb, k < a.K ? xo + kb * 512 + j * 64 : BUF_OFF);
        }
    };
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    auto use = [&](const Stage& st) {
#pragma unroll
        for (int j = 0; j < 8; ++j) xl[(j >> 1) * 128 + w4_place(rw, (j & 1) * 4 + pc)] = st.x[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int g = j * 32 / G;
            const float z = has_z ? (float)((st.z[g] >> ((fr & 3) * 8)) & 255u) : 8.0f;
            f32x4 x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) x[e] = __builtin_bit_cast(f32x4, xl[j * 128 + w4_place(fr, 2 * fq + e)]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = (w4_value(w4_word(st.w, j), i) - z) * st.s[g];
                acc[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, x[i >> 2][i & 3], acc[i & 1], 0, 0, 0);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    if (a.KB <= NW) {                                                    // one block per wave: nothing to request ahead
        Stage A;
        if (wave < a.KB) {
            load(A, wave);
            use(A);
        }
    } else {
        Stage A, B;
        load(A, wave);
        // (one way out, behind both halves' loads: from any other the compiler carries loads that are not under way into the loop's head
        // and waits for those that are)
        for (int kb = wave; kb < a.KB; kb += 2 * NW) {
            load(B, kb + NW);
            __builtin_amdgcn_sched_barrier(0);                           // (left alone the compiler sinks the loads behind the products)
            use(A);
            load(A, kb + 2 * NW);
            __builtin_amdgcn_sched_barrier(0);
            if (kb + NW < a.KB) use(B);
        }
    }
    typedef f32x4 part_t[64];
    part_t* part = reinterpret_cast<part_t*>(lds);
    __syncthreads();
    part[wave][lane] = f32x4{acc[0][0] + acc[1][0], acc[0][1] + acc[1][1], acc[0][2] + acc[1][2], acc[0][3] + acc[1][3]};
    __syncthreads();
    if (threadIdx.x < 64) {
        f32x4 s = part[0][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const f32x4 v = part[w][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] += v[r];
        }
        w4_store<float>(a, m0 + fr, nt * 16 + fq * 4, s);
    }
}

// ---- fp32, one row: the vector unit's products (a matrix instruction would do 16 rows' work), and column tiles of CW = 4 so that a narrow
// layer still fills the chip: lane = column, quarter of the 32 inputs of a word, and (CW = 4) one of four k blocks.  Sums whole numbers
// times x per group, then scales: another order than the matrix form's, so a row alone is not bit-equal to the same row among others.
template <int G, int CW, int NW>
__global__ __launch_bounds__(NW * 64) void linear_w4_row_kernel(W4Args a) {
    constexpr int GPB = 128 / G, BL = 16 / CW, FPG = G / 32;             // k blocks side by side in a wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane % CW, fq = lane / CW % 4, bl = lane / CW / 4;
    const long nt = blockIdx.x / BL;
    const int fr = blockIdx.x % BL * CW + c;                             // column in the tile of 16
    const __amdgpu_buffer_rsrc_t xb = buf_rsrc(a.x, (uint32_t)a.K * 4);
    const __amdgpu_buffer_rsrc_t wb = buf_rsrc(a.wq + nt * a.KB * 64, a.KB * 1024);
    const __amdgpu_buffer_rsrc_t sb = buf_rsrc((const float*)a.scales + nt * a.KB * GPB * 16, a.KB * GPB * 64);
    const __amdgpu_buffer_rsrc_t zb = buf_rsrc(a.zeros + nt * a.KB * GPB * 16, a.zeros ? a.KB * GPB * 16 : 0);
    const bool has_z = a.zeros != nullptr;
    struct Stage { uint4 w; uint32_t s[GPB], z[GPB]; uint4 x[8]; };
    auto load = [&](Stage& st, int kb) {                                 // (behind the last block: zeros)
        st.w = buf_load16(wb, kb * 1024 + (fq * 16 + fr) * 16);
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            st.s[g] = buf_load4(sb, (kb * GPB + g) * 64 + fr * 4);
            st.z[g] = buf_load4(zb, (kb * GPB + g) * 16 + (fr & 12));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = kb * 128 + (j >> 1) * 32;
            st.x[j] = buf_load16(xb, (uint32_t)(k + fq * 8 + (j & 1) * 4) * 4);
        }
    };
    float acc = 0.f;
    auto use = [&](const Stage& st) {
        float p = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int g = j / FPG;
            const float z = has_z ? (float)((st.z[g] >> ((fr & 3) * 8)) & 255u) : 8.0f;
            if (j % FPG == 0) p = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = w4_value(w4_word(st.w, j), i) - z;       // exact
                p = fmaf(w, __builtin_bit_cast(f32x4, st.x[2 * j + (i >> 2)])[i & 3], p);
            }
            if (j % FPG == FPG - 1) acc = fmaf(__builtin_bit_cast(float, st.s[g]), p, acc);
        }
    };
    constexpr int STEP = NW * BL;
    Stage A, B;
    load(A, wave * BL + bl);
    for (int kb = wave * BL; kb < a.KB; kb += 2 * STEP) {
        load(B, kb + STEP + bl);
        __builtin_amdgcn_sched_barrier(0);
        use(A);
        load(A, kb + 2 * STEP + bl);
        __builtin_amdgcn_sched_barrier(0);
        if (kb + STEP < a.KB) use(B);
    }
    __shared__ f32x4 part[NW][CW / 4];
#pragma unroll
    for (int o = CW; o < 64; o <<= 1) acc += __shfl_xor(acc, o, 64);
    if (lane < CW) reinterpret_cast<float*>(&part[wave][0])[c] = acc;
    __syncthreads();
    if (threadIdx.x < CW / 4) {
        const int i = threadIdx.x;
        f32x4 v = part[0][i];
#pragma unroll
        for (int w = 1; w < NW; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += part[w][i][e];
        w4_store<float>(a, 0, (int)nt * 16 + blockIdx.x % BL * CW + i * 4, v);
    }
}
template <int G>
static void w4_launch_row(const W4Args& a, hipStream_t s) {
    const int tiles = ceil_div(a.N, 16);                                 // us with CW = 4 / 16: 4096 -> 1024 4.2 / 5.4, 1024 -> 2048 3.4 / 3.9; 1024 -> 4096 5.0 / 4.0
    if (tiles < 256) linear_w4_row_kernel<G, 4, 8><<<tiles * 4, 512, 0, s>>>(a);
    else linear_w4_row_kernel<G, 16, 8><<<tiles, 512, 0, s>>>(a);
}

// Row tiles per workgroup: the fewest (more workgroups) that keep the launch within one workgroup per CU, else equal blocks of up to `most`
// (8192 -> 8192, 32 rows as one block of two 13.4 us, as two of one 2 x 9.4; 64 rows as one of four 21.0, as two of two 24.9, and on
// 1024 -> 8192 5.9 / 7.1; 40 rows on 1024 -> 1024 as three of one 3.1).
static int w4_row_tiles(int M, int gx, int most) {
    for (int mt = 1; mt < most; ++mt)
        if ((long)gx * ceil_div(M, 16 * mt) <= 256) return mt;
    return ceil_div(ceil_div(M, ceil_div(M, 16 * most)), 16);
}
template <int G, int NT>
static void w4_launch_bf16(const W4Args& a, hipStream_t s) {
    const int gx = ceil_div(ceil_div(a.N, 16), NT), mt = w4_row_tiles(a.M, gx, 4);
    const dim3 grid(gx, ceil_div(a.M, 16 * mt));
    if (mt == 1) linear_w4_kernel<G, NT, 1, 8><<<grid, 512, 0, s>>>(a);
    else if (mt == 2) linear_w4_kernel<G, NT, 2, 8><<<grid, 512, 0, s>>>(a);
    else if (mt == 3) linear_w4_kernel<G, NT, 3, 8><<<grid, 512, 0, s>>>(a);
    else linear_w4_kernel<G, NT, 4, 8><<<grid, 512, 0, s>>>(a);
}
template <int G>
static void w4_launch(const W4Args& a, int dtype, hipStream_t s) {
    if (dtype == VALLE_BF16) {
        // Two column tiles per wave share the row fragments where that leaves a workgroup per CU; us with one / two: 8192 -> 8192, 1 row
        // 10.8 / 9.5, 32 rows 19.9 / 13.4, 40 rows 24.2 / 16.1; 1024 -> 4096, 64 rows 5.7 / 4.3, but 16 rows (128 workgroups of two) 3.1 / 3.5.
        // (Between 4,096 and 8,192 columns one tile per wave is more than a workgroup per CU, two rounds where the rows fill its LDS: 8192 -> 6144
        // takes 18.1 us for 32 rows and 23.2 for 40, 8192 -> 8192 13.2 and 16.5.  Two tiles were not measured there.)
        if ((long)ceil_div(a.N, 32) * ceil_div(a.M, 48) >= 256) w4_launch_bf16<G, 2>(a, s);
        else w4_launch_bf16<G, 1>(a, s);
        return;
    }
    // one row on the vector unit against the matrix form: 4096 -> 1024 4.1 / 9.8 us, 1024 -> 8192 5.7 / 5.8, 8192 -> 8192 12.5 / 27; two rows
    // took 5.6 / 9.8, 9.1 / 5.8 and 23.8 / 27, four more than the matrix form everywhere
    if (a.M == 1) return w4_launch_row<G>(a, s);
    // (two row tiles per workgroup take as long as two workgroups: 55.3 against 2 x 27.2 us at 8192 -> 8192; the MFMAs bound it)
    linear_w4_f32_kernel<G, 8><<<dim3(ceil_div(a.N, 16), ceil_div(a.M, 16)), 512, 0, s>>>(a);
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
    VALLE_REQUIRE(x_row_stride <= 1 << 23 && (int64_t)ceil_div(K, 128) * 1024 <= INT32_MAX / 2, VALLE_E_ARG, "valle_linear_w4: x_row_stride %lld or K %d too large",
                  (long long)x_row_stride, K);
    VALLE_REQUIRE(M <= 65535 * 16, VALLE_E_ARG, "valle_linear_w4: %d rows", M);
    if (M == 0) return VALLE_OK;
    W4Args a{x, (const uint4*)wq, scales, zeros, bias, resid, C, x_row_stride, M, N, K, ceil_div(K, 128), ldc, epilogue};
    hipStream_t st = (hipStream_t)stream;
    if (group == 32) w4_launch<32>(a, dtype, st);
    else if (group == 64) w4_launch<64>(a, dtype, st);
    else w4_launch<128>(a, dtype, st);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}
