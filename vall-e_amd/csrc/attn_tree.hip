// Attention of each request's drafted tokens (a tree of up to 64 nodes; one node: a plain decode step) over a paged KV cache.
//   out_i = sum_t softmax_t(q_i . k_t * scale) v_t   over the context rows t < ctx and the nodes j whose bit is set in mask_i
// Per (request, kv head) the queries are the n nodes x g grouped heads; the score tile is computed transposed, S^T = K . Q^T
// (16 keys x 16 queries per MFMA, A = K rows straight from the page, B = Q), so a lane owns one query and four keys of every
// 16: running maximum and sum are per-lane values (fp32) and P^T is already the B operand of O^T += V^T . P^T.  V is loaded
// as 4 keys x 4 dims per lane and its 16-bit 4 x 4 blocks are turned in registers (8 v_perm per 16 keys): nothing but the
// final merge goes through LDS.  The waves of a workgroup split the keys, so do up to 64 workgroups (grid x) where requests and
// heads alone do not fill the chip; a second launch joins their partial sums.
// Bound: the K / V bytes (2 x T x Hkv x 64 x es); 16 queries use the MFMA columns fully.
#include "common.h"

struct TreeArgs {
    const void *q, *kc, *vc;
    void* out;
    const int32_t *table, *ctx, *cu;
    const int64_t* mask;                // bit j of row i: node i sees node j; NULL: a chain (nodes 0 .. i)
    float* part;                        // [rows * H][nsplit][64] sums, then [rows * H][nsplit][2] (maximum, denominator)
    long q_rs, o_rs;                    // elements
    float scale_log2;
    int width, n_pages, shift, rows, H, Hkv, g, max_nodes, nsplit;
};

#define TREE_MAX_NODES 64
#define TREE_MAX_SPLIT 64

// one tile of a wave: SUB sub-tiles of 16 keys in fragment order
template <typename T> struct TreeTile;
template <> struct TreeTile<bf16> {
    static constexpr int SUB = 2;
    uint4 k[2][2];                      // key fr, dims fq * 8 .. + 8 of either half
    uint2 v[2][4];                      // key fq * 4 + r, dims fr * 4 .. + 4
    uint32_t live;                      // bit s: the page of sub-tile s is one of the cache's
};
template <> struct TreeTile<float> {
    static constexpr int SUB = 1;
    f32x4 k[1][4];                      // key fr, dims fq * 16 + 4 i .. + 4
    f32x4 v[1][4];                      // key fq * 4 + r, dims fr * 4 .. + 4
    uint32_t live;
};

__device__ __forceinline__ void tree_load_sub(TreeTile<bf16>& t, int s, const bf16* kp, const bf16* vp, int fr, int fq) {
    t.k[s][0] = *reinterpret_cast<const uint4*>(kp + fr * 64 + fq * 8);
    t.k[s][1] = *reinterpret_cast<const uint4*>(kp + fr * 64 + fq * 8 + 32);
#pragma unroll
    for (int r = 0; r < 4; ++r) t.v[s][r] = *reinterpret_cast<const uint2*>(vp + (fq * 4 + r) * 64 + fr * 4);
}
__device__ __forceinline__ void tree_load_sub(TreeTile<float>& t, int s, const float* kp, const float* vp, int fr, int fq) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t.k[s][i] = *reinterpret_cast<const f32x4*>(kp + fr * 64 + fq * 16 + i * 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) t.v[s][r] = *reinterpret_cast<const f32x4*>(vp + (fq * 4 + r) * 64 + fr * 4);
}
__device__ __forceinline__ void tree_zero_sub(TreeTile<bf16>& t, int s) {
    t.k[s][0] = t.k[s][1] = uint4{0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 4; ++r) t.v[s][r] = uint2{0, 0};
}
__device__ __forceinline__ void tree_zero_sub(TreeTile<float>& t, int s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t.k[s][i] = t.v[s][i] = f32x4{0.f, 0.f, 0.f, 0.f};
}

template <typename T> struct TreeQuery;
template <> struct TreeQuery<bf16> { bf16x8 x[2]; };
template <> struct TreeQuery<float> { f32x4 x[4]; };
__device__ __forceinline__ void tree_load_q(TreeQuery<bf16>& q, const bf16* p, int fq) {
    q.x[0] = *reinterpret_cast<const bf16x8*>(p + fq * 8);
    q.x[1] = *reinterpret_cast<const bf16x8*>(p + fq * 8 + 32);
}
__device__ __forceinline__ void tree_load_q(TreeQuery<float>& q, const float* p, int fq) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.x[i] = *reinterpret_cast<const f32x4*>(p + fq * 16 + i * 4);
}
__device__ __forceinline__ f32x4 tree_scores(const TreeTile<bf16>& t, int s, const TreeQuery<bf16>& q) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[s][0]), q.x[0], a, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[s][1]), q.x[1], a, 0, 0, 0);
}
__device__ __forceinline__ f32x4 tree_scores(const TreeTile<float>& t, int s, const TreeQuery<float>& q) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) a = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[s][i][e], q.x[i][e], a, 0, 0, 0);
    return a;
}
// o[dt] rows i = dims i * 4 + dt: the lane holds dims (fq * 4 + r) * 4 + dt of its query
template <int QB>
__device__ __forceinline__ void tree_pv(const TreeTile<bf16>& t, const f32x4 (&p)[QB][2], f32x4 (&o)[QB][4]) {
    bf16x8 pf[QB];
#pragma unroll
    for (int j = 0; j < QB; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) pf[j][e] = (bf16)p[j][e >> 2][e & 3];      // P rounded to bf16 for the MFMA (the denominator keeps fp32)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
        uint32_t w[4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t sel = dt & 1 ? 0x07060302u : 0x05040100u;
            const uint32_t a0 = dt < 2 ? t.v[s][0].x : t.v[s][0].y, a1 = dt < 2 ? t.v[s][1].x : t.v[s][1].y;
            const uint32_t a2 = dt < 2 ? t.v[s][2].x : t.v[s][2].y, a3 = dt < 2 ? t.v[s][3].x : t.v[s][3].y;
            w[2 * s] = __builtin_amdgcn_perm(a1, a0, sel);
            w[2 * s + 1] = __builtin_amdgcn_perm(a3, a2, sel);
        }
        const bf16x8 vt = __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
#pragma unroll
        for (int j = 0; j < QB; ++j) o[j][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, pf[j], o[j][dt], 0, 0, 0);
    }
}
template <int QB>
__device__ __forceinline__ void tree_pv(const TreeTile<float>& t, const f32x4 (&p)[QB][1], f32x4 (&o)[QB][4]) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < QB; ++j) o[j][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.v[0][r][dt], p[j][0][r], o[j][dt], 0, 0, 0);
}

// element e (0 .. 3) of a lane's V row r in sub-tile s
__device__ __forceinline__ float tree_v(const TreeTile<bf16>& t, int s, int r, int e) {
    const uint32_t w = e < 2 ? t.v[s][r].x : t.v[s][r].y;
    return __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ float tree_v(const TreeTile<float>& t, int s, int r, int e) { return t.v[s][r][e]; }
__device__ __forceinline__ void tree_zero_v(TreeTile<bf16>& t, int s, int r) { t.v[s][r] = uint2{0, 0}; }
__device__ __forceinline__ void tree_zero_v(TreeTile<float>& t, int s, int r) { t.v[s][r] = f32x4{0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ void tree_clean_v(TreeTile<bf16>& t, int s, int r) {           // infinities and NaN -> 0
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t& w = e < 2 ? t.v[s][r].x : t.v[s][r].y;
        const uint32_t half = e & 1 ? 0xffff0000u : 0x0000ffffu;
        if (!(fabsf(tree_v(t, s, r, e)) < INFINITY)) w &= ~half;
    }
}
__device__ __forceinline__ void tree_clean_v(TreeTile<float>& t, int s, int r) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!(fabsf(t.v[s][r][e]) < INFINITY)) t.v[s][r][e] = 0.f;
}

template <typename T, int QB, int NW>
__global__ __launch_bounds__(NW * 64) void attn_tree_kernel(TreeArgs a) {
    typedef TreeTile<T> Tile;
    constexpr int SUB = Tile::SUB, KT = 16 * SUB;
    const int split = blockIdx.x, kvh = blockIdx.y % a.Hkv, qblk = blockIdx.y / a.Hkv, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 15, fq = lane >> 4;
    const int ctx_in = a.ctx[b], r0 = a.cu[b];
    if (ctx_in < 0 || r0 < 0) return;                                    // a finished request: its rows stay as they are
    const int nk = min(max(a.cu[b + 1] - r0, 0), TREE_MAX_NODES);        // nodes that are keys
    const int n = min(min(nk, a.max_nodes), a.rows - r0);                // nodes that ask
    const int nq = n * a.g, q0 = qblk * 16 * QB;
    if (n <= 0 || q0 >= nq) return;
    const int T_all = (int)min((long)ctx_in + nk, (long)a.width << a.shift);
    const int ctx = min(ctx_in, T_all);
    const int tiles = (T_all + KT - 1) / KT, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(tiles, t0 + per);

    const int32_t* tab = a.table + (long)b * a.width;
    const T* kbase = (const T*)a.kc + ((long)kvh << a.shift) * 64;
    const T* vbase = (const T*)a.vc + ((long)kvh << a.shift) * 64;
    const long page_stride = ((long)a.Hkv << a.shift) * 64;

    TreeQuery<T> qf[QB];
    uint64_t see[QB];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        const int qi = min(q0 + j * 16 + fr, nq - 1), node = qi / a.g, head = kvh * a.g + qi % a.g;
        tree_load_q(qf[j], (const T*)a.q + (long)(r0 + node) * a.q_rs + head * 64, fq);
        see[j] = a.mask ? (uint64_t)a.mask[r0 + node] : (2ull << node) - 1;
    }
    float m[QB], l[QB];
    f32x4 o[QB][4];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        m[j] = -INFINITY; l[j] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[j][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __shared__ float so[NW][16][68];
    __shared__ float sm[NW][16], sl[NW][16];
    // page of the wave's sub-tiles, 64 at a time: lane i holds sub-tile i of the current window
    int pages = -1;
    auto load = [&](Tile& t, int i) {                                    // tile number i of this wave
        const int w = (i * SUB) & 63;
        if (w == 0) {
            const long key = (long)(t0 + wave + NW * (i + lane / SUB)) * KT + (lane % SUB) * 16;
            pages = key < T_all ? tab[key >> a.shift] : -1;
            if (pages >= a.n_pages) pages = -1;
        }
        t.live = 0;
        const int key0 = (t0 + wave + NW * i) * KT;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int page = __builtin_amdgcn_readlane(pages, w + s);
            if (page >= 0) {
                const long at = page * page_stride + (long)((key0 + s * 16) & ((1 << a.shift) - 1)) * 64;
                tree_load_sub(t, s, kbase + at, vbase + at, fr, fq);
                t.live |= 1u << s;
            } else tree_zero_sub(t, s);
        }
    };
    auto use = [&](Tile& t, int i) {
        const int key0 = (t0 + wave + NW * i) * KT;
        f32x4 st[QB][SUB];
#pragma unroll
        for (int j = 0; j < QB; ++j)
#pragma unroll
            for (int s = 0; s < SUB; ++s) st[j][s] = tree_scores(t, s, qf[j]);
        const bool edge = key0 + KT > ctx || t.live != (1u << SUB) - 1;  // wave-uniform: only the tiles with nodes, or with pages missing
        bool odd = false;                                                // a drafted row holds infinities or NaN
        if (edge) {
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + s * 16 + fq * 4 + r;
                    const bool there = key < T_all && ((t.live >> s) & 1);
                    const int node = key - ctx;
#pragma unroll
                    for (int j = 0; j < QB; ++j)
                        if (!there || (node >= 0 && !((see[j] >> (node & 63)) & 1))) st[j][s][r] = -INFINITY;
                    if (!there) tree_zero_v(t, s, r);                    // rows behind the sequence may hold anything (0 x NaN)
                    else if (node >= 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= !(fabsf(tree_v(t, s, r, e)) < INFINITY);
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < QB; ++j) {
            float mx = st[j][0][0];
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[j][s][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float mn = fmaxf(m[j], mx * a.scale_log2);             // scale > 0: the maximum commutes with it
            const float ms = mn == -INFINITY ? 0.f : mn;                 // nothing seen so far: keep the arguments finite
            const float alpha = __builtin_amdgcn_exp2f(m[j] - ms);
            float sum = 0.f;
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[j][s][r], a.scale_log2, -ms));
                    st[j][s][r] = p;
                    sum += p;
                }
            l[j] = l[j] * alpha + sum;
            m[j] = mn;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[j][dt][r] *= alpha;
        }
        if (edge && __any(odd)) {
            // A node's V row with infinities or NaN belongs to the queries that see it and to no other: 0 x inf in the MFMA
            // would reach them all.  Such elements leave the tile and are added to the seeing queries alone, read once more.
            uint32_t rows = 0;                                           // keys of the tile
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bool bad = false;
                    if (key0 + s * 16 + fq * 4 + r >= ctx) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) bad |= !(fabsf(tree_v(t, s, r, e)) < INFINITY);
                    }
                    const uint64_t lanes = __ballot(bad);
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        if ((lanes >> (16 * f)) & 0xffff) rows |= 1u << (s * 16 + f * 4 + r);
                    if (bad) tree_clean_v(t, s, r);
                }
            float* pl = &so[wave][0][0];                                 // the wave's own merge area: P as [key][16 queries]
#pragma unroll
            for (int j = 0; j < QB; ++j) {
#pragma unroll
                for (int s = 0; s < SUB; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pl[(s * 16 + fq * 4 + r) * 16 + fr] = st[j][s][r];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (uint32_t left = rows; left; left &= left - 1) {
                    const int kk = __builtin_ctz(left), key = key0 + kk;
                    const float p = pl[kk * 16 + fr];
                    const T* vp = vbase + tab[key >> a.shift] * page_stride + (long)(key & ((1 << a.shift) - 1)) * 64 + fq * 16;
                    if (p > 0.f) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int dt = 0; dt < 4; ++dt) {
                                const float v = to_f32<T>(vp[r * 4 + dt]);
                                if (!(fabsf(v) < INFINITY)) o[j][dt][r] += p * v;
                            }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        tree_pv<QB>(t, st, o);
    };
    const int mine = t0 + wave < t1 ? (t1 - t0 - wave + NW - 1) / NW : 0;
    if (mine > 0) {
        Tile A, B;
        load(A, 0);
        for (int i = 0; i < mine; i += 2) {
            if (i + 1 < mine) load(B, i + 1);
            use(A, i);
            if (i + 1 < mine) {
                if (i + 2 < mine) load(A, i + 2);
                use(B, i + 1);
            }
        }
    }
    // ---- merge of the waves, one block of 16 queries at a time
    constexpr int DPT = 16 / NW;                                         // dims per thread in the merge
    const int mq = threadIdx.x / (64 / DPT), md = threadIdx.x % (64 / DPT) * DPT;
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        if (q0 + j * 16 < nq) {                                          // uniform
        float lt = l[j];
        lt += __shfl_xor(lt, 16, 64);
        lt += __shfl_xor(lt, 32, 64);
        if (j) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f32x4*>(&so[wave][fr][(fq * 4 + r) * 4]) = f32x4{o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]};
        if (fq == 0) { sm[wave][fr] = m[j]; sl[wave][fr] = lt; }
        __syncthreads();
        const int qi = q0 + j * 16 + mq;
        if (qi < nq) {
            float M = -INFINITY, L = 0.f, acc[DPT] = {};
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][mq]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float sc = sm[w][mq] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[w][mq] - M);
                if (sc == 0.f) continue;                                 // that wave saw nothing of weight
                L += sl[w][mq] * sc;
#pragma unroll
                for (int d = 0; d < DPT; ++d) acc[d] += so[w][mq][md + d] * sc;
            }
            const int node = qi / a.g, head = kvh * a.g + qi % a.g;
            const long row = r0 + node;
            if (a.nsplit == 1) {
                T* op = (T*)a.out + row * a.o_rs + head * 64 + md;
#pragma unroll
                for (int d = 0; d < DPT; ++d) op[d] = from_f32<T>(L == 0.f ? 0.f : acc[d] / L);     // a row that sees nothing is zero
            } else {
                const long at = (row * a.H + head) * a.nsplit + split;
#pragma unroll
                for (int d = 0; d < DPT; ++d) a.part[at * 64 + md + d] = acc[d];
                if (md == 0) {
                    float* ml = a.part + (long)a.rows * a.H * a.nsplit * 64 + at * 2;
                    ml[0] = M; ml[1] = L;
                }
            }
        }
        }
    }
}

// joins the workgroups' partial sums: one wave per (row, head), a lane per dimension
template <typename T>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs a) {
    const int b = blockIdx.x, node = blockIdx.y, lane = threadIdx.x & 63;
    const int head = blockIdx.z * 4 + (threadIdx.x >> 6);
    const int r0 = a.cu[b];
    if (a.ctx[b] < 0 || r0 < 0 || head >= a.H) return;
    if (node >= min(min(a.cu[b + 1] - r0, a.max_nodes), a.rows - r0)) return;
    const long row = r0 + node, at = (row * a.H + head) * a.nsplit;
    const float* ml = a.part + (long)a.rows * a.H * a.nsplit * 64 + at * 2;
    const float mv = lane < a.nsplit ? ml[2 * lane] : -INFINITY;
    const float lv = lane < a.nsplit ? ml[2 * lane + 1] : 0.f;
    const float M = wave_max(mv);
    const float w = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - M);
    const float L = wave_sum(w == 0.f ? 0.f : lv * w);
    float acc = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float ws = __shfl(w, s, 64);
        if (ws != 0.f) acc += a.part[(at + s) * 64 + lane] * ws;
    }
    ((T*)a.out)[row * a.o_rs + head * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : acc / L);
}

static int tree_qb(int nq) { return nq <= 16 ? 1 : nq <= 32 ? 2 : 4; }
// Workgroups over the key axis: requests x kv heads x query blocks fill the chip alone from 512 on; below that the keys are
// split until they do, as long as a wave keeps two tiles.
static int tree_splits(int B, int Hkv, int g, int max_nodes, int max_ctx, int kt, int nw) {
    const int nq = max_nodes * g;
    const long base = (long)B * Hkv * ceil_div(nq, 16 * tree_qb(nq));
    const long tiles = ((long)max_ctx + max_nodes + kt - 1) / kt;
    long s = (512 + base - 1) / base;
    if (s > tiles / (2 * nw)) s = tiles / (2 * nw);
    if (base >= 256) s = 1;
    return (int)(s < 1 ? 1 : s > TREE_MAX_SPLIT ? TREE_MAX_SPLIT : s);
}
static bool tree_shape_ok(int rows, int B, int H, int Hkv, int max_nodes, int max_ctx) {
    return rows >= 0 && B >= 0 && B <= 65535 && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 65535 && max_nodes > 0 && max_nodes <= TREE_MAX_NODES && max_ctx >= 0;
}
#define TREE_NW 8

extern "C" size_t valle_attn_tree_workspace_bytes(int rows, int B, int max_nodes, int max_ctx, int H, int Hkv, int dtype) {
    if (!tree_shape_ok(rows, B, H, Hkv, max_nodes, max_ctx) || B == 0) return 0;
    const int ns = tree_splits(B, Hkv, H / Hkv, max_nodes, max_ctx, dtype == VALLE_BF16 ? 32 : 16, TREE_NW);
    return ns == 1 ? 0 : (size_t)rows * H * ns * 66 * sizeof(float);
}

template <typename T>
static void tree_launch(const TreeArgs& a, int B, hipStream_t s) {
    const int nq = a.max_nodes * a.g, qb = tree_qb(nq);
    dim3 grid(a.nsplit, a.Hkv * ceil_div(nq, 16 * qb), B);
    if (qb == 1) attn_tree_kernel<T, 1, TREE_NW><<<grid, TREE_NW * 64, 0, s>>>(a);
    else if (qb == 2) attn_tree_kernel<T, 2, TREE_NW><<<grid, TREE_NW * 64, 0, s>>>(a);
    else attn_tree_kernel<T, 4, TREE_NW><<<grid, TREE_NW * 64, 0, s>>>(a);
    if (a.nsplit > 1) attn_tree_join_kernel<T><<<dim3(B, a.max_nodes, ceil_div(a.H, 4)), 256, 0, s>>>(a);
}

extern "C" int valle_attn_tree(const void* q, int64_t q_row_stride, const void* kcache, const void* vcache, int n_pages, int page_size,
                               const int32_t* block_table, int max_blocks, const int32_t* ctx_len, const int32_t* cu_rows,
                               const int64_t* tree_mask, void* out, int64_t out_row_stride, int rows, int B, int max_nodes, int max_ctx,
                               int H, int Hkv, int Dh, float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    VALLE_REQUIRE(q && kcache && vcache && block_table && ctx_len && cu_rows && out, VALLE_E_ARG, "valle_attn_tree: null pointer");
    VALLE_REQUIRE(dtype == VALLE_BF16 || dtype == VALLE_F32, VALLE_E_ARG, "valle_attn_tree: unknown dtype %d", dtype);
    VALLE_REQUIRE(Dh == 64, VALLE_E_UNSUPPORTED, "valle_attn_tree: head_dim %d (64 is built)", Dh);
    VALLE_REQUIRE(tree_shape_ok(rows, B, H, Hkv, max_nodes, max_ctx), VALLE_E_ARG,
                  "valle_attn_tree: rows=%d B=%d H=%d Hkv=%d max_nodes=%d (1 .. %d) max_ctx=%d", rows, B, H, Hkv, max_nodes, TREE_MAX_NODES, max_ctx);
    int shift = -1;
    for (int i = 4; i <= 8; ++i)
        if (page_size == 1 << i) shift = i;
    VALLE_REQUIRE(shift > 0, VALLE_E_ARG, "valle_attn_tree: page_size %d (16, 32, 64, 128 or 256)", page_size);
    VALLE_REQUIRE(n_pages > 0 && ((int64_t)n_pages << shift) <= INT32_MAX && max_blocks > 0 && ((int64_t)max_blocks << shift) <= INT32_MAX, VALLE_E_ARG,
                  "valle_attn_tree: n_pages %d, max_blocks %d", n_pages, max_blocks);
    VALLE_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, VALLE_E_ARG, "valle_attn_tree: softmax_scale must be positive");
    const int vec = 16 / (int)dtype_size(dtype);
    const void* ptrs[] = {q, kcache, vcache};
    for (const void* p : ptrs) VALLE_REQUIRE(((uintptr_t)p & 15) == 0, VALLE_E_ARG, "valle_attn_tree: tensors must be 16-byte aligned");
    VALLE_REQUIRE(q_row_stride >= 0 && q_row_stride % vec == 0, VALLE_E_ARG, "valle_attn_tree: q rows must stay 16-byte aligned");
    VALLE_REQUIRE(rows <= 1 || out_row_stride >= (int64_t)H * 64, VALLE_E_ARG, "valle_attn_tree: rows of out overlap");
    if (B == 0 || rows == 0) return VALLE_OK;
    TreeArgs a{q, kcache, vcache, out, block_table, ctx_len, cu_rows, tree_mask, (float*)workspace, q_row_stride, out_row_stride,
               softmax_scale * 1.4426950408889634f, max_blocks, n_pages, shift, rows, H, Hkv, H / Hkv, max_nodes, 1};
    a.nsplit = tree_splits(B, Hkv, a.g, max_nodes, max_ctx, dtype == VALLE_BF16 ? 32 : 16, TREE_NW);
    const size_t need = valle_attn_tree_workspace_bytes(rows, B, max_nodes, max_ctx, H, Hkv, dtype);
    VALLE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), VALLE_E_WORKSPACE,
                  "valle_attn_tree: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    const long gy = (long)Hkv * ceil_div(max_nodes * a.g, 16 * tree_qb(max_nodes * a.g));
    VALLE_REQUIRE(gy <= 65535, VALLE_E_ARG, "valle_attn_tree: %d heads are too many", H);
    if (dtype == VALLE_BF16) tree_launch<bf16>(a, B, (hipStream_t)stream);
    else tree_launch<float>(a, B, (hipStream_t)stream);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}
