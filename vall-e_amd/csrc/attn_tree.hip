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

// one tile of a wave: SUB sub-tiles of 16 keys (32 keys of bf16, 16 of fp32: 4 KB of K, 4 KB of V)
template <typename T> struct TreeTile {
    static constexpr int SUB = 4 / sizeof(T);
    typedef T vrow __attribute__((ext_vector_type(4)));
    uint4 k[4];                         // the tile's K bytes as they lie: load i, lane l = bytes i * 1024 + l * 16
    vrow v[SUB][4];                     // key fq * 4 + r, dims fr * 4 .. + 4
    uint32_t live;                      // bit s: the page of sub-tile s is one of the cache's
};
// K goes from the loads' order (whole 128-byte lines; a key per lane, as the fragments have it, loads at a quarter of the rate) to
// fragment order through 4 KB of the wave's own LDS.  A row is CH pieces of 16 bytes, piece c of row r at r * CH + (c ^ (r mod CH)):
// both sides free of bank conflicts.
template <typename T>
__device__ __forceinline__ void tree_stage_k(const TreeTile<T>& t, uint4* kl, int lane) {
    constexpr int CH = 4 * (int)sizeof(T), RPL = 64 / CH;                // pieces per row, rows per load
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * RPL + lane / CH;
        kl[r * CH + ((lane % CH) ^ (r % CH))] = t.k[i];
    }
}
template <typename T>
__device__ __forceinline__ uint4 tree_k_piece(const uint4* kl, int r, int c) {
    constexpr int CH = 4 * (int)sizeof(T);
    return kl[r * CH + (c ^ (r % CH))];
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
// scores of sub-tile s for QB query blocks: lane = query fr, keys fq * 4 + r
template <int QB>
__device__ __forceinline__ void tree_scores(const uint4* kl, int s, int fr, int fq, const TreeQuery<bf16> (&q)[QB], f32x4 (&st)[QB][2]) {
    const bf16x8 k0 = __builtin_bit_cast(bf16x8, tree_k_piece<bf16>(kl, s * 16 + fr, fq)), k1 = __builtin_bit_cast(bf16x8, tree_k_piece<bf16>(kl, s * 16 + fr, fq + 4));
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        st[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q[j].x[0], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        st[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q[j].x[1], st[j][s], 0, 0, 0);
    }
}
template <int QB>
__device__ __forceinline__ void tree_scores(const uint4* kl, int s, int fr, int fq, const TreeQuery<float> (&q)[QB], f32x4 (&st)[QB][1]) {
#pragma unroll
    for (int j = 0; j < QB; ++j) st[j][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 k = __builtin_bit_cast(f32x4, tree_k_piece<float>(kl, fr, fq * 4 + i));
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < QB; ++j) st[j][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[j].x[i][e], st[j][0], 0, 0, 0);
    }
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
            uint32_t a[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint2 row = __builtin_bit_cast(uint2, t.v[s][r]);
                a[r] = dt < 2 ? row.x : row.y;
            }
            w[2 * s] = __builtin_amdgcn_perm(a[1], a[0], sel);
            w[2 * s + 1] = __builtin_amdgcn_perm(a[3], a[2], sel);
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

template <typename T>
__device__ __forceinline__ bool tree_odd(const TreeTile<T>& t, int s, int r) {           // infinities or NaN in the lane's 4 dims of V row r
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= !(fabsf(to_f32<T>(t.v[s][r][e])) < INFINITY);
    return odd;
}
template <typename T>
__device__ __forceinline__ void tree_clean_v(TreeTile<T>& t, int s, int r) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!(fabsf(to_f32<T>(t.v[s][r][e])) < INFINITY)) t.v[s][r][e] = from_f32<T>(0.f);
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
    // Every load of the loop is issued whatever the case, through bounds-checked descriptors: what lies behind the wave's last tile
    // moves no data, and the loads stay countable.
    const int mine = t0 + wave < t1 ? (t1 - t0 - wave + NW - 1) / NW : 0;
    const __amdgpu_buffer_rsrc_t tb = buf_rsrc(tab, a.width * 4);
    auto page_of = [&](int i) {                                          // lane s (mod SUB): the page of sub-tile s of this wave's tile i
        const int key = (t0 + wave + NW * i) * KT + (lane % SUB) * 16;
        return (int)buf_load4(tb, i < mine && key < T_all ? (uint32_t)(key >> a.shift) * 4 : BUF_OFF);
    };
    auto load = [&](Tile& t, int i, int pages) {
        t.live = 0;
        const int key0 = (t0 + wave + NW * i) * KT;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int page = __builtin_amdgcn_readlane(pages, s), key = key0 + s * 16;
            const bool on = i < mine && key < T_all && page >= 0 && page < a.n_pages;
            const long at = (on ? page : 0) * page_stride + (long)(key & ((1 << a.shift) - 1)) * 64;
            const uint32_t bytes = on ? min(16, T_all - key) * 64 * (int)sizeof(T) : 0;
            const __amdgpu_buffer_rsrc_t k = buf_rsrc(kbase + at, bytes), v = buf_rsrc(vbase + at, bytes);      // rows behind the sequence read zeros
#pragma unroll
            for (int i = 0; i < 4 / SUB; ++i) t.k[s * (4 / SUB) + i] = buf_load16(k, i * 1024 + lane * 16);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t off = ((fq * 4 + r) * 64 + fr * 4) * (int)sizeof(T);
                if constexpr (sizeof(T) == 2) t.v[s][r] = __builtin_bit_cast(typename Tile::vrow, buf_load8(v, off));
                else t.v[s][r] = __builtin_bit_cast(typename Tile::vrow, buf_load16(v, off));
            }
            if (on) t.live |= 1u << s;
        }
    };
    auto use = [&](Tile& t, int i) {
        const int key0 = (t0 + wave + NW * i) * KT;
        uint4* kl = reinterpret_cast<uint4*>(&so[wave][0][0]);
        tree_stage_k(t, kl, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f32x4 st[QB][SUB];
#pragma unroll
        for (int s = 0; s < SUB; ++s) tree_scores<QB>(kl, s, fr, fq, qf, st);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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
                    if (node >= 0) odd |= tree_odd(t, s, r);             // (rows behind the sequence were read as zeros)
                }
        }
        // The shift of the exponentials needs to be near the maximum, not the maximum: it follows only when a score lies more than 8
        // (a factor of 256 in a weight) above it, so that most tiles reduce nothing over lanes and scale nothing.
        float top[QB];
        bool grow = false;
#pragma unroll
        for (int j = 0; j < QB; ++j) {
            top[j] = st[j][0][0];
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) top[j] = fmaxf(top[j], st[j][s][r]);
            grow |= top[j] * a.scale_log2 > m[j] + 8.0f;                 // scale > 0: the maximum commutes with it
        }
        if (__any(grow)) {
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                float mx = fmaxf(top[j], __shfl_xor(top[j], 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = mx * a.scale_log2 > m[j] + 8.0f ? mx * a.scale_log2 : m[j];      // by the query's own scores alone
                const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[j] - mn);
                l[j] *= alpha;
                m[j] = mn;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][dt][r] *= alpha;
            }
        }
#pragma unroll
        for (int j = 0; j < QB; ++j) {
            const float ms = m[j] == -INFINITY ? 0.f : m[j];             // nothing seen so far: keep the arguments finite
            float sum = 0.f;
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[j][s][r], a.scale_log2, -ms));
                    st[j][s][r] = p;
                    sum += p;
                }
            l[j] += sum;
        }
        if (edge && __any(odd)) {
            // A node's V row with infinities or NaN belongs to the queries that see it and to no other: 0 x inf in the MFMA
            // would reach them all.  Such elements leave the tile and are added to the seeing queries alone, read once more.
            uint32_t rows = 0;                                           // keys of the tile
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool bad = key0 + s * 16 + fq * 4 + r >= ctx && tree_odd(t, s, r);
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
    if (mine > 0) {
        Tile A, B;
        int next = page_of(0);
        load(A, 0, next);
        next = page_of(1);
        for (int i = 0;; i += 2) {
            int after = page_of(i + 2);
            load(B, i + 1, next);
            __builtin_amdgcn_sched_barrier(0);                           // (left alone the compiler sinks the loads behind the products)
            use(A, i);
            if (i + 1 >= mine) break;
            next = page_of(i + 3);
            load(A, i + 2, after);
            __builtin_amdgcn_sched_barrier(0);
            use(B, i + 1);
            if (i + 2 >= mine) break;
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
    for (int s0 = 0; s0 < a.nsplit; s0 += 8) {                           // eight loads under way
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a.part[(at + min(s0 + i, a.nsplit - 1)) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ws = s0 + i < a.nsplit ? __shfl(w, (s0 + i) & 63, 64) : 0.f;
            acc = ws == 0.f ? acc : acc + v[i] * ws;                     // (a part that saw nothing wrote no sums)
        }
    }
    ((T*)a.out)[row * a.o_rs + head * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : acc / L);
}

static int tree_qb(int nq) { return nq <= 16 ? 1 : nq <= 32 ? 2 : 4; }
// Workgroups over the key axis: requests x kv heads x query blocks fill the chip alone from 256 on; below that the keys are
// split until they do (two workgroups of one query block share a CU, larger ones have it alone), as long as a wave keeps two tiles.
static int tree_splits(int B, int Hkv, int g, int max_nodes, int max_ctx, int kt, int nw) {
    const int nq = max_nodes * g;
    const long base = (long)B * Hkv * ceil_div(nq, 16 * tree_qb(nq));
    const long tiles = ((long)max_ctx + max_nodes + kt - 1) / kt;
    const long fill = tree_qb(nq) == 1 ? 512 : 256;
    long s = (fill + base - 1) / base;
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
    VALLE_REQUIRE(n_pages > 0 && ((int64_t)n_pages << shift) <= INT32_MAX && max_blocks > 0 && ((int64_t)max_blocks << shift) <= INT32_MAX - (1 << 20), VALLE_E_ARG,
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
