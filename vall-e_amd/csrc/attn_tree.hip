// Attention of each request's drafted tokens (a tree of up to 64 nodes; one node: a plain decode step) over a paged KV cache.
//   out_i = sum_t softmax_t(q_i . k_t * scale) v_t   over the context rows t < ctx and the nodes j whose bit is set in mask_i
// Per (request, kv head) the queries are the n nodes x g grouped heads; the score tile is computed transposed, S^T = K . Q^T
// (16 keys x 16 queries per MFMA, A = K, B = Q), so a lane owns one query and four keys of every 16: running maximum and sum are per-lane
// values (fp32) and P^T is already the B operand of O^T += V^T . P^T.  K goes from whole-line loads to fragments through the wave's own
// LDS; V is loaded as 4 keys x 4 dims per lane and its 16-bit 4 x 4 blocks are turned in registers (8 v_perm per 16 keys).  The four or eight
// waves of a workgroup split the keys, so do up to 64 workgroups (grid x) where requests and heads alone do not fill the chip; a second launch
// joins their partial sums.  Inside the loop waves never wait for one another.
// Bound: the K / V bytes (2 x T x Hkv x 64 x es) with few queries, us on inputs that change from call to call (replayed on the same ones, part of
// which stays cached): 16 requests x 311 .. 761 keys x 16 heads, one token (35 MB) 9.2 (7.5); 32 x 1,800 .. 2,561 keys, 9 .. 26 nodes
// (290 MB) 55 (46) = 5.3 TB/s.  With 64 nodes x 4 grouped heads the bytes no longer count (1 x 130,001 keys: 34 GFLOP in 60 us): two waves per
// SIMD (244 registers) cover each other's latencies in part.  There the vector unit issues in 0.58 of a busy CU's cycles and the matrix unit works in 0.28,
// waves wait in 0.31 of theirs.  When that call took 69.6 us it took 63.7 without its exponentials, 59.2 without the P.V products, 57.6 without
// the loads, 68.0 without K's way through LDS.  Tried there and not faster: products placed between the exponentials by scheduling groups, one block's P.V delayed under the next one's exponentials,
// two loops (with and without masks: spills), query groups of a workgroup sharing tiles, pages of many tiles in one load, tiles requested into
// L2 two ahead.
#include "common.h"
#include <algorithm>
#include <type_traits>

struct TreeArgs {
    const void *q, *kc, *vc;
    void* out;
    const int32_t *table, *ctx, *cu;
    const int64_t* mask;                // bit j of row i: node i sees node j; NULL: a chain (nodes 0 .. i)
    float* part;                        // [rows * H][nsplit][64] sums, then [rows * H][nsplit][2] (maximum, denominator)
    long q_rs, o_rs;                    // elements
    float scale_log2;
    uint32_t g_inv;                     // ceil(2^32 / g): qi / g = high word of qi * g_inv for qi < 64 g, g <= 1024
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
// K fragments of a tile out of LDS, and the scores of one query block: lane = query fr, keys fq * 4 + r of each sub-tile
template <typename T> struct TreeKeys { uint4 x[4]; };
__device__ __forceinline__ void tree_keys(TreeKeys<bf16>& k, const uint4* kl, int fr, int fq) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        k.x[2 * s] = tree_k_piece<bf16>(kl, s * 16 + fr, fq);
        k.x[2 * s + 1] = tree_k_piece<bf16>(kl, s * 16 + fr, fq + 4);
    }
}
__device__ __forceinline__ void tree_keys(TreeKeys<float>& k, const uint4* kl, int fr, int fq) {
#pragma unroll
    for (int i = 0; i < 4; ++i) k.x[i] = tree_k_piece<float>(kl, fr, fq * 4 + i);
}
__device__ __forceinline__ void tree_scores(const TreeKeys<bf16>& k, const TreeQuery<bf16>& q, f32x4 (&st)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        st[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k.x[2 * s]), q.x[0], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        st[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k.x[2 * s + 1]), q.x[1], st[s], 0, 0, 0);
    }
}
__device__ __forceinline__ void tree_scores(const TreeKeys<float>& k, const TreeQuery<float>& q, f32x4 (&st)[1]) {
    st[0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 kk = __builtin_bit_cast(f32x4, k.x[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) st[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], q.x[i][e], st[0], 0, 0, 0);
    }
}
// V^T as the A operand.  o[dt] rows i = dims i * 4 + dt: the lane holds dims (fq * 4 + r) * 4 + dt of its query
__device__ __forceinline__ void tree_vt(const TreeTile<bf16>& t, bf16x8 (&vt)[4]) {
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
        vt[dt] = __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
    }
}
__device__ __forceinline__ void tree_pv(const bf16x8 (&vt)[4], const f32x4 (&p)[2], f32x4 (&o)[4]) {
    // P is rounded to bf16, the type of V and of the matrix instruction (the denominator keeps fp32): half a step, 2^-8, of each weight.  The result is
    // 0.0022 .. 0.0024 off the 64-bit one in the 2-norm (its own rounding alone: 0.0017); P in two parts would double the products.
    bf16x8 pf;
#pragma unroll
    for (int e = 0; e < 8; ++e) pf[e] = (bf16)p[e >> 2][e & 3];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[dt], pf, o[dt], 0, 0, 0);
}
__device__ __forceinline__ void tree_vt(const TreeTile<float>& t, f32x4 (&vt)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) vt[r] = t.v[0][r];
}
__device__ __forceinline__ void tree_pv(const f32x4 (&v)[4], const f32x4 (&p)[1], f32x4 (&o)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][dt], p[0][r], o[dt], 0, 0, 0);
}
template <typename T> struct TreeVt;
template <> struct TreeVt<bf16> { typedef bf16x8 type[4]; };
template <> struct TreeVt<float> { typedef f32x4 type[4]; };

// any infinity or NaN in the lane's part of a tile's V rows: exponent bits all ones carry into the sign's place
__device__ __forceinline__ bool tree_any_odd(const TreeTile<bf16>& t) {
    uint32_t any = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint2 w = __builtin_bit_cast(uint2, t.v[s][r]);
            any |= ((w.x & 0x7f807f80u) + 0x00800080u) | ((w.y & 0x7f807f80u) + 0x00800080u);
        }
    return (any & 0x80008000u) != 0;
}
__device__ __forceinline__ bool tree_any_odd(const TreeTile<float>& t) {
    bool any = false;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= !(fabsf(t.v[0][r][e]) < INFINITY);
    return any;
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

// waves per SIMD that the registers are held down to
template <typename T> constexpr int tree_waves(int qb) { return qb == 4 ? 2 : qb == 2 ? 3 : sizeof(T) == 2 ? 4 : 3; }

// WHOLE: a tile lies in one page (pages of 32 rows and more)
template <typename T, int QB, int NW, bool WHOLE>
__global__ __launch_bounds__(NW * 64, tree_waves<T>(QB)) void attn_tree_kernel(TreeArgs a) {
    typedef TreeTile<T> Tile;
    constexpr int SUB = Tile::SUB, KT = 16 * SUB, NP = WHOLE ? 1 : SUB, PK = KT / NP;       // pages of a tile, keys in each
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
    const uint32_t page_bytes = (uint32_t)page_stride * (uint32_t)sizeof(T);

    const auto node_of = [&](int qi) { return a.g == 1 ? qi : (int)__umulhi((uint32_t)qi, a.g_inv); };    // qi / g
    TreeQuery<T> qf[QB];
    uint64_t see[QB];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        const int qi = min(q0 + j * 16 + fr, nq - 1), node = node_of(qi), head = kvh * a.g + qi - node * a.g;
        tree_load_q(qf[j], (const T*)a.q + (long)(r0 + node) * a.q_rs + head * 64, fq);
        see[j] = a.mask ? (uint64_t)a.mask[r0 + node] : (2ull << node) - 1;
    }
    float m[QB], l[QB], lim[QB], shift[QB];                              // lim: the score beyond which m follows; shift = -m (0 while nothing was seen)
    f32x4 o[QB][4];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        m[j] = lim[j] = -INFINITY; l[j] = shift[j] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[j][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __shared__ float so[QB][NW][16][68];
    __shared__ float sm[QB][NW][16], sl[QB][NW][16];
    __shared__ uint32_t s_odd[2];                                        // nodes whose V rows hold infinities or NaN
    if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
    __syncthreads();
    // Every load of the loop is issued whatever the case, through bounds-checked descriptors: what lies behind the wave's last tile
    // moves no data, and the loads stay countable.
    const int mine = t0 + wave < t1 ? (t1 - t0 - wave + NW - 1) / NW : 0;
    const __amdgpu_buffer_rsrc_t tb = buf_rsrc(tab, a.width * 4);
    auto page_of = [&](int i) {                                          // lane s (mod NP): the page of part s of this wave's tile i
        const int key = (t0 + wave + NW * i) * KT + (lane % NP) * PK;
        return (int)buf_load4(tb, i < mine && key < T_all ? (uint32_t)(key >> a.shift) * 4 : BUF_OFF);
    };
    // (The scalar work of a tile counts: a descriptor per page and tensor; with one per 16 keys whatever the page 4 % more for 1 x 130,001 keys,
    // 64 nodes, and 8 % for 32,768, side by side.)
    auto load = [&](Tile& t, int i, int pages) {
        t.live = 0;
        uint32_t ko = lane * 16, vo = (fq * 256 + fr * 4) * (int)sizeof(T);
        asm("" : "+v"(ko), "+v"(vo));                                    // (kept next to the loads: their constants go into the instructions, not registers)
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            const int page = __builtin_amdgcn_readlane(pages, s), key = (t0 + wave + NW * i) * KT + s * PK;
            const bool on = i < mine && key < T_all && (uint32_t)page < (uint32_t)a.n_pages;
            const uint64_t at = (uint64_t)(uint32_t)page * page_bytes + (uint32_t)((key & ((1 << a.shift) - 1)) * 64 * (int)sizeof(T));
            const uint32_t bytes = on ? min(PK, T_all - key) * 64 * (int)sizeof(T) : 0;      // rows behind the sequence read zeros; 0: nothing is read, wherever `at` is
            const __amdgpu_buffer_rsrc_t k = buf_rsrc((const char*)kbase + at, bytes), v = buf_rsrc((const char*)vbase + at, bytes);
#pragma unroll
            for (int n = 0; n < 4 / NP; ++n) t.k[s * (4 / NP) + n] = buf_load16(k, ko + n * 1024);
#pragma unroll
            for (int n = 0; n < 4 * (SUB / NP); ++n) {
                const uint32_t off = vo + (n / 4 * 16 + n % 4) * 64 * (int)sizeof(T);
                typename Tile::vrow& row = t.v[s * (SUB / NP) + n / 4][n % 4];
                if constexpr (sizeof(T) == 2) row = __builtin_bit_cast(typename Tile::vrow, buf_load8(v, off));
                else row = __builtin_bit_cast(typename Tile::vrow, buf_load16(v, off));
            }
            if (on) {
                if constexpr (NP == SUB) t.live |= 1u << s;
                else t.live = key + 16 < T_all ? 3u : 1u;
            }
        }
    };
    TreeKeys<T> kf;
    typename TreeVt<T>::type vt;
    uint32_t win[QB];                                                    // bit s * 16 + r: the query sees key s * 16 + fq * 4 + r of the tile
    bool edge;
    auto open = [&](Tile& t, int i) {                                    // the tile leaves its registers: K over LDS into fragments, V turned
        const int key0 = (t0 + wave + NW * i) * KT;
        uint4* kl = reinterpret_cast<uint4*>(&so[0][wave][0][0]);
        tree_stage_k(t, kl, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        tree_keys(kf, kl, fr, fq);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        edge = key0 + KT > ctx || t.live != (1u << SUB) - 1;             // wave-uniform: only the tiles with nodes, or with pages missing
        if (edge) {
            // A node's V row with infinities or NaN belongs to the queries that see it and to no other: 0 x inf in the MFMA would
            // reach them all.  Such elements are taken out here and added to the seeing queries in the merge.
            if (__any(tree_any_odd(t))) {
                uint32_t odd = 0;
#pragma unroll
                for (int s = 0; s < SUB; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {                            // (rows behind the sequence were read as zeros)
                        const bool bad = key0 + s * 16 + fq * 4 + r >= ctx && tree_odd(t, s, r);
                        odd |= (uint32_t)bad << (s * 16 + r);
                        if (bad) tree_clean_v(t, s, r);
                    }
                if (odd) {
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (((0x000f000fu >> c) & 1) && ((odd >> c) & 1)) {
                            const int node = key0 + c + fq * 4 - ctx;
                            atomicOr(&s_odd[node >> 5 & 1], 1u << (node & 31));
                        }
                }
            }
            const int nb = key0 - ctx;                                   // node number of the tile's first key; negative: -nb context rows first
            uint32_t there = 0;
#pragma unroll
            for (int s = 0; s < SUB; ++s)
                if ((t.live >> s) & 1) there |= 0xffffu << (16 * s);
            if (T_all - key0 < KT) there &= (1u << (T_all - key0)) - 1;
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                const uint32_t w = nb >= 64 ? 0 : nb >= 0 ? (uint32_t)(see[j] >> nb) : nb <= -32 ? ~0u : ((uint32_t)see[j] << -nb) | ((1u << -nb) - 1);
                win[j] = (w & there) >> (fq * 4);
            }
        }
        if constexpr (QB == 4) tree_vt(t, vt);
    };
    // Query block by query block, so that the matrix unit works under the vector unit: the next block's scores and the last block's
    // products run while one block's exponentials are taken.
    auto use = [&](const Tile& t) {
        f32x4 st[2][SUB];
        tree_scores(kf, qf[0], st[0]);
#pragma unroll
        for (int j = 0; j < QB; ++j) {
            f32x4 (&p)[SUB] = st[j & 1];
            if (edge) {
#pragma unroll
                for (int s = 0; s < SUB; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[s][r] = win[j] & (1u << (s * 16 + r)) ? p[s][r] : -INFINITY;
            }
            // The shift of the exponentials needs to be near the maximum, not the maximum: it follows only when a score lies more than
            // 8 (a factor of 256 in a weight) above it, so that most tiles reduce nothing over lanes and scale nothing.
            float top = p[0][0];
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, p[s][r]);
            if (__any(top > lim[j])) {                                   // scale > 0: the maximum commutes with it
                float mx = fmaxf(top, __shfl_xor(top, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                if (mx > lim[j]) {                                       // by the query's own scores alone: its four lanes agree
                    const float alpha = __builtin_amdgcn_exp2f(m[j] - mx * a.scale_log2);
                    m[j] = mx * a.scale_log2;
                    lim[j] = mx + 8.0f / a.scale_log2;
                    shift[j] = -m[j];
                    l[j] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[j][dt][r] *= alpha;
                }
            }
            if (j + 1 < QB) tree_scores(kf, qf[j + 1], st[(j + 1) & 1]);
            float sum = 0.f;
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(p[s][r], a.scale_log2, shift[j]));
                    p[s][r] = e;
                    sum += e;
                }
            l[j] += sum;
            if constexpr (QB != 4) {                                     // (the tile's registers are still its own: fewer live at once)
                if (j == 0) tree_vt(t, vt);
            }
            tree_pv(vt, p, o[j]);
        }
    };
    if (mine > 0) {
        Tile A;
        int after = page_of(0), next = page_of(1);                       // a page is requested one tile's loads ahead of its use
        load(A, 0, after);
        if constexpr (QB == 4) {                               // one set of registers: the next tile is requested once this one has left them
            for (int i = 0; i < mine; ++i) {
                after = page_of(i + 2);
                open(A, i);
                load(A, i + 1, next);
                next = after;
                __builtin_amdgcn_sched_barrier(0);                       // (left alone the compiler sinks the loads behind the products)
                use(A);
            }
        } else {
            Tile B;
            for (int i = 0;; i += 2) {
                after = page_of(i + 2);
                load(B, i + 1, next);
                __builtin_amdgcn_sched_barrier(0);
                open(A, i);
                use(A);
                if (i + 1 >= mine) break;
                next = page_of(i + 3);
                load(A, i + 2, after);
                __builtin_amdgcn_sched_barrier(0);
                open(B, i + 1);
                use(B);
                if (i + 2 >= mine) break;
            }
        }
    }
    // ---- merge of the waves: a thread owns DPT dims of a query of every block
    constexpr int DPT = 1024 / (NW * 64);
    typedef float part_t __attribute__((ext_vector_type(DPT)));
    const int mq = threadIdx.x / (64 / DPT), md = threadIdx.x % (64 / DPT) * DPT;
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        float lt = l[j];
        lt += __shfl_xor(lt, 16, 64);
        lt += __shfl_xor(lt, 32, 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f32x4*>(&so[j][wave][fr][(fq * 4 + r) * 4]) = f32x4{o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]};
        if (fq == 0) { sm[j][wave][fr] = m[j]; sl[j][wave][fr] = lt; }
    }
    __syncthreads();
    const uint64_t odd_nodes = ((uint64_t)s_odd[1] << 32) | s_odd[0];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        const int qi = q0 + j * 16 + mq;
        if (qi < nq) {
            float M = -INFINITY, L = 0.f, mw[NW], lw[NW];
            part_t acc = {}, ov[NW];
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                mw[k] = sm[j][k][mq]; lw[k] = sl[j][k][mq];
                ov[k] = *reinterpret_cast<const part_t*>(&so[j][k][mq][md]);
                M = fmaxf(M, mw[k]);
            }
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const float sc = mw[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[k] - M);
                L += lw[k] * sc;                                         // (a wave whose scores are all NaN has no maximum, and its NaN goes on)
#pragma unroll
                for (int d = 0; d < DPT; ++d) acc[d] += ov[k][d] * sc;
            }
            const int node = node_of(qi), head = kvh * a.g + qi - node * a.g;
            const long row = r0 + node;
            uint64_t odd = odd_nodes;
            if (odd) {                                                   // infinities and NaN of the nodes this query sees
                odd &= a.mask ? (uint64_t)a.mask[row] : (2ull << node) - 1;
                for (; odd; odd &= odd - 1) {
                    const int key = ctx + __builtin_ctzll(odd);
                    const T* vp = vbase + tab[key >> a.shift] * page_stride + (long)(key & ((1 << a.shift) - 1)) * 64 + md;
#pragma unroll
                    for (int d = 0; d < DPT; ++d) {
                        const float v = to_f32<T>(vp[d]);
                        if (!(fabsf(v) < INFINITY)) acc[d] += v;
                    }
                }
            }
            if (a.nsplit == 1) {
                typedef T out_t __attribute__((ext_vector_type(DPT)));
                const float inv = L == 0.f ? 0.f : 1.0f / L;             // a row that sees nothing is zero
                out_t y;
#pragma unroll
                for (int d = 0; d < DPT; ++d) y[d] = from_f32<T>(acc[d] * inv);
                *reinterpret_cast<out_t*>((T*)a.out + row * a.o_rs + head * 64 + md) = y;
            } else {
                const long at = (row * a.H + head) * a.nsplit + split;
                *reinterpret_cast<part_t*>(a.part + at * 64 + md) = acc;
                if (md == 0) {
                    float* ml = a.part + (long)a.rows * a.H * a.nsplit * 64 + at * 2;
                    ml[0] = M; ml[1] = L;
                }
            }
        }
    }
}

// joins the workgroups' partial sums of a (row, head): one wave, a lane per dimension; or (many parts) four waves that deal them out
template <typename T, int W>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs a) {
    const int b = blockIdx.x, node = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = W == 4 ? blockIdx.z : blockIdx.z * 4 + wave, first = W == 4 ? wave : 0;
    const int r0 = a.cu[b];
    if (a.ctx[b] < 0 || r0 < 0) return;
    if (node >= min(min(a.cu[b + 1] - r0, a.max_nodes), a.rows - r0)) return;
    if (W == 1 && head >= a.H) return;
    const long row = r0 + node, at = (row * a.H + head) * a.nsplit;
    const float* ml = a.part + (long)a.rows * a.H * a.nsplit * 64 + at * 2;
    const float mv = lane < a.nsplit ? ml[2 * lane] : -INFINITY;
    const float lv = lane < a.nsplit ? ml[2 * lane + 1] : 0.f;
    float acc = 0.f, M = 0.f, w = 0.f, L = 0.f;
    for (int s0 = first; s0 < a.nsplit; s0 += 4 * W) {                   // four parts under way
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a.part[(at + min(s0 + i * W, a.nsplit - 1)) * 64 + lane];
        if (s0 == first) {
            M = wave_max(mv);
            w = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - M);
            L = wave_sum(lv * w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * W;
            const float ws = __shfl(w, s & 63, 64);
            if (s < a.nsplit) acc += v[i] * ws;                          // (a part that saw nothing holds zeros)
        }
    }
    if constexpr (W == 4) {
        __shared__ float red[4][64];
        red[wave][lane] = acc;
        __syncthreads();
        if (wave) return;
        acc = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    }
    ((T*)a.out)[row * a.o_rs + head * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : acc / L);
}

// How the work is cut: qb blocks of 16 queries per wave (up to two in fp32, where 8 registers of the second go through scratch at three waves per
// SIMD: the sweep below has it so), nw waves per workgroup over the keys, `blocks`
// workgroups over the queries of a (request, kv head), `split` over its keys.  More blocks per wave save key traffic and the turning of K
// and V, but hold more registers (four, three, two waves per SIMD at one, two, four blocks) and start and end longer; eight waves finish a
// request sooner, workgroups of four overlap one's start and end with another's tiles; splitting fills the chip but needs the join.
// The choice is the least of an estimate in us, fitted to 624 measurements of 33 shapes (it takes 1.3 % more than the best of them, in the
// mean).  Some of them in bf16, us a call in graph replays on the same inputs at the time of that sweep, with qb x nw (requests x context, nodes, heads / kv heads):
//                                  1 x 4   1 x 8   2 x 4   2 x 8   4 x 4   4 x 8
//   1 x 130,001, 64, 16/4           114     111      75      74      66      64
//   32 x 2,200, 64, 16/16            95      93      58      74      52      59
//   32 x 2,200, 26, 16/16            56      55      46      51
//   48 x 300, 64, 16/16              27      38      24      42      26      37
//   16 x 536, 64, 16/4             14.0    16.5    11.2    15.8    12.3    12.8
//   16 x 536, 26, 16/16             9.4    10.1     9.9     9.7
//   1 x 300, 64, 16/16              5.5     5.7     7.0     7.4     9.9    10.6
//   16 x 536, 1, 16/16              7.4     6.9
// and in fp32: 64 x 536, 26, 16/16 65 / 85 / 57 / 75; 1 x 4,000, 26, 16/16 15 / 14 / 18 / 18.
struct TreeShape { int qb, nw, blocks, split; };
struct TreeCost {
    float issue[3], tile[3];            // of one tile by qb: of the SIMD's issue slots, and of a wave alone
    float ends[3], ends4;               // start and end of a workgroup of eight waves, and the factor for four
    float join, part;                   // second launch (and 0.05 per part it joins); per MB of partial sums
    float mem, again;                   // per MB of keys and values; share of it for every further workgroup that reads them
    float both;                         // share of the shorter of compute and memory that is not hidden
};
static TreeShape tree_shape(int B, int Hkv, int g, int max_nodes, int max_ctx, int kt) {
    static const TreeCost bf{{.354f, .432f, .684f}, {.55f, .69f, 1.02f}, {2.24f, 3.89f, 6.1f}, .79f, 2.6f, .26f, 1 / 7800.f, .08f, .43f};
    static const TreeCost fp{{.496f, 1.048f, 0.f}, {.734f, 1.26f, 0.f}, {2.57f, 4.68f, 0.f}, .62f, 2.45f, .28f, 1 / 7400.f, .17f, .32f};
    const bool bf16s = kt == 32;
    const TreeCost& c = bf16s ? bf : fp;
    const int nq = max_nodes * g;
    const long tiles = ((long)max_ctx + max_nodes + kt - 1) / kt;
    const float kb = (float)B * Hkv * tiles * 8.192f;                     // a tile's K and V are 8 KB in either type
    TreeShape best{0, 0, 0, 0};
    float least = 0.f;
    for (int q = 0; q < (bf16s ? 3 : 2) && (q == 0 || nq > 8 << q); ++q) {
        const int qb = 1 << q;
        const long blocks = ceil_div(nq, 16 * qb), base = (long)B * Hkv * blocks;
        if (Hkv * blocks > 65535) continue;                              // (no such grid)
        const float mem = kb * c.mem * (1.f + c.again * (blocks - 1));
        for (int nw = 8; nw >= 4; nw -= 4) {
            const long room = 256 * ((q == 0 && bf16s ? 16 : q == 2 ? 8 : 12) / nw);       // workgroups at a time
            const long most = std::min<long>(std::min<long>(room / base, TREE_MAX_SPLIT), tiles / (2 * nw));    // (a wave keeps two tiles)
            long last = 0;
            for (int part = 2; part >= 0; --part) {                      // one, half of the most, the most
                const long split = part == 2 ? 1 : part == 1 ? most / 2 : most;
                if (split <= last) continue;
                last = split;
                const long groups = base * split, rounds = (groups + room - 1) / room, deep = (tiles + nw * split - 1) / (nw * split);
                const long per_cu = (std::min(groups, room) + 255) / 256;
                const float tile = std::max(c.tile[q], c.issue[q] * (per_cu * nw * .25f));
                const float work = rounds * (c.ends[q] * (nw == 4 ? c.ends4 : 1.f) + deep * tile);
                float t = std::max(work, mem) + c.both * std::min(work, mem);
                if (split > 1) t += c.join + .05f * split + c.part * ((float)B * nq * Hkv * split * 512e-6f);
                if (!best.qb || t < least) { best = TreeShape{qb, nw, (int)blocks, (int)split}; least = t; }
            }
        }
    }
    return best;
}
static bool tree_shape_ok(int rows, int B, int H, int Hkv, int max_nodes, int max_ctx) {
    return rows >= 0 && B >= 0 && B <= 65535 && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 65535 && H / Hkv <= 1024 && max_nodes > 0 && max_nodes <= TREE_MAX_NODES && max_ctx >= 0;
}

static size_t tree_bytes(int rows, int H, int split) { return split <= 1 ? 0 : (size_t)rows * H * split * 66 * sizeof(float); }

extern "C" size_t valle_attn_tree_workspace_bytes(int rows, int B, int max_nodes, int max_ctx, int H, int Hkv, int dtype) {
    if (!tree_shape_ok(rows, B, H, Hkv, max_nodes, max_ctx) || B == 0) return 0;
    return tree_bytes(rows, H, tree_shape(B, Hkv, H / Hkv, max_nodes, max_ctx, dtype == VALLE_BF16 ? 32 : 16).split);
}

template <typename T>
static void tree_launch(const TreeArgs& a, const TreeShape& t, int B, hipStream_t s) {
    const dim3 grid(a.nsplit, a.Hkv * t.blocks, B);
    auto go = [&](auto qb, auto nw) {
        constexpr int QB = decltype(qb)::value, NW = decltype(nw)::value;
        if (sizeof(T) == 4 || a.shift >= 5) attn_tree_kernel<T, QB, NW, true><<<grid, NW * 64, 0, s>>>(a);
        else if constexpr (sizeof(T) == 2) attn_tree_kernel<T, QB, NW, false><<<grid, NW * 64, 0, s>>>(a);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    if (t.qb == 1) t.nw == 8 ? go(one, eight) : go(one, four);
    else if (t.qb == 2) t.nw == 8 ? go(two, eight) : go(two, four);
    else if constexpr (sizeof(T) == 2) t.nw == 8 ? go(four, eight) : go(four, four);
    if (a.nsplit > 16) attn_tree_join_kernel<T, 4><<<dim3(B, a.max_nodes, a.H), 256, 0, s>>>(a);
    else if (a.nsplit > 1) attn_tree_join_kernel<T, 1><<<dim3(B, a.max_nodes, ceil_div(a.H, 4)), 256, 0, s>>>(a);
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
    VALLE_REQUIRE(((int64_t)Hkv << shift) * 64 * 4 <= INT32_MAX, VALLE_E_ARG, "valle_attn_tree: a page of %d kv heads is too large", Hkv);
    VALLE_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, VALLE_E_ARG, "valle_attn_tree: softmax_scale must be positive");
    const int vec = 16 / (int)dtype_size(dtype);
    const void* ptrs[] = {q, kcache, vcache, out};
    for (const void* p : ptrs) VALLE_REQUIRE(((uintptr_t)p & 15) == 0, VALLE_E_ARG, "valle_attn_tree: tensors must be 16-byte aligned");
    VALLE_REQUIRE(q_row_stride >= 0 && q_row_stride % vec == 0 && out_row_stride % vec == 0, VALLE_E_ARG, "valle_attn_tree: rows of q and out must stay 16-byte aligned");
    VALLE_REQUIRE(rows <= 1 || out_row_stride >= (int64_t)H * 64, VALLE_E_ARG, "valle_attn_tree: rows of out overlap");
    if (B == 0 || rows == 0) return VALLE_OK;
    TreeArgs a{q, kcache, vcache, out, block_table, ctx_len, cu_rows, tree_mask, (float*)workspace, q_row_stride, out_row_stride,
               softmax_scale * 1.4426950408889634f, (uint32_t)(((1ull << 32) + H / Hkv - 1) / (H / Hkv)), max_blocks, n_pages, shift, rows, H, Hkv, H / Hkv, max_nodes, 1};
    const TreeShape shape = tree_shape(B, Hkv, a.g, max_nodes, max_ctx, dtype == VALLE_BF16 ? 32 : 16);
    a.nsplit = shape.split;
    const size_t need = tree_bytes(rows, H, shape.split);
    VALLE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), VALLE_E_WORKSPACE,
                  "valle_attn_tree: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    VALLE_REQUIRE(shape.qb, VALLE_E_ARG, "valle_attn_tree: %d heads are too many", H);
    if (dtype == VALLE_BF16) tree_launch<bf16>(a, shape, B, (hipStream_t)stream);
    else tree_launch<float>(a, shape, B, (hipStream_t)stream);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}
