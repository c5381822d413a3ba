// The bookkeeping and the data movement of a paged KV cache: pages of `page_size` rows (a power of two), per layer
// [n_pages][Hkv][page_size][64], a head's keys in one page contiguous as in the slot cache of valle_rope_kv.
//   valle_page_plan          block tables, slot map, positions and tree masks from the requests' lengths
//   valle_rope_kv_paged      RoPE on q and k rows, k and v into the pages the slot map names
//   valle_paged_kv_commit    the accepted path of a draft tree to the end of the context, all layers; valle_paged_kv_commit_served:
//                            for the requests that the plan served, inside the pages they hold
// The reference has no counterpart: it recomputes the whole sequence per step (models/base.py:521, use_cache=False).
#include "common.h"

// ------------------------------------------------------------------------------------ page plan
// need_b = ceil(len_new_b / page), held_b = pages in hand.  held > need: the surplus goes back on the free stack; held < need:
// the difference comes off it, in request order, until it runs dry.  With F = free pages after all returns and x the running
// number of a page over all requests, both are one formula: page x <-> free_list[F - 1 - x] (taking the same pages back and
// forth leaves the stack as it was).
#define PLAN_MAX_B 4096
struct PlanArgs {
    const int32_t *len_old, *len_new;
    int32_t* table;
    const int32_t* nb_in; int32_t* nb_out;
    int32_t* free_list;
    const int32_t* fc_in; int32_t* fc_out;
    int32_t *status, *cu, *slots, *pos;
    const int32_t* parents; int64_t* mask;                    // parents NULL: plain rows, chains; mask NULL: none is written
    int32_t* ticket;
    int B, width, n_pages, shift, max_rows;
};

__device__ __forceinline__ long plan_wave_scan(long v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}
// exclusive prefix of v over the workgroup's threads, and the total
template <int NT>
__device__ __forceinline__ long plan_block_scan(long v, long* tmp, long& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long inc = plan_wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) tmp[wave] = inc;
    __syncthreads();
    long base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const long t = tmp[w];
        if (w < wave) base += t;
        sum += t;
    }
    total = sum;
    return base + inc - v;
}
// first b in [0, B) with incl[b] > x (the caller knows that there is one)
__device__ __forceinline__ int plan_find(const int* incl, int B, int x) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (incl[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ int plan_slot(const PlanArgs& a, int b, int p, bool served) {
    if (!served) return -1;
    const int blk = p >> a.shift;                              // served: len_new <= width << shift, so blk < width
    const int page = a.table[(size_t)b * a.width + blk];
    return page >= 0 && page < a.n_pages ? (page << a.shift) + (p & ((1 << a.shift) - 1)) : -1;
}
// the mask of row i of a chain: itself and the rows in front of it (from row 63 on a word holds no more)
__device__ __forceinline__ int64_t plan_chain(int i) { return i < 63 ? (int64_t)((2ull << i) - 1) : -1; }
// plain rows: row r belongs to the request whose end lies behind it; rows behind the last request are padding (slot -1)
__device__ __forceinline__ void plan_row(const PlanArgs& a, const int* ends, const int* stat, int r) {
    int slot = -1, p = 0;
    int64_t m = 0;
    if (r < ends[a.B - 1]) {
        const int b = plan_find(ends, a.B, r), i = r - (b ? ends[b - 1] : 0);
        p = a.len_old[b] + i;
        slot = plan_slot(a, b, p, stat[b] == 0);
        m = plan_chain(i);
    }
    a.slots[r] = slot; a.pos[r] = p;
    if (a.mask) a.mask[r] = m;
}
// tree rows of one request: lane i = node i, its slot given.  Ancestor bits and depths by pointer doubling (6 rounds cover 64 levels).
__device__ __forceinline__ void plan_tree(const PlanArgs& a, int len_old, int start, int n, int slot, int lane) {
    int up = -1;
    if (lane < n && start + lane < a.max_rows) {
        const int p = a.parents[start + lane];
        if (p >= 0 && p < lane) up = p;
    }
    uint64_t m = 1ull << lane;
    int depth = up >= 0;
#pragma unroll
    for (int it = 0; it < 6; ++it) {
        const int src = up >= 0 ? up : lane;
        const uint32_t lo = __shfl((uint32_t)m, src, 64), hi = __shfl((uint32_t)(m >> 32), src, 64);
        const int du = __shfl(depth << 8 | (up & 255), src, 64);         // depth and parent in one word: both stay below 64 (parent 255: none)
        if (up >= 0) {
            m |= ((uint64_t)hi << 32) | lo;
            depth += du >> 8;
            up = (du & 255) == 255 ? -1 : du & 255;
        }
    }
    const int r = start + lane;
    if (lane < n && r < a.max_rows) { a.slots[r] = slot; a.pos[r] = len_old + depth; a.mask[r] = (int64_t)m; }
}

// inclusive sum over the lanes of a wave, on the cross-lane paths of the vector unit
template <int CTRL, int ROWS>
__device__ __forceinline__ int plan_dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int plan_lane_scan(int v) {
    v = plan_dpp_add<0x111, 0xf>(v);          // row_shr 1, 2, 4, 8: sums inside each row of 16
    v = plan_dpp_add<0x112, 0xf>(v);
    v = plan_dpp_add<0x114, 0xf>(v);
    v = plan_dpp_add<0x118, 0xf>(v);
    v = plan_dpp_add<0x142, 0xa>(v);          // row_bcast 15: the row before, into rows 1 and 3
    return plan_dpp_add<0x143, 0xc>(v);       // row_bcast 31: rows 0 and 1, into rows 2 and 3
}

// Up to 64 E requests, E neighbours per lane of a wave.  Every workgroup works the whole batch out for itself (at E = 1 every wave: the sums cost
// a few dozen cycles; beyond, its first wave, between two barriers), and what the rows need is taken from the state as it was (a page that changes hands in this very call is looked up where it
// came from), so nobody waits for anybody.  Only the counters may be read and written in one place (n_blocks_out may be n_blocks_in):
// the last workgroup to have read them, by the ticket, writes them.  The latency is two dependent memory round trips and the ticket's.
// One workgroup up to 1,024 rows or 16 trees, then one per as many more; us when it was built, in the general form / in one workgroup / so: 16
// trees of 26 nodes 7.3 / 3.5 / 3.6, 64 trees of 26 - / 7.2 / 3.8, 64 prompts of 700 rows - / 6.3 (their rows in a second launch) / 3.9; with E = 8
// 128 trees of 26 8.3 / - / 5.8, 512 of 8 9.0 / - / 6.3, 512 requests with a row each 6.0 / - / 5.1 (every wave for itself there too: 9.7, 17, 22).
// 16 trees of 26 and 64 prompts of 305 .. 761 rows, 50 plans in a graph: 4.3 and 3.7.
template <int E>
__global__ __launch_bounds__(1024) void page_plan_wave_kernel(PlanArgs a) {
    __shared__ int s_f[64 * E], s_from[64 * E], s_end[64 * E], s_lo[64 * E], s_held[64 * E], s_q[64 * E], s_sum[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int lo[E], ln[E], held[E];
    if constexpr (E == 1) {
        const int b = min(lane, a.B - 1);
        lo[0] = a.len_old[b]; ln[0] = a.len_new[b]; held[0] = a.nb_in[b];
    } else if (threadIdx.x < 64 * E) {                                   // whole lines, for the first wave
        const int b = min((int)threadIdx.x, a.B - 1);
        s_lo[threadIdx.x] = a.len_old[b]; s_f[threadIdx.x] = a.len_new[b]; s_held[threadIdx.x] = a.nb_in[b];
    }
    const int fc = min(max(*a.fc_in, 0), a.n_pages);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");         // the counters are in registers before any of them is written over
    __syncthreads();
    int turn = 0;
    if (gridDim.x > 1 && threadIdx.x == 0) turn = atomicAdd(a.ticket, 1);
    const long cap = (long)a.width << a.shift;
    int want[E], rows[E], f[E], q[E], end[E], freed = 0, F = 0, all = 0, taken = 0;
    bool valid[E], ok[E], served[E];
    if (E == 1 || wave == 0) {
        if constexpr (E > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) { lo[e] = s_lo[lane * E + e]; ln[e] = s_f[lane * E + e]; held[e] = s_held[lane * E + e]; }
        }
        int low = 0, high = 0, gone = 0, asked = 0;                          // of the lane's requests: rows (16 bits and the rest), pages back, pages asked for
#pragma unroll
        for (int e = 0; e < E; ++e) {
            valid[e] = lane * E + e < a.B && lo[e] >= 0 && ln[e] >= 0 && lo[e] <= cap && ln[e] <= cap && held[e] >= 0 && held[e] <= a.width && !(a.parents && ln[e] - lo[e] > 64);
            want[e] = valid[e] ? (int)(((long)ln[e] + (1 << a.shift) - 1) >> a.shift) : 0;
            rows[e] = valid[e] && ln[e] > lo[e] ? ln[e] - lo[e] : 0;
            low += rows[e] & 0xffff; high += rows[e] >> 16;
        }
        long at = (long)plan_lane_scan(low) - low + ((long)(plan_lane_scan(high) - high) << 16);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += rows[e];
            end[e] = (int)min(at, (long)INT32_MAX);
            ok[e] = valid[e] && at <= a.max_rows;
            f[e] = gone += ok[e] ? max(held[e] - want[e], 0) : 0;
            q[e] = asked += ok[e] ? max(want[e] - held[e], 0) : 0;
        }
        const int f_all = plan_lane_scan(gone), q_all = plan_lane_scan(asked);
        freed = __builtin_amdgcn_readlane(f_all, 63); F = fc + freed; all = __builtin_amdgcn_readlane(end[E - 1], 63);
        int last = 0;                                                        // pages taken up to the lane's last served request that takes some
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int need = ok[e] ? max(want[e] - held[e], 0) : 0;
            f[e] += f_all - gone; q[e] += q_all - asked;
            served[e] = ok[e] && (need == 0 || q[e] <= F);
            if (served[e] && need > 0) last = q[e];
        }
        const uint64_t takers = __ballot(last > 0);
        taken = takers ? __shfl(last, 63 - __builtin_clzll(takers), 64) : 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {                                    // (E == 1: every wave writes the same and reads what it wrote)
            const int b = lane * E + e;
            s_f[b] = f[e]; s_from[b] = want[e] - f[e] + (ok[e] ? max(held[e] - want[e], 0) : 0);
            s_end[b] = end[e]; s_lo[b] = lo[e]; s_held[b] = served[e] ? held[e] : -1; s_q[b] = q[e];
        }
    }
    if constexpr (E == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        if (threadIdx.x == 0) { s_sum[0] = freed; s_sum[1] = all; }
        __syncthreads();
        freed = s_sum[0]; all = s_sum[1]; F = fc + freed;
    }
    auto page_x = [&](int x) -> int {                                    // the page a request takes as number x: one given back in this call, or off the stack
        if (x < freed) {
            const int b = plan_find(s_f, a.B, x);
            return a.table[(size_t)b * a.width + s_from[b] + x];
        }
        const int src = F - 1 - x;
        return src >= 0 && src < a.n_pages ? a.free_list[src] : -1;
    };
    auto slot_of = [&](int b, int p) -> int {                            // of cached row p, a new one, of request b
        const int held_b = s_held[b], blk = p >> a.shift;
        if (held_b < 0) return -1;
        const int page = blk < held_b ? a.table[(size_t)b * a.width + blk] : page_x((b ? s_q[b - 1] : 0) + blk - held_b);
        return page >= 0 && page < a.n_pages ? (page << a.shift) + (p & ((1 << a.shift) - 1)) : -1;
    };
    for (int b = blockIdx.x * 16 + wave; b < a.B; b += gridDim.x * 16) {
        const int f0 = b ? s_f[b - 1] : 0, back = s_f[b] - f0, q0 = b ? s_q[b - 1] : 0, need = s_q[b] - q0, held_b = s_held[b];
        int32_t* tab = a.table + (size_t)b * a.width;
        for (int k = lane; k < back; k += 64) {
            const int dst = F - 1 - (f0 + k);
            if (dst >= 0 && dst < a.n_pages) a.free_list[dst] = tab[s_from[b] + f0 + k];
        }
        if (held_b >= 0)
            for (int k = lane; k < need; k += 64) tab[held_b + k] = page_x(q0 + k);
        if (a.parents) {
            const int start = b ? s_end[b - 1] : 0, n = s_end[b] - start;
            plan_tree(a, s_lo[b], start, n, lane < n ? slot_of(b, s_lo[b] + lane) : -1, lane);
        }
    }
    for (long r = (a.parents ? all : 0) + (long)blockIdx.x * 1024 + threadIdx.x; r < a.max_rows; r += gridDim.x * 1024) {
        int slot = -1, pos = 0;
        int64_t m = 0;
        if (r < all) {
            const int b = plan_find(s_end, a.B, (int)r), i = (int)r - (b ? s_end[b - 1] : 0);
            pos = s_lo[b] + i;
            slot = slot_of(b, pos);
            m = plan_chain(i);
        }
        a.slots[r] = slot; a.pos[r] = pos;
        if (a.mask) a.mask[r] = m;
    }
    if (wave == 0 && (gridDim.x == 1 || __builtin_amdgcn_readfirstlane(turn) == (int)gridDim.x - 1)) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int b = lane * E + e;
            if (b < a.B) {
                a.cu[b + 1] = end[e];
                a.status[b] = !valid[e] ? 2 : !ok[e] ? 3 : served[e] ? 0 : 1;
                a.nb_out[b] = served[e] ? want[e] : held[e];
            }
        }
        if (lane == 0) {
            a.cu[0] = 0; *a.fc_out = F - taken;
            if (gridDim.x > 1) *a.ticket = 0;
        }
    }
}

// One workgroup plans the batch, five rounds of barriers (4,096 requests, a row each: 14 us) (a request per thread, up to four); ROWS: it also fills the rows (no trees), else page_rows_kernel does.
template <int NT, bool ROWS>
__global__ __launch_bounds__(NT) void page_plan_kernel(PlanArgs a) {
    constexpr int E = 4;
    __shared__ int s_f[NT * E], s_a[NT * E], s_held[NT * E], s_end[NT * E];
    __shared__ long tmp[NT / 64];
    const int tid = threadIdx.x, per = (a.B + NT - 1) / NT, b0 = tid * per;
    const long cap = (long)a.width << a.shift;
    const int fc = min(max(*a.fc_in, 0), a.n_pages);
    int held[E], want[E], rows[E];
    bool ok[E], valid[E];
    long sum = 0, total;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        held[e] = want[e] = rows[e] = 0; ok[e] = valid[e] = false;
        const int b = b0 + e;
        if (e < per && b < a.B) {
            const int lo = a.len_old[b], ln = a.len_new[b];
            held[e] = a.nb_in[b];
            valid[e] = lo >= 0 && ln >= 0 && lo <= cap && ln <= cap && held[e] >= 0 && held[e] <= a.width && !(a.parents && ln - lo > 64);
            want[e] = valid[e] ? (int)(((long)ln + (1 << a.shift) - 1) >> a.shift) : 0;
            rows[e] = valid[e] && ln > lo ? ln - lo : 0;
        }
        sum += rows[e];
    }
    long at = plan_block_scan<NT>(sum, tmp, total);
    long moved = 0;                                            // (pages given back) << 32 | pages asked for
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int b = b0 + e;
        if (e < per && b < a.B) {
            if (b == 0) a.cu[0] = 0;
            at += rows[e];
            const int end = (int)min(at, (long)INT32_MAX);
            a.cu[b + 1] = end; s_end[b] = end;
            ok[e] = valid[e] && at <= a.max_rows;
            if (ok[e]) moved += ((long)max(held[e] - want[e], 0) << 32) + max(want[e] - held[e], 0);
        }
    }
    long pre = plan_block_scan<NT>(moved, tmp, total);
    const int freed = (int)(total >> 32), F = fc + freed;      // (B * width is bounded on the host: both halves stay below 2^31)
    int f = (int)(pre >> 32), q = (int)(pre & 0xffffffff), taken = 0;
    int stat[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int b = b0 + e;
        stat[e] = 0;
        if (e < per && b < a.B) {
            const int back = ok[e] ? max(held[e] - want[e], 0) : 0, need = ok[e] ? max(want[e] - held[e], 0) : 0;
            f += back; q += need;
            s_f[b] = f; s_a[b] = q; s_held[b] = held[e];
            const bool served = ok[e] && (need == 0 || q <= F);
            if (served && need) taken = q;                     // q ascends: the last served one is the largest
            stat[e] = !valid[e] ? 2 : !ok[e] ? 3 : served ? 0 : 1;
            a.status[b] = stat[e];
            a.nb_out[b] = served ? want[e] : held[e];
        }
    }
    // the number of pages taken: maximum over the threads
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) taken = max(taken, __shfl_xor(taken, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) tmp[tid >> 6] = taken;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) taken = max(taken, (int)tmp[w]);
    if (tid == 0) *a.fc_out = F - taken;
    for (int x = tid; x < freed; x += NT) {
        const int b = plan_find(s_f, a.B, x), p0 = b ? s_f[b - 1] : 0;
        const int j = s_held[b] - (s_f[b] - p0) + x - p0, dst = F - 1 - x;
        if (dst >= 0 && dst < a.n_pages) a.free_list[dst] = a.table[(size_t)b * a.width + j];
    }
    __syncthreads();
    for (int x = tid; x < taken; x += NT) {
        const int b = plan_find(s_a, a.B, x), p0 = b ? s_a[b - 1] : 0, src = F - 1 - x;
        a.table[(size_t)b * a.width + s_held[b] + x - p0] = src < a.n_pages ? a.free_list[src] : -1;
    }
    if constexpr (ROWS) {
        __syncthreads();                                       // the tables are whole, s_f is free
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < per && b0 + e < a.B) s_f[b0 + e] = stat[e];
        __syncthreads();
        for (int r = tid; r < a.max_rows; r += NT) plan_row(a, s_end, s_f, r);
    }
}

__global__ __launch_bounds__(256) void page_rows_kernel(PlanArgs a) {
    __shared__ int s_end[PLAN_MAX_B], s_stat[PLAN_MAX_B];
    for (int b = threadIdx.x; b < a.B; b += 256) { s_end[b] = a.cu[b + 1]; s_stat[b] = a.status[b]; }
    __syncthreads();
    if (a.parents) {
        for (int b = blockIdx.x * 4 + (threadIdx.x >> 6); b < a.B; b += gridDim.x * 4) {
            const int start = b ? s_end[b - 1] : 0;
            const int i = threadIdx.x & 63, n = s_end[b] - start;
            plan_tree(a, a.len_old[b], start, n, i < n ? plan_slot(a, b, a.len_old[b] + i, s_stat[b] == 0) : -1, i);
        }
        for (long r = (long)s_end[a.B - 1] + blockIdx.x * 256 + threadIdx.x; r < a.max_rows; r += gridDim.x * 256) {
            a.slots[r] = -1; a.pos[r] = 0; a.mask[r] = 0;
        }
    } else {
        for (long r = (long)blockIdx.x * 256 + threadIdx.x; r < a.max_rows; r += gridDim.x * 256) plan_row(a, s_end, s_stat, (int)r);
    }
}

static int page_shift(int page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

static int page_plan(const int32_t* len_old, const int32_t* len_new, int B, int page_size, int32_t* block_table, int max_blocks,
                     const int32_t* n_blocks_in, int32_t* n_blocks_out, int32_t* free_list, int n_pages,
                     const int32_t* free_count_in, int32_t* free_count_out, int32_t* status, int32_t* cu_rows,
                     int32_t* slots, int32_t* positions, int max_rows, const int32_t* parents, int64_t* tree_mask, int32_t* ticket, void* stream) {
    VALLE_REQUIRE(len_old && len_new && block_table && n_blocks_in && n_blocks_out && free_list && free_count_in && free_count_out && status && cu_rows &&
                  slots && positions && ticket, VALLE_E_ARG, "valle_page_plan: null pointer");
    VALLE_REQUIRE(B > 0 && B <= PLAN_MAX_B, VALLE_E_ARG, "valle_page_plan: %d requests (1 .. %d)", B, PLAN_MAX_B);
    const int shift = page_shift(page_size);
    VALLE_REQUIRE(shift > 0, VALLE_E_ARG, "valle_page_plan: page_size %d (16, 32, 64, 128 or 256)", page_size);
    VALLE_REQUIRE(max_blocks > 0 && (int64_t)B * max_blocks <= INT32_MAX && ((int64_t)max_blocks << shift) <= INT32_MAX, VALLE_E_ARG,
                  "valle_page_plan: max_blocks %d", max_blocks);
    VALLE_REQUIRE(n_pages > 0 && ((int64_t)n_pages << shift) <= INT32_MAX, VALLE_E_ARG, "valle_page_plan: n_pages %d", n_pages);
    VALLE_REQUIRE(max_rows > 0, VALLE_E_ARG, "valle_page_plan: max_rows %d", max_rows);
    PlanArgs a{len_old, len_new, block_table, n_blocks_in, n_blocks_out, free_list, free_count_in, free_count_out, status, cu_rows, slots, positions,
               parents, tree_mask, ticket, B, max_blocks, n_pages, shift, max_rows};
    hipStream_t s = (hipStream_t)stream;
    // Beyond 512 requests: the rows in the planning workgroup, or in a launch of their own over the chip, trees always (512 x 8: 36.7 / 9.0 us)
    if (B <= 512) {
        const int groups = min(max(ceil_div(max_rows, parents ? 16384 : 1024), parents || B > 64 ? ceil_div(B, 16) : 1), 256);
        if (B <= 64) page_plan_wave_kernel<1><<<groups, 1024, 0, s>>>(a);
        else page_plan_wave_kernel<8><<<groups, 1024, 0, s>>>(a);
    } else if (max_rows <= 4096 && !parents) page_plan_kernel<1024, true><<<1, 1024, 0, s>>>(a);
    else {
        page_plan_kernel<1024, false><<<1, 1024, 0, s>>>(a);
        page_rows_kernel<<<min(max(ceil_div(max_rows, 256), parents ? ceil_div(B, 4) : 0), 1024), 256, 0, s>>>(a);
    }
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}

extern "C" int valle_page_plan(const int32_t* len_old, const int32_t* len_new, int B, int page_size, int32_t* block_table, int max_blocks,
                               const int32_t* n_blocks_in, int32_t* n_blocks_out, int32_t* free_list, int n_pages,
                               const int32_t* free_count_in, int32_t* free_count_out, int32_t* status, int32_t* cu_rows,
                               int32_t* slots, int32_t* positions, int max_rows, const int32_t* parents, int64_t* tree_mask, int32_t* ticket, void* stream) {
    VALLE_REQUIRE((parents == nullptr) == (tree_mask == nullptr), VALLE_E_ARG, "valle_page_plan: parents and tree_mask go together");
    return page_plan(len_old, len_new, B, page_size, block_table, max_blocks, n_blocks_in, n_blocks_out, free_list, n_pages, free_count_in, free_count_out, status,
                     cu_rows, slots, positions, max_rows, parents, tree_mask, ticket, stream);
}

extern "C" int valle_page_plan_masked(const int32_t* len_old, const int32_t* len_new, int B, int page_size, int32_t* block_table, int max_blocks,
                                      const int32_t* n_blocks_in, int32_t* n_blocks_out, int32_t* free_list, int n_pages,
                                      const int32_t* free_count_in, int32_t* free_count_out, int32_t* status, int32_t* cu_rows,
                                      int32_t* slots, int32_t* positions, int max_rows, const int32_t* parents, int64_t* tree_mask, int32_t* ticket, void* stream) {
    VALLE_REQUIRE(tree_mask, VALLE_E_ARG, "valle_page_plan_masked: null pointer");
    return page_plan(len_old, len_new, B, page_size, block_table, max_blocks, n_blocks_in, n_blocks_out, free_list, n_pages, free_count_in, free_count_out, status,
                     cu_rows, slots, positions, max_rows, parents, tree_mask, ticket, stream);
}

// ------------------------------------------------------------------------------------ RoPE + write into pages
// Elements (2i, 2i + 1) of a q or k head rotate by rope[position][i] = (cos, sin), products and sums in fp32, one rounding at
// the end (valle_rope_kv rounds cos and sin to bf16 first, as the reference's cast tables are; here the table stays fp32: the
// result is the formula's within one rounding).  Memory-bound: 2 x 64 x es bytes per head and row.  16 rows of 16 heads 2.4 us (a launch and
// two round trips: position -> table row; slot), 12,176 rows bf16 (150 MB) 23.9 us = 6.3 TB/s, 29.1 us with caches of other data = 5.2.
struct RopePagedArgs {
    const void *q, *k, *v; void* qo;
    const int32_t* pos; const float* rope; const int32_t* slots;
    void *kc, *vc;
    long q_rs, k_rs, v_rs, qo_rs;       // row strides, elements
    long n_slots;
    int rope_rows, H, Hkv, shift;
};

template <typename T>
__device__ __forceinline__ void rope_turn(const uint4& in, const float4* cs, uint4& out) {
    constexpr int V = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(V)));
    const vec_t x = __builtin_bit_cast(vec_t, in);
    vec_t y;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {                          // two pairs per float4 of the table
        const float4 t = cs[i];
        const float a0 = to_f32<T>(x[4 * i]), b0 = to_f32<T>(x[4 * i + 1]), a1 = to_f32<T>(x[4 * i + 2]), b1 = to_f32<T>(x[4 * i + 3]);
        y[4 * i] = from_f32<T>(a0 * t.x - b0 * t.y); y[4 * i + 1] = from_f32<T>(b0 * t.x + a0 * t.y);
        y[4 * i + 2] = from_f32<T>(a1 * t.z - b1 * t.w); y[4 * i + 3] = from_f32<T>(b1 * t.z + a1 * t.w);
    }
    out = __builtin_bit_cast(uint4, y);
}

// One row per workgroup of 128 threads: a thread owns one 16-byte piece of the head and walks the heads, so it reads its
// piece of the table once.
template <typename T>
__global__ __launch_bounds__(128) void rope_kv_paged_kernel(RopePagedArgs a) {
    constexpr int V = 16 / sizeof(T), CH = 64 / V, HS = 128 / CH;       // elements and pieces per head, heads at a time
    const long r = blockIdx.x;
    const int c = threadIdx.x % CH, h0 = threadIdx.x / CH;
    const int slot = a.slots[r];
    const int p = min(max(a.pos[r], 0), a.rope_rows - 1);
    float4 cs[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) cs[i] = *reinterpret_cast<const float4*>(a.rope + (long)p * 64 + c * V + 4 * i);
    if (a.q) {
        const T* q = (const T*)a.q + r * a.q_rs + c * V;
        T* o = (T*)a.qo + r * a.qo_rs + c * V;
        for (int h = h0; h < a.H; h += HS) {
            const uint4 x = *reinterpret_cast<const uint4*>(q + h * 64);
            uint4 y;
            rope_turn<T>(x, cs, y);
            *reinterpret_cast<uint4*>(o + h * 64) = y;
        }
    }
    if (slot < 0 || slot >= a.n_slots) return;                          // padding, a refused request: nothing is cached
    const long page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
    const T* k = (const T*)a.k + r * a.k_rs + c * V;
    const T* v = (const T*)a.v + r * a.v_rs + c * V;
    for (int h = h0; h < a.Hkv; h += HS) {
        const uint4 x = *reinterpret_cast<const uint4*>(k + h * 64);
        const uint4 w = *reinterpret_cast<const uint4*>(v + h * 64);
        uint4 y;
        rope_turn<T>(x, cs, y);
        const long at = (((page * a.Hkv + h) << a.shift) + off) * 64 + c * V;
        *reinterpret_cast<uint4*>((T*)a.kc + at) = y;
        *reinterpret_cast<uint4*>((T*)a.vc + at) = w;
    }
}

extern "C" int valle_rope_kv_paged(const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, const void* v, int64_t v_row_stride,
                                   void* q_out, int64_t q_out_row_stride, const int32_t* positions, const float* rope, int rope_rows,
                                   const int32_t* slots, int M, int H, int Hkv, int Dh, void* kcache, void* vcache, int n_pages, int page_size,
                                   int dtype, void* stream) {
    VALLE_REQUIRE(k && v && positions && rope && slots && kcache && vcache, VALLE_E_ARG, "valle_rope_kv_paged: null pointer");
    VALLE_REQUIRE((q == nullptr) == (q_out == nullptr), VALLE_E_ARG, "valle_rope_kv_paged: q and q_out go together");
    VALLE_REQUIRE(dtype == VALLE_BF16 || dtype == VALLE_F32, VALLE_E_ARG, "valle_rope_kv_paged: unknown dtype %d", dtype);
    VALLE_REQUIRE(Dh == 64, VALLE_E_UNSUPPORTED, "valle_rope_kv_paged: head_dim %d (64 is built)", Dh);
    VALLE_REQUIRE(M >= 0 && H > 0 && Hkv > 0 && rope_rows > 0, VALLE_E_ARG, "valle_rope_kv_paged: M=%d H=%d Hkv=%d rope_rows=%d", M, H, Hkv, rope_rows);
    const int shift = page_shift(page_size);
    VALLE_REQUIRE(shift > 0, VALLE_E_ARG, "valle_rope_kv_paged: page_size %d (16, 32, 64, 128 or 256)", page_size);
    VALLE_REQUIRE(n_pages > 0 && ((int64_t)n_pages << shift) <= INT32_MAX, VALLE_E_ARG, "valle_rope_kv_paged: n_pages %d", n_pages);
    const int vec = 16 / (int)dtype_size(dtype);
    const void* ptrs[] = {q, k, v, q_out, rope, kcache, vcache};
    for (const void* p : ptrs) VALLE_REQUIRE(((uintptr_t)p & 15) == 0, VALLE_E_ARG, "valle_rope_kv_paged: tensors must be 16-byte aligned");
    const int64_t strides[] = {q ? q_row_stride : 0, k_row_stride, v_row_stride, q ? q_out_row_stride : 0};
    for (int64_t st : strides) VALLE_REQUIRE(st % vec == 0 && st >= 0, VALLE_E_ARG, "valle_rope_kv_paged: row strides must keep rows 16-byte aligned");
    VALLE_REQUIRE(!q || M <= 1 || q_out_row_stride >= (int64_t)H * 64, VALLE_E_ARG, "valle_rope_kv_paged: rows of q_out overlap");
    if (M == 0) return VALLE_OK;
    RopePagedArgs a{q, k, v, q_out, positions, rope, slots, kcache, vcache, q_row_stride, k_row_stride, v_row_stride, q_out_row_stride,
                    (long)n_pages << shift, rope_rows, H, Hkv, shift};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == VALLE_BF16) rope_kv_paged_kernel<bf16><<<M, 128, 0, s>>>(a);
    else rope_kv_paged_kernel<float><<<M, 128, 0, s>>>(a);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}

// ------------------------------------------------------------------------------------ commit of an accepted path
// cache[layer][ctx + j] = cache[layer][ctx + path[j]], j < n_accept.  Source and destination ranges overlap: a workgroup reads
// every row it moves of one (request, head, layer) into registers, meets at a barrier, and writes.  With the plan's status and page counts a
// request that was not served moves nothing, and no table entry at or behind its page count is followed: such entries are left over
// and name pages of others.  Three dependent round trips (path, table, row) bound it while the rows are few: one request, 12 layers, 3 rows 2.8 us
// (2.9 with status and counts); 16 requests, up to 5 rows 4.0 (4.2); 48 requests, 26 rows (123 MB) 22.0 (22.3) = 5.6 TB/s.
struct CommitArgs {
    void *kc, *vc;
    const int32_t *table, *ctx, *n_blocks, *status, *path, *n_accept;      // n_blocks, status: may be NULL (all entries hold, all were served)
    int32_t* len_out;
    long layer_stride;                  // elements
    int width, max_path, n_pages, shift, Hkv;
};

template <typename T>
__global__ __launch_bounds__(256) void kv_commit_kernel(CommitArgs a) {
    constexpr int V = 16 / sizeof(T), CH = 64 / V, TPI = 256 / (2 * CH), IT = 64 / TPI;   // pieces per row, rows at a time, rounds
    const int h = blockIdx.x, b = blockIdx.y;
    const long layer = blockIdx.z;
    const int ctx = a.ctx[b];
    const bool served = !a.status || a.status[b] == 0;
    const long cap = (long)(a.n_blocks ? min(max(a.n_blocks[b], 0), a.width) : a.width) << a.shift;
    const int n = served ? min(max(a.n_accept[b], 0), a.max_path) : 0;
    if (h == 0 && layer == 0 && threadIdx.x == 0) {
        const long len = min((long)ctx + n, a.n_blocks && served ? cap : (long)INT32_MAX);
        a.len_out[b] = ctx < 0 ? ctx : (int)len;
    }
    if (ctx < 0 || n == 0) return;
    const int c = threadIdx.x % CH, isv = (threadIdx.x / CH) & 1, t0 = threadIdx.x / (2 * CH);
    T* cache = (T*)(isv ? a.vc : a.kc) + layer * a.layer_stride;
    const int32_t* tab = a.table + (long)b * a.width;
    auto place = [&](long p) -> long {                                  // element offset of cached row p, -1: not in the cache
        if (p >= cap) return -1;
        const int page = tab[p >> a.shift];
        if (page < 0 || page >= a.n_pages) return -1;
        return ((((long)page * a.Hkv + h) << a.shift) + (p & ((1 << a.shift) - 1))) * 64 + c * V;
    };
    uint4 x[IT];
    long dst[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int j = i * TPI + t0;
        x[i] = uint4{0, 0, 0, 0}; dst[i] = -1;
        if (j < n) {
            const int from = a.path[(long)b * a.max_path + j];
            if (from >= 0 && from < 64 && from != j) {
                const long src = place((long)ctx + from);
                if (src >= 0) {
                    x[i] = *reinterpret_cast<const uint4*>(cache + src);
                    dst[i] = place((long)ctx + j);
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                    // the rows are in registers before any of them is written over
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IT; ++i)
        if (dst[i] >= 0) *reinterpret_cast<uint4*>(cache + dst[i]) = x[i];
}

extern "C" int valle_paged_kv_commit_served(void* kcache, void* vcache, int n_layers, int64_t layer_stride, const int32_t* block_table, int max_blocks,
                                            int n_pages, int page_size, const int32_t* ctx_len, const int32_t* n_blocks, const int32_t* status,
                                            const int32_t* path, int max_path, const int32_t* n_accept, int32_t* len_out, int B, int Hkv, int Dh,
                                            int dtype, void* stream) {
    VALLE_REQUIRE(kcache && vcache && block_table && ctx_len && path && n_accept && len_out, VALLE_E_ARG, "valle_paged_kv_commit: null pointer");
    VALLE_REQUIRE(len_out != ctx_len && len_out != n_blocks && len_out != status, VALLE_E_ARG,
                  "valle_paged_kv_commit: len_out must not be ctx_len, n_blocks or status (every workgroup reads them)");
    VALLE_REQUIRE(dtype == VALLE_BF16 || dtype == VALLE_F32, VALLE_E_ARG, "valle_paged_kv_commit: unknown dtype %d", dtype);
    VALLE_REQUIRE(Dh == 64, VALLE_E_UNSUPPORTED, "valle_paged_kv_commit: head_dim %d (64 is built)", Dh);
    VALLE_REQUIRE(B >= 0 && B <= 65535 && n_layers > 0 && n_layers <= 65535 && Hkv > 0 && max_blocks > 0, VALLE_E_ARG,
                  "valle_paged_kv_commit: B=%d n_layers=%d Hkv=%d max_blocks=%d", B, n_layers, Hkv, max_blocks);
    VALLE_REQUIRE(max_path > 0 && max_path <= 64, VALLE_E_ARG, "valle_paged_kv_commit: max_path %d (1 .. 64)", max_path);
    const int shift = page_shift(page_size);
    VALLE_REQUIRE(shift > 0, VALLE_E_ARG, "valle_paged_kv_commit: page_size %d (16, 32, 64, 128 or 256)", page_size);
    VALLE_REQUIRE(n_pages > 0 && ((int64_t)n_pages << shift) <= INT32_MAX, VALLE_E_ARG, "valle_paged_kv_commit: n_pages %d", n_pages);
    VALLE_REQUIRE(n_layers == 1 || layer_stride >= ((int64_t)n_pages << shift) * Hkv * 64, VALLE_E_ARG, "valle_paged_kv_commit: layers overlap");
    VALLE_REQUIRE((((uintptr_t)kcache | (uintptr_t)vcache) & 15) == 0 && layer_stride % 8 == 0, VALLE_E_ARG, "valle_paged_kv_commit: caches must be 16-byte aligned");
    if (B == 0) return VALLE_OK;
    CommitArgs a{kcache, vcache, block_table, ctx_len, n_blocks, status, path, n_accept, len_out, layer_stride, max_blocks, max_path, n_pages, shift, Hkv};
    dim3 grid(Hkv, B, n_layers);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == VALLE_BF16) kv_commit_kernel<bf16><<<grid, 256, 0, s>>>(a);
    else kv_commit_kernel<float><<<grid, 256, 0, s>>>(a);
    VALLE_LAUNCH_CHECK();
    return VALLE_OK;
}

extern "C" int valle_paged_kv_commit(void* kcache, void* vcache, int n_layers, int64_t layer_stride, const int32_t* block_table, int max_blocks,
                                     int n_pages, int page_size, const int32_t* ctx_len, const int32_t* path, int max_path,
                                     const int32_t* n_accept, int32_t* len_out, int B, int Hkv, int Dh, int dtype, void* stream) {
    return valle_paged_kv_commit_served(kcache, vcache, n_layers, layer_stride, block_table, max_blocks, n_pages, page_size, ctx_len, nullptr, nullptr, path,
                                        max_path, n_accept, len_out, B, Hkv, Dh, dtype, stream);
}
