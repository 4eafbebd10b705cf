// Attention of one new token per sequence where groups of sequences share their first pages, specialised at compile time for one head size
// (IK_HD, a multiple of 16).  bfloat16 pages of 64 keys, as attention_bf16.cu has them.
//
// o[i,h] = sum_j p_j v[j] with p = softmax_j(q[i,h] . k[j] scale) over the keys j of sequence i, head h reading kv head h / G, G = nh / nkv.  Sequences
// starts[g] <= i < starts[g+1] form group g, whose first shared[i] pages are the same.  A tile is some of a group's members with their G heads of a kv head: ROWS rows
// at most (heads in parts where G is more than that).  It sees a list of pages: the shared ones, which count for all of its rows, then every member's own,
// which count for that member's rows.  So a shared page is read once for all members of a tile, as the keys and values of one product.
//
// The pages of all tiles, one list behind the other, are cut into equal runs, a block each (per kv head): every block streams as many pages as every other,
// however unequal the groups are.  Where a run passes from one tile to the next, the block leaves the first one's partial result (unnormalised output,
// maximum, sum) and goes on; a second kernel joins each row's partials in the order of their runs.  Run j's partial of tile t is kept at t + j: each new
// partial is one tile or one run further, so the numbers are distinct and dense.
//
// A block: one warp brings pages into a ring of shared memory (by TMA with the 128-byte swizzle for head sizes that are multiples of 64, else by cp.async into
// padded rows: a warp takes 1,700 cycles to issue a page of head size 128 that way, one thread a hundred by TMA), four compute on mma.sync m16n8k16 tiles.
// A warp owns 16 rows and 64 / KQ of a page's keys (RT = 1, 2 or 4 tiles of 16 rows, KQ = 4 / RT), with running maximum and sum as floats, base 2; the
// warps of equal rows are merged at the end of a tile.  us with the join, one group of 4 / 8 of 4 / 12 of 1 to 8 / 2 of 16: 11.4 / 38.2 / 30.7 / 111.  (A warp to a page,
// KQ pages at a time, measured 13.5 / 39.2 / 29.1 / 109.6 at a step that took 12.4 / 38.2 / 30.4 / 110.7 this way: the small call loses what the third gains, and it needs more
// registers than two blocks leave.  Shorter runs, 1.5 to 3 to a block's place, took 42 to 49 for the second, whether handed out in order or taken by the blocks that finish
// first: a run costs 2.5 us besides its pages.)
//
// Rounded to fewer bits than the inputs ask for, as in the other attention kernels: probabilities, to bfloat16 for the second product (their sum takes them as floats; 1.2 to 1.5e-3
// of the result, which itself is rounded to bfloat16, 1.7e-3: together 1.8 to 2.0e-3 from 64 bits), and the cap's tanh.approx, off by up to 2^-11 of the cap.
//
// Keys behind a sequence's length are masked by position and their values are brought as zeros, so what lies in the unused part of a page never
// matters.  A page index outside the pool sets *status and is not followed.  A sequence without keys gets zeros.
#include <math.h>
#include <atomic>
#define IK_FAMILY 4
#include "common.cuh"
#include "tc_common.cuh"

#ifndef IK_HD
#error "compile with -DIK_HD=<head size>"
#endif

namespace {

typedef __nv_bfloat16 bf16;

constexpr int HD = IK_HD;
constexpr int PAGE = 64;
constexpr bool TMA = HD % 64 == 0;
constexpr int LD = TMA ? HD : HD + 8;      // row of a page in shared memory: swizzled blocks of 64 columns, or padded so that consecutive rows fall into different banks
constexpr int HALF = PAGE * LD, STAGE = 2 * HALF;        // keys (or values) of a page, both, in elements
constexpr int BLOCKS = HD <= 64 ? 3 : HD <= 128 ? 2 : 1;   // blocks of an SM
constexpr int FIT = 196608 / BLOCKS / (STAGE * 2), NS = FIT > 8 ? 8 : FIT < 3 ? 3 : FIT;         // pages of the ring: 192 KB an SM
constexpr int THREADS = 160;               // four computing warps, one that loads
constexpr size_t RING = (size_t)NS * STAGE * sizeof(bf16), FIXED = RING + 64 * 8 + 2 * NS * 8 + 8;         // bytes of the ring; with results' maxima and sums, barriers, a flag
constexpr int JOIN_FAMILY = IK_FAMILY_ELEMENTWISE;
constexpr int TILES = 1024, SEQS = 1024;   // most tiles and sequences of a launch
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 up to 256");

__device__ __forceinline__ void cp16(uint32_t smem, const void* gmem, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" :: "r"(smem), "l"(gmem), "r"(n));
}
// Arrives on the barrier when this thread's copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t s) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t s) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes from a tile's start to the 8 columns number `chunk` of `row`; row7 = row % 8 (rows of 128 bytes, 64 to a block, their 16-byte pieces exchanged by row % 8).
__device__ __forceinline__ uint32_t piece(int row, int row7, int chunk) {
    return TMA ? (uint32_t)((chunk >> 3) * PAGE * 128 + row * 128 + (((chunk & 7) ^ row7) << 4)) : (uint32_t)(row * LD + chunk * 8) * 2;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// A score in base 2: s * a, or with a cap b * tanh(s * a); see attention_bf16.cu.
__device__ __forceinline__ float capped(float s, float a, float b) {
    if (b == 0.f) return s * a;
    float y;
    asm("tanh.approx.f32 %0, %1;" : "=f"(y) : "f"(s * a));
    return b * y;
}

// What both kernels get.  Tile number: (group, part of its members, part of the heads), tiles_per_group to each group whether it has so many members or not.
struct Call {
    const int *kv_lens, *table, *starts, *shared;
    int table_stride, table_cols, n_groups, B, nh, nkv, G;
    int max_members, members, heads, head_parts, tiles_per_group, n_tiles;       // most members of a group; members and heads of a tile; parts of the heads; tiles
    int runs;
};
struct TileOf { int first, last, part, S; };                          // members first <= i < last, part of the heads, pages they share
__device__ __forceinline__ TileOf tile_of(const Call& c, const int* starts, const int* shared, int t) {
    const int g = t / c.tiles_per_group, k = t % c.tiles_per_group;
    const int a = min(max(starts[g], 0), c.B), b = min(max(starts[g + 1], a), min(c.B, a + c.max_members));       // (a part of its last tile may lie beyond the bound)
    TileOf o;
    o.part = k % c.head_parts;
    o.first = min(a + k / c.head_parts * c.members, b);
    o.last = min(o.first + c.members, b);
    o.S = a < b ? min(max(shared[a], 0), c.table_cols) : 0;
    return o;
}
// The order in which a tile's members' own pages come: members whose rows are different warps' take turns, so that several warps have work at a time (where
// members' rows do not fill 16s evenly: one after the other).  Number i's member, or -1.
__device__ __forceinline__ int member_at(const Call& c, const TileOf& o, int rt, int i) {
    const int per_warp = 16 / c.heads, m = 16 % c.heads == 0 ? (i % rt) * per_warp + i / rt : i;
    return o.first + m < o.last ? o.first + m : -1;
}
// pages: how many every sequence has, shared ones included.
__device__ __forceinline__ int own_pages(const int* pages, const TileOf& o, int seq) { return seq < 0 ? 0 : max(0, pages[seq] - o.S); }
__device__ __forceinline__ int pages_in(const int* pages, const TileOf& o) {
    if (o.first >= o.last) return 0;
    int n = o.S;
    for (int i = o.first; i < o.last; i++) n += own_pages(pages, o, i);
    return n;
}
// The runs in use: so many of `len` + 1 pages, then of `len`.  The first page of a run, the run of a page.
struct Cut { int runs, len, longer; };
__device__ __forceinline__ Cut cut_of(int pages, int most) {
    Cut c;
    c.runs = min(most, pages);                                       // (two pages at least to a run: small calls 9.9 us instead of 8.7)
    c.len = pages / max(c.runs, 1);
    c.longer = pages - c.len * c.runs;
    return c;
}
__device__ __forceinline__ int run_start(const Cut& c, int j) { return j * c.len + min(j, c.longer); }
__device__ __forceinline__ int run_of(const Cut& c, int page) {
    const int split = c.longer * (c.len + 1);
    return page < split ? page / (c.len + 1) : c.longer + (page - split) / c.len;
}

// The plan that the first block leaves for the join: per sequence its first tile and row, per tile its first and last run (no run: 1, 0).
struct Plan { int2* seqs; int2* tiles; };

template <int RT>
__global__ void __launch_bounds__(THREADS, BLOCKS)
attn_shared_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k_pages, const bf16* __restrict__ v_pages, float* __restrict__ part_o,
                   float2* __restrict__ part_ml, const Call c, const Plan plan, float scale_log2e, float cap_log2e, int n_pages, int* status,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    constexpr int ROWS = 16 * RT, KQ = 4 / RT, KEYS = PAGE / KQ, NB = KEYS / 8, CH = HD / 8;
    ik_pdl_wait();
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    bf16* const ring = (bf16*)smem_raw;                              // [NS][keys, values][PAGE][LD]
    float2* const sm_ml = (float2*)(smem_raw + RING);                // [4][16]: maxima and sums
    uint64_t* const full = (uint64_t*)(sm_ml + 64);                  // [NS]
    uint64_t* const empty = full + NS;                               // [NS]
    int& abort_flag = *(int*)(empty + NS);
    int* const ends = &abort_flag + 2;                               // [n_tiles]: pages up to and with a tile
    int* const pages = ends + c.n_tiles;                             // [B]
    int* const shared = pages + c.B;                                 // [B]
    int* const starts = shared + c.B;                                // [n_groups + 1]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = blockIdx.x, kvh = blockIdx.y;

    if (tid == 0) {
        abort_flag = 0;
        #pragma unroll
        for (int s = 0; s < NS; s++) { mbar_init(&full[s], TMA ? 1 : 32); mbar_init(&empty[s], 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (TMA && tid == 0) {
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map_v) : "memory");
    }
    // the block tables, on their way to L2 while the plan is made (all blocks together)
    for (long long i = (long long)(blockIdx.y * gridDim.x + blockIdx.x) * THREADS + tid; i * 32 < (long long)c.B * c.table_stride; i += (long long)gridDim.x * gridDim.y * THREADS)
        asm volatile("prefetch.global.L2 [%0];" :: "l"(c.table + min(i * 32, (long long)(c.B - 1) * c.table_stride + c.table_cols - 1)));
    for (int i = tid; i < c.B; i += THREADS) {
        shared[i] = c.shared[i];
        pages[i] = min((max(c.kv_lens[i], 0) + PAGE - 1) / PAGE, c.table_cols);
    }
    for (int i = tid; i <= c.n_groups; i += THREADS) starts[i] = c.starts[i];
    if (TMA && tid == 0 && (smem_u32(smem_raw) & 1023)) { abort_flag = 1; ik_set_status(status, IK_STATUS_SMEM_ALIGN); }
    __syncthreads();
    for (int t = tid; t < c.n_tiles; t += THREADS) ends[t] = pages_in(pages, tile_of(c, starts, shared, t));
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        for (int t0 = 0; t0 < c.n_tiles; t0 += 32) {
            int x = t0 + lane < c.n_tiles ? ends[t0 + lane] : 0;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
            if (t0 + lane < c.n_tiles) ends[t0 + lane] = before + x;
            before += __shfl_sync(0xffffffffu, x, 31);
        }
    }
    __syncthreads();
    const Cut cut = cut_of(ends[c.n_tiles - 1], c.runs);
    if (run == 0 && kvh == 0) {
        for (int i = tid; i < c.n_groups; i += THREADS)
            if (starts[i] < 0 || starts[i + 1] < starts[i] || starts[i + 1] > c.B || starts[i + 1] - starts[i] > c.max_members) ik_set_status(status, IK_STATUS_BAD_GROUP);
        for (int i = tid; i < c.B; i += THREADS) plan.seqs[i] = make_int2(-1, 0);
        __syncthreads();
        for (int t = tid; t < c.n_tiles; t += THREADS) {
            const int lo = t ? ends[t - 1] : 0, hi = ends[t];
            plan.tiles[t] = lo < hi ? make_int2(run_of(cut, lo), run_of(cut, hi - 1)) : make_int2(1, 0);
            const TileOf o = tile_of(c, starts, shared, t);
            if (o.part == 0)
                for (int i = o.first; i < o.last; i++) plan.seqs[i] = make_int2(t, (i - o.first) * c.heads);
        }
    }
    if (run >= cut.runs || abort_flag) return;
    const int u_first = run_start(cut, run), u_end = run_start(cut, run + 1);
    int t = 0;
    for (int past = c.n_tiles - 1; t < past;) {                       // the first tile that ends behind the run's first page
        const int mid = (t + past) >> 1;
        if (ends[mid] <= u_first) t = mid + 1;
        else past = mid;
    }

    if (warp == 4) {
        // ---- the loader: 32 pages' numbers at a time, one each lane
        int step = 0;
        bool alive = true;
        for (int u = u_first; u < u_end && alive;) {
            while (ends[t] <= u) t++;
            const int lo = t ? ends[t - 1] : 0, n = min(min(ends[t], u_end) - u, 32);
            const TileOf o = tile_of(c, starts, shared, t);
            int page = 0, filled = PAGE;
            if (lane < n) {
                int i = u + lane - lo, seq = o.first, col = i;
                if (i >= o.S) {
                    i -= o.S;
                    int n = 0;
                    seq = member_at(c, o, RT, 0);
                    for (int own = own_pages(pages, o, seq); i >= own; own = own_pages(pages, o, seq)) { i -= own; seq = member_at(c, o, RT, ++n); }
                    col = o.S + i;
                    filled = c.kv_lens[seq] - col * PAGE;
                }
                page = c.table[(size_t)seq * c.table_stride + col];
                if (page < 0 || page >= n_pages) { ik_set_status(status, IK_STATUS_READ_NO_PAGE); page = 0; }
            }
            for (int l = 0; l < n; l++, step++) {
                const int stage = step % NS, pg = __shfl_sync(0xffffffffu, page, l), rows = __shfl_sync(0xffffffffu, filled, l);
                alive = __all_sync(0xffffffffu, step < NS || mbar_wait(&empty[stage], (step / NS - 1) & 1, &abort_flag, status, IK_WAIT_LIMIT_NS, 41, step));
                if (!alive) break;
                bf16* const to = ring + stage * STAGE;
                if (TMA) {
                    if (elect_one()) {
                        mbar_expect_tx(&full[stage], STAGE * sizeof(bf16));
                        const int y = (pg * c.nkv + kvh) * PAGE;
                        #pragma unroll
                        for (int x = 0; x < HD; x += 64) tma_load_2d(to + x * PAGE, &map_k, x, y, &full[stage]);
                        #pragma unroll
                        for (int x = 0; x < HD; x += 64) tma_load_2d(to + HALF + x * PAGE, &map_v, x, y, &full[stage]);
                    }
                    __syncwarp();
                } else {
                    const bf16* const kg = k_pages + ((size_t)pg * c.nkv + kvh) * PAGE * HD;
                    const bf16* const vg = v_pages + ((size_t)pg * c.nkv + kvh) * PAGE * HD;
                    const uint32_t at = smem_u32(to);
                    #pragma unroll 8
                    for (int idx = lane; idx < PAGE * CH; idx += 32) cp16(at + piece(idx / CH, 0, idx % CH), kg + idx * 8, true);
                    #pragma unroll 8
                    for (int idx = lane; idx < PAGE * CH; idx += 32) cp16(at + HALF * 2 + piece(idx / CH, 0, idx % CH), vg + idx * 8, idx / CH < rows);
                    cp_arrive(&full[stage]);
                }
            }
            u += n;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (TMA && !alive)                                            // what was asked for lands before the block's memory goes (a limit here, too)
            for (int i = max(0, step - NS); i < step; i++) {
                const long long c0 = wait_clock();
                while (!mbar_test(&full[i % NS], (i / NS) & 1) && !wait_ran_out(c0, IK_WAIT_LIMIT_NS)) {}
            }
        return;
    }

    // ---- the computing warps
    const int g = lane >> 2, q2 = lane & 3, rt = warp % RT, kq = warp / RT;
    int step = 0;
    bool alive = true;                                               // behind a wait that ran out a warp does no more work, but meets the others where they wait for it
    for (int u = u_first; u < u_end;) {
        while (ends[t] <= u) t++;
        const int lo = t ? ends[t - 1] : 0, stop = min(ends[t], u_end);
        const TileOf o = tile_of(c, starts, shared, t);
        const int n_rows = (o.last - o.first) * c.heads;             // rows of this tile (fewer where the last part of the heads is not full)
        int seq_of[2], pos[2];
        const bf16* qrow[2];
        #pragma unroll
        for (int r = 0; r < 2; r++) {
            const int rho = rt * 16 + g + 8 * r, head = o.part * c.heads + rho % c.heads;
            const bool is = rho < n_rows && head < c.G;
            seq_of[r] = is ? o.first + rho / c.heads : -1;
            pos[r] = is ? c.kv_lens[seq_of[r]] - 1 : -1;
            qrow[r] = is ? q + ((size_t)seq_of[r] * c.nh + kvh * c.G + head) * HD + 2 * q2 : nullptr;
        }
        uint32_t qf[HD / 16][4];
        #pragma unroll
        for (int ks = 0; ks < HD / 16; ks++)
            #pragma unroll
            for (int e = 0; e < 4; e++) qf[ks][e] = qrow[e & 1] ? *reinterpret_cast<const uint32_t*>(qrow[e & 1] + ks * 16 + (e >> 1) * 8) : 0u;
        // rows of a sequence that ends inside the shared pages, against what was asked for, are masked there, too
        const bool ends_early = __any_sync(0xffffffffu, (seq_of[0] >= 0 && pos[0] + 1 < o.S * PAGE) || (seq_of[1] >= 0 && pos[1] + 1 < o.S * PAGE));
        // which own page comes first
        int nth = 0, member = member_at(c, o, RT, 0), col = u - lo;
        if (col >= o.S) {
            int i = col - o.S;
            for (int own = own_pages(pages, o, member); i >= own; own = own_pages(pages, o, member)) { i -= own; member = member_at(c, o, RT, ++nth); }
            col = o.S + i;
        }
        float acc[HD / 8][4], m_i[2] = {-INFINITY, -INFINITY}, l_i[2] = {0.f, 0.f};
        #pragma unroll
        for (int d = 0; d < HD / 8; d++)
            #pragma unroll
            for (int e = 0; e < 4; e++) acc[d][e] = 0.f;

        for (; u < stop; u++, step++) {
            const bool own = u - lo >= o.S;
            if (own && (u - lo == o.S || col >= pages[member])) {            // the next member that has pages of its own
                if (u - lo != o.S) member = member_at(c, o, RT, ++nth);
                while (own_pages(pages, o, member) == 0) member = member_at(c, o, RT, ++nth);
                col = o.S;
            }
            const int at = own ? col++ : u - lo, stage = step % NS;          // the page's number in the sequence
            alive = alive && __all_sync(0xffffffffu, mbar_wait(&full[stage], (step / NS) & 1, &abort_flag, status, IK_WAIT_LIMIT_NS, 42, step));
            if (!alive) continue;
            if (own && RT > 1 && !__any_sync(0xffffffffu, seq_of[0] == member || seq_of[1] == member)) {       // another warp's rows
                if (lane == 0 && (KQ == 1 || u + 1 < stop)) mbar_arrive(&empty[stage]);
                continue;
            }
            const uint32_t ks_ = smem_u32(ring + stage * STAGE), vs_ = ks_ + HALF * 2;
            if (TMA && own) {                                         // values behind the last key: zeros (by cp.async they come so)
                const int from = max(c.kv_lens[member] - at * PAGE, kq * KEYS);         // (of this warp's keys)
                if (from < (kq + 1) * KEYS) {
                    for (int i = lane; i < ((kq + 1) * KEYS - from) * 8; i += 32)
                        #pragma unroll
                        for (int x = 0; x < HD; x += 64) *reinterpret_cast<uint4*>((unsigned char*)(ring + stage * STAGE + HALF + x * PAGE) + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                    fence_async();
                }
            }
            float s[NB][4];
            #pragma unroll
            for (int n = 0; n < NB; n++)
                #pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] = 0.f;
            #pragma unroll
            for (int ks = 0; ks < HD / 16; ks++)
                #pragma unroll
                for (int np = 0; np < NB / 2; np++) {
                    uint32_t bfr[4];
                    ldsm4(bfr, ks_ + piece(kq * KEYS + np * 16 + (lane & 7) + (lane >> 4) * 8, lane & 7, ks * 2 + ((lane >> 3) & 1)));
                    mma(s[2 * np], qf[ks], bfr[0], bfr[1]);
                    mma(s[2 * np + 1], qf[ks], bfr[2], bfr[3]);
                }
            float mx[2] = {-INFINITY, -INFINITY};
            if (own || ends_early) {
                const int jbase = at * PAGE + kq * KEYS + 2 * q2;
                #pragma unroll
                for (int n = 0; n < NB; n++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = e >> 1;
                        const bool ok = (!own || seq_of[r] == member) && jbase + n * 8 + (e & 1) <= pos[r];
                        s[n][e] = ok ? capped(s[n][e], scale_log2e, cap_log2e) : -INFINITY;
                        mx[r] = fmaxf(mx[r], s[n][e]);
                    }
            } else {
                #pragma unroll
                for (int n = 0; n < NB; n++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[n][e] = capped(s[n][e], scale_log2e, cap_log2e);
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
                    }
            }
            float alpha[2], rs[2] = {0.f, 0.f};
            #pragma unroll
            for (int r = 0; r < 2; r++) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float m_new = fmaxf(m_i[r], mx[r]), m_use = m_new == -INFINITY ? 0.f : m_new;
                alpha[r] = ik_ex2(m_i[r] - m_use);
                m_i[r] = m_new;
                mx[r] = m_use;
            }
            uint32_t pa[NB / 2][4];
            #pragma unroll
            for (int n = 0; n < NB; n++) {
                #pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[n][e] = ik_ex2(s[n][e] - mx[e >> 1]);
                    rs[e >> 1] += s[n][e];
                }
                pa[n / 2][(n & 1) * 2] = pack_bf16(s[n][0], s[n][1]);
                pa[n / 2][(n & 1) * 2 + 1] = pack_bf16(s[n][2], s[n][3]);
            }
            #pragma unroll
            for (int r = 0; r < 2; r++) l_i[r] = l_i[r] * alpha[r] + rs[r];
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
                #pragma unroll
                for (int d = 0; d < HD / 8; d++) { acc[d][0] *= alpha[0]; acc[d][1] *= alpha[0]; acc[d][2] *= alpha[1]; acc[d][3] *= alpha[1]; }
            }
            auto values = [&](uint32_t (&bfr)[4], int kk, int dp) {
                ldsm4t(bfr, vs_ + piece(kq * KEYS + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, lane & 7, dp * 2 + (lane >> 4)));
            };
            if (!own) {
                #pragma unroll
                for (int kk = 0; kk < NB / 2; kk++)
                    #pragma unroll
                    for (int dp = 0; dp < HD / 16; dp++) {
                        uint32_t bfr[4];
                        values(bfr, kk, dp);
                        mma(acc[2 * dp], pa[kk], bfr[0], bfr[1]);
                        mma(acc[2 * dp + 1], pa[kk], bfr[2], bfr[3]);
                    }
            } else {
                // other members' rows have weight 0 on a page that is not theirs, but 0 x inf is not 0: they do not take part
                #pragma unroll
                for (int dp = 0; dp < HD / 16; dp++) {
                    float part[2][4] = {};
                    #pragma unroll
                    for (int kk = 0; kk < NB / 2; kk++) {
                        uint32_t bfr[4];
                        values(bfr, kk, dp);
                        mma(part[0], pa[kk], bfr[0], bfr[1]);
                        mma(part[1], pa[kk], bfr[2], bfr[3]);
                    }
                    #pragma unroll
                    for (int i = 0; i < 2; i++)
                        #pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (seq_of[e >> 1] == member) acc[2 * dp + i][e] += part[i][e];
                }
            }
            __syncwarp();
            // the last page of a tile is given back behind the merge below, which uses its space
            if (lane == 0 && (KQ == 1 || u + 1 < stop)) mbar_arrive(&empty[stage]);
        }
        const size_t slot = (size_t)(t + run) * c.nkv + kvh;
        #pragma unroll
        for (int r = 0; r < 2; r++) {
            l_i[r] += __shfl_xor_sync(0xffffffffu, l_i[r], 1);
            l_i[r] += __shfl_xor_sync(0xffffffffu, l_i[r], 2);
        }
        if (KQ == 1) {
            #pragma unroll
            for (int r = 0; r < 2; r++) {
                const int rho = rt * 16 + g + 8 * r;
                if (rho < n_rows) {
                    float* const to = part_o + (slot * ROWS + rho) * HD + 2 * q2;
                    #pragma unroll
                    for (int d = 0; d < HD / 8; d++) *reinterpret_cast<float2*>(to + d * 8) = make_float2(acc[d][2 * r], acc[d][2 * r + 1]);
                    if (q2 == 0) part_ml[slot * ROWS + rho] = make_float2(m_i[r], l_i[r]);
                }
            }
        } else {
            // the warps' parts of the keys meet in the space of the tile's last page, which the loader does not have back yet
            static_assert(4 * 16 * HD * sizeof(float) <= STAGE * sizeof(bf16), "a page's space holds four warps' results");
            float* const sm_o = (float*)(ring + (step - 1) % NS * STAGE);        // [4][16][HD], fours of columns exchanged by row
            compute_sync();
            #pragma unroll
            for (int r = 0; r < 2; r++) {
                float* const to = sm_o + (warp * 16 + g + 8 * r) * HD;
                #pragma unroll
                for (int d = 0; d < HD / 8; d++) *reinterpret_cast<float2*>(to + ((d * 8 + 2 * q2) ^ ((g & 3) << 2))) = make_float2(acc[d][2 * r], acc[d][2 * r + 1]);
                if (q2 == 0) sm_ml[warp * 16 + g + 8 * r] = make_float2(m_i[r], l_i[r]);
            }
            compute_sync();
            for (int idx = tid; idx < n_rows * (HD / 4); idx += 128) {
                const int rho = idx / (HD / 4), x = idx % (HD / 4) * 4;
                float mm = -INFINITY;
                #pragma unroll
                for (int w = 0; w < KQ; w++) mm = fmaxf(mm, sm_ml[w * ROWS + rho].x);
                const float m_use = mm == -INFINITY ? 0.f : mm;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                float ll = 0.f;
                #pragma unroll
                for (int w = 0; w < KQ; w++) {
                    const float2 ml = sm_ml[w * ROWS + rho];
                    const float a = ik_ex2(ml.x - m_use);
                    const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * ROWS + rho) * HD + (x ^ ((rho & 3) << 2)));
                    sum.x += v.x * a; sum.y += v.y * a; sum.z += v.z * a; sum.w += v.w * a;
                    ll += ml.y * a;
                }
                *reinterpret_cast<float4*>(part_o + (slot * ROWS + rho) * HD + x) = sum;
                if (x == 0) part_ml[slot * ROWS + rho] = make_float2(mm, ll);
            }
            if (TMA) fence_async();
            compute_sync();
            if (lane == 0) mbar_arrive(&empty[(step - 1) % NS]);
        }
    }
    ik_pdl_launch_dependents();
}

// Joins a (sequence, head)'s partials, then the sink, by groups of HD / 4 threads.  SPLIT: a block each, of so many times JG groups, which share the runs out and are summed in
// their order; 0: a group each.  us with the kernel before, twice JG / JG / a group: 4 sequences of 32 heads 11.3 / 12.4 / 16.8, 18 15.1 / 15.3 / 17.5, 32 39.7 / 38.5 / 38.6, 64 35.3 /
// 33.7 / 32.7, 256 72 / 66 / 60, 1,024 120 / 94 / 65.
constexpr int JV = HD / 4, JG = HD <= 128 ? 128 / JV : 2, JT = JV * JG;
struct Sum { float4 o; float m, l; };
__device__ __forceinline__ void add(Sum& s, const float4& v, float m, float l) {
    const float m_new = fmaxf(s.m, m), m_use = m_new == -INFINITY ? 0.f : m_new, a = ik_ex2(s.m - m_use), w = ik_ex2(m - m_use);
    s.o = make_float4(s.o.x * a + v.x * w, s.o.y * a + v.y * w, s.o.z * a + v.z * w, s.o.w * a + v.w * w);
    s.l = s.l * a + l * w;
    s.m = m_new;
}
template <int SPLIT>
__global__ void __launch_bounds__(JT * (SPLIT ? SPLIT : 1))
attn_shared_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, bf16* __restrict__ out, const Plan plan, int rows, int heads, int nh,
                        int nkv, int sink, const float* __restrict__ sink_v) {
    constexpr int GROUPS = SPLIT ? JG * SPLIT : 1;                     // of a head
    __shared__ float4 sums[GROUPS][JV];
    __shared__ float2 ml_of[GROUPS];
    ik_pdl_wait();
    ik_pdl_launch_dependents();
    IK_AFTER_WAIT(part_o);
    IK_AFTER_WAIT(part_ml);
    const int grp = threadIdx.x / JV, x = threadIdx.x % JV, b = blockIdx.x, h = SPLIT ? blockIdx.y : blockIdx.y * JG + grp, G = nh / nkv;
    if (!SPLIT && h >= nh) return;
    const int2 where = plan.seqs[b];
    const int in = h % G, t = where.x + in / heads, row = where.y + in % heads, kvh = h / G;
    const int2 over = where.x >= 0 ? plan.tiles[t] : make_int2(1, 0);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    Sum s{zero, -INFINITY, 0.f};
    #pragma unroll 4
    for (int j = over.x + (SPLIT ? grp : 0); j <= over.y; j += GROUPS) {
        const size_t at = ((size_t)(t + j) * nkv + kvh) * rows + row;
        const float2 ml = part_ml[at];
        const float4 v = *reinterpret_cast<const float4*>(part_o + at * HD + x * 4);
        add(s, ml.y == 0.f ? zero : v, ml.x, ml.y);                    // a sequence without keys takes nothing from its neighbours' pages, be they infinite
    }
    if (SPLIT) {
        sums[grp][x] = s.o;
        if (x == 0) ml_of[grp] = make_float2(s.m, s.l);
        __syncthreads();
        if (grp != 0) return;
        #pragma unroll
        for (int i = 1; i < GROUPS; i++) add(s, sums[i][x], ml_of[i].x, ml_of[i].y);
    }
    if (sink) add(s, zero, sink_v ? sink_v[h] * 1.4426950408889634f : 0.f, 1.f);
    const float inv = s.l > 0.f ? 1.0f / s.l : 0.f;                    // (no keys: zeros; a sum that is not a number is passed on below)
    ik_st4(out, ((size_t)b * nh + h) * HD + x * 4, s.l == s.l ? make_float4(s.o.x * inv, s.o.y * inv, s.o.z * inv, s.o.w * inv) : make_float4(s.l, s.l, s.l, s.l));
}

template <int RT>
int launch(const void* q, const void* k_pages, const void* v_pages, void* out, float* scratch, const Call& c, const Plan& plan, float sc_a, float sc_b, int sink,
           const float* sink_v, int n_pages, int* status, cudaStream_t stream) {
    const size_t slots = (size_t)(c.n_tiles + c.runs) * c.nkv * 16 * RT;
    float2* const part_ml = (float2*)(scratch + slots * HD);
    const size_t smem = FIXED + (size_t)(c.n_tiles + 2 * c.B + c.n_groups + 1) * sizeof(int);
    auto kern = attn_shared_kernel<RT>;
    // one amount whatever the call needs: the attribute belongs to the kernel, and several host threads may launch it
    // (and once a device: asked for at every call it costs the host 1 us)
    const int most = (int)FIXED + (2 * TILES + 2 * SEQS + 1) * (int)sizeof(int);
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev >= 64 || !(set.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return (int)e;
        set.fetch_or(bit, std::memory_order_release);
    }
    CUtensorMap map_k = {}, map_v = {};
    if (TMA) {
        const unsigned long long rows = (unsigned long long)n_pages * c.nkv * PAGE;
        if (rows > 0x7fffffffull) return IK_UNSUPPORTED;
        int st = ik_make_map(&map_k, k_pages, rows, HD, HD, PAGE);
        if (st == IK_OK) st = ik_make_map(&map_v, v_pages, rows, HD, HD, PAGE);
        if (st != IK_OK) return st;
    }
    IK_RETURN_IF_ERROR(ik_launch(kern, dim3(c.runs, c.nkv), THREADS, smem, stream, (const bf16*)q, (const bf16*)k_pages, (const bf16*)v_pages, scratch, part_ml, c, plan,
                                 sc_a, sc_b, n_pages, status, map_k, map_v));
    // a group each where blocks of a head each would not fit at a time; of twice the threads where they take a quarter of the space
    const long long place = 2048ll / JT * ik_sm_count(), blocks = (long long)c.B * c.nh;
    const int split = blocks * 4 <= place ? 2 : blocks <= place ? 1 : 0;
    auto join = split == 2 ? attn_shared_join_kernel<2> : split == 1 ? attn_shared_join_kernel<1> : attn_shared_join_kernel<0>;
    IK_RETURN_IF_ERROR(ik_launch_family(JOIN_FAMILY, join, dim3(c.B, split ? c.nh : (c.nh + JG - 1) / JG), JT * (split ? split : 1), 0,
                                        stream, (const float*)scratch, (const float2*)part_ml, (bf16*)out, plan, 16 * RT, c.heads, c.nh, c.nkv, sink, sink_v));
    IK_LAUNCH_STATUS();
}

// How a call is cut into tiles and runs; RT, or a negative status.
int cut(Call& c, int n_groups, int max_members, int B, int nh, int nkv) {
    c.n_groups = n_groups; c.max_members = max_members; c.B = B; c.nh = nh; c.nkv = nkv; c.G = nh / nkv;
    const long long rows = (long long)max_members * c.G;
    const int rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4, most = 16 * rt;
    c.heads = c.G < most ? c.G : most;
    c.head_parts = (c.G + c.heads - 1) / c.heads;
    c.members = most / c.heads < max_members ? most / c.heads : max_members;
    const long long per = (long long)((max_members + c.members - 1) / c.members) * c.head_parts;
    if (per * n_groups > TILES || B > SEQS || nkv > 65535) return IK_UNSUPPORTED;
    c.tiles_per_group = (int)per;
    c.n_tiles = (int)per * n_groups;
    const int runs = BLOCKS * ik_sm_count() / nkv;
    c.runs = runs > 1 ? runs : 1;
    return rt;
}

}  // namespace

IK_EXPORT int ik_attn_shared_head_dim() { return HD; }
// Sites of the kernel's waits: 41 = loader for a page's space, 42 = computing warps for a page.
IK_EXPORT int ik_attn_shared_take_wait_record(int* out4) { return ik_take_wait_record(out4); }

// Bytes of scratch of a call, or a negative status where there are more tiles or sequences than a launch takes.
IK_EXPORT long long ik_attn_shared_scratch(int n_groups, int max_members, int B, int nh, int nkv) {
    if (n_groups <= 0 || max_members <= 0 || max_members > B || B <= 0 || nh <= 0 || nkv <= 0 || nh % nkv) return IK_BAD_ARGUMENT;
    Call c;
    const int rt = cut(c, n_groups, max_members, B, nh, nkv);
    if (rt < 0) return rt;
    return (long long)(c.n_tiles + c.runs) * nkv * 16 * rt * (HD + 2) * 4 + ((long long)B + c.n_tiles) * 8;
}

// scratch: ik_attn_shared_scratch bytes on 16 bytes.  starts: [n_groups + 1], shared: [B], on the device; max_members: no group is larger (else *status is set, and what is beyond is left out).
IK_EXPORT int ik_attn_shared(const void* q, const void* k_pages, const void* v_pages, void* out, void* scratch, const int* kv_lens, const int* table, int table_stride,
                             int table_cols, const int* starts, const int* shared, int n_groups, int max_members, int B, int nh, int nkv, float scale, float softcap,
                             int sink, const float* sink_v, int page_size, int n_pages, int* status, cudaStream_t stream) {
    const float sc_a = softcap > 0.f ? scale / softcap : scale * 1.4426950408889634f, sc_b = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
    if (B <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || page_size != PAGE || n_groups <= 0 || max_members <= 0 || max_members > B || nh > 65535 || table_cols <= 0 ||
        table_stride < table_cols || n_pages <= 0 || ((uintptr_t)scratch & 15))
        return IK_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) return IK_UNSUPPORTED;
    Call c;
    c.kv_lens = kv_lens; c.table = table; c.starts = starts; c.shared = shared; c.table_stride = table_stride; c.table_cols = table_cols;
    const int rt = cut(c, n_groups, max_members, B, nh, nkv);
    if (rt < 0) return rt;
    const size_t parts = (size_t)(c.n_tiles + c.runs) * nkv * 16 * rt * (HD + 2);
    int2* const seqs = (int2*)((float*)scratch + parts);
    const Plan plan{seqs, seqs + B};
    if (rt == 1) return launch<1>(q, k_pages, v_pages, out, (float*)scratch, c, plan, sc_a, sc_b, sink, sink_v, n_pages, status, stream);
    if (rt == 2) return launch<2>(q, k_pages, v_pages, out, (float*)scratch, c, plan, sc_a, sc_b, sink, sink_v, n_pages, status, stream);
    return launch<4>(q, k_pages, v_pages, out, (float*)scratch, c, plan, sc_a, sc_b, sink, sink_v, n_pages, status, stream);
}
