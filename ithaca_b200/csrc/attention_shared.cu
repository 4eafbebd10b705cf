// Attention of one new token per sequence where groups of sequences share their first pages, specialised at compile time for one head size
// (IK_HD, a multiple of 16).  bfloat16 pages of 64 keys, as attention_bf16.cu has them.
//
// o[i,h] = sum_j p_j v[j] with p = softmax_j(q[i,h] . k[j] scale) over the keys of sequence i, head h reading kv head h / (nh / nkv).  Sequences starts[g] <= i <
// starts[g+1] form group g, whose first shared[i] pages are the same: what they contribute is formed once for the group, with the rows (sequence, query
// head of the kv head) of all members as the rows of one tile, so that a shared key or value is read once for all of them; the pages behind are
// each sequence's own.  A block owns a tile of rows, a kv head and one chunk of pages and leaves an unnormalised partial (maximum,
// sum, output) per row; a second kernel joins a row's partials in the order of its chunks.
//
// Keys behind a sequence's length are masked by position.  A page index outside the pool sets *status and is not followed.  A sequence
// without keys gets zeros.
#include <math.h>
#define IK_FAMILY 4
#include "common.cuh"

#ifndef IK_HD
#error "compile with -DIK_HD=<head size>"
#endif

namespace {

constexpr int HD = IK_HD;
constexpr int PAGE = 64;
constexpr int LD = HD + 8;                 // padded row: consecutive rows fall into different banks
constexpr int MT = HD <= 64 ? 4 : HD <= 128 ? 2 : 1;     // tiles of 16 rows a block: what the registers hold of their outputs
constexpr int ROWS = 16 * MT;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 up to 256");

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ void cp16(void* smem, const void* gmem, bool valid) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(smem);
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" :: "r"(s), "l"(gmem), "r"(n));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" :: "n"(N)); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
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

// How the work is cut: shared pages into at most n_shared chunks of shared_chunk pages, own pages into at most n_own of own_chunk; the last
// chunk of a kind takes all that is left, so that a bound that was too small costs time and nothing else.
struct Cut { int shared_chunk, n_shared, own_chunk, n_own; };
__device__ __forceinline__ int chunks_of(int pages, int chunk, int most) { return min(most, (pages + chunk - 1) / chunk); }

// Rows of a block: (sequence, head) pairs; row r is head `first_head + r % heads` of sequence `first_seq + r / heads`.
template <int NS>
__global__ void __launch_bounds__(128)
attn_shared_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k_pages, const bf16* __restrict__ v_pages, float* __restrict__ part_o,
                   float* __restrict__ part_ml, const int* __restrict__ kv_lens, const int* __restrict__ table, int table_stride, int table_cols,
                   const int* __restrict__ starts, const int* __restrict__ shared, int n_groups, int row_tiles, int B, int nh, int nkv, float scale_log2e,
                   float cap_log2e, int n_pages, Cut cut, int* status) {
    ik_pdl_wait();
    constexpr int CH = HD / 8;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    bf16* Qs = (bf16*)smem_raw;                      // [ROWS][LD]
    bf16* Ks = Qs + ROWS * LD;                       // [NS][PAGE][LD]
    bf16* Vs = Ks + NS * PAGE * LD;                  // [NS][PAGE][LD]
    __shared__ int row_pos[ROWS];                    // the query's position, -1: no such row

    const int kvh = blockIdx.y, G = nh / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int shared_blocks = n_groups * row_tiles * cut.n_shared;
    int first_seq, n_rows, first_row, p_first, p_end, split;      // rows first_row .. of the (sequence, head) pairs from first_seq on
    int filled = 0x7fffffff;                                       // positions of own pages that hold keys (shared pages are full)
    if ((int)blockIdx.x < shared_blocks) {
        int i = blockIdx.x;
        split = i % cut.n_shared; i /= cut.n_shared;
        const int rt = i % row_tiles, grp = i / row_tiles;
        first_seq = min(max(starts[grp], 0), B);
        const int members = min(max(starts[grp + 1], first_seq), B) - first_seq;
        first_row = rt * ROWS;
        n_rows = min(ROWS, members * G - first_row);
        if (n_rows <= 0) return;
        const int pages = min(max(shared[first_seq], 0), table_cols), n = chunks_of(pages, cut.shared_chunk, cut.n_shared);
        if (split >= n) return;
        p_first = split * cut.shared_chunk;
        p_end = split == n - 1 ? pages : p_first + cut.shared_chunk;
    } else {
        const int hc_n = (G + ROWS - 1) / ROWS;
        int i = blockIdx.x - shared_blocks;
        const int os = i % cut.n_own; i /= cut.n_own;
        first_seq = i / hc_n;
        first_row = (i % hc_n) * ROWS;
        n_rows = min(ROWS, G - first_row);
        filled = kv_lens[first_seq];
        const int pages = min((max(filled, 0) + PAGE - 1) / PAGE, table_cols), mine = min(max(shared[first_seq], 0), pages);
        const int n = chunks_of(pages - mine, cut.own_chunk, cut.n_own);
        if (os >= n) return;
        p_first = mine + os * cut.own_chunk;
        p_end = os == n - 1 ? pages : p_first + cut.own_chunk;
        split = cut.n_shared + os;
    }
    const int n_mt = (n_rows + 15) / 16;
    const int* const pages_of = table + (size_t)first_seq * table_stride;
    for (int r = threadIdx.x; r < ROWS; r += 128) row_pos[r] = r < n_rows ? kv_lens[first_seq + (first_row + r) / G] - 1 : -1;
    for (int idx = threadIdx.x; idx < n_mt * 16 * CH; idx += 128) {
        const int r = idx / CH, c = idx % CH, rho = first_row + r;
        const bool v = r < n_rows;
        cp16(Qs + r * LD + c * 8, v ? q + ((size_t)(first_seq + rho / G) * nh + kvh * G + rho % G) * HD + c * 8 : q, v);
    }
    auto load_page = [&](int stage, int p) {
        int page = pages_of[p];
        if (page < 0 || page >= n_pages) { if (threadIdx.x == 0) ik_set_status(status, IK_STATUS_READ_NO_PAGE); page = 0; }
        const bf16* kg = k_pages + ((size_t)page * nkv + kvh) * PAGE * HD;
        const bf16* vg = v_pages + ((size_t)page * nkv + kvh) * PAGE * HD;
        bf16* ks = Ks + stage * PAGE * LD;
        bf16* vs = Vs + stage * PAGE * LD;
        for (int idx = threadIdx.x; idx < PAGE * CH; idx += 128) {
            const int r = idx / CH, c = idx % CH;
            cp16(ks + r * LD + c * 8, kg + r * HD + c * 8, true);
            cp16(vs + r * LD + c * 8, vg + r * HD + c * 8, p * PAGE + r < filled);      // what lies behind the last key has weight 0 and may be anything: not even 0 x NaN
        }
    };
    #pragma unroll
    for (int s = 0; s < NS; s++) {
        if (p_first + s < p_end) load_page(s, p_first + s);
        cp_commit();
    }

    float o[MT][HD / 8][4], m_i[MT][2], l_i[MT][2];
    #pragma unroll
    for (int m = 0; m < MT; m++) {
        #pragma unroll
        for (int d = 0; d < HD / 8; d++)
            #pragma unroll
            for (int e = 0; e < 4; e++) o[m][d][e] = 0.f;
        m_i[m][0] = m_i[m][1] = -INFINITY;
        l_i[m][0] = l_i[m][1] = 0.f;
    }

    for (int p = p_first; p < p_end; p++) {
        const int stage = (p - p_first) % NS;
        cp_wait<NS - 1>();
        __syncthreads();
        const bf16* ks_ = Ks + (stage * PAGE + warp * 16) * LD;
        const bf16* vs_ = Vs + (stage * PAGE + warp * 16) * LD;
        float s[MT][2][4];
        #pragma unroll
        for (int m = 0; m < MT; m++)
            #pragma unroll
            for (int n = 0; n < 2; n++)
                #pragma unroll
                for (int e = 0; e < 4; e++) s[m][n][e] = 0.f;
        #pragma unroll
        for (int ks = 0; ks < HD / 16; ks++) {
            uint32_t bfr[4];
            ldsm4(bfr, ks_ + ((lane & 7) + (lane >> 4) * 8) * LD + ks * 16 + ((lane >> 3) & 1) * 8);
            #pragma unroll
            for (int m = 0; m < MT; m++)
                if (m < n_mt) {
                    uint32_t qf[4];
                    ldsm4(qf, Qs + (m * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * LD + ks * 16 + (lane >> 4) * 8);
                    mma(s[m][0], qf, bfr[0], bfr[1]);
                    mma(s[m][1], qf, bfr[2], bfr[3]);
                }
        }
        const int jbase = p * PAGE + warp * 16 + 2 * t;
        uint32_t pa[MT][4];
        #pragma unroll
        for (int m = 0; m < MT; m++)
            if (m < n_mt) {
                const int pos[2] = {row_pos[m * 16 + g], row_pos[m * 16 + g + 8]};
                float mx[2] = {-INFINITY, -INFINITY}, alpha[2], rs[2] = {0.f, 0.f};
                #pragma unroll
                for (int n = 0; n < 2; n++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = e >> 1, j = jbase + n * 8 + (e & 1);
                        const float v = j <= pos[r] ? capped(s[m][n][e], scale_log2e, cap_log2e) : -INFINITY;
                        s[m][n][e] = v;
                        mx[r] = fmaxf(mx[r], v);
                    }
                #pragma unroll
                for (int r = 0; r < 2; r++) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    const float m_new = fmaxf(m_i[m][r], mx[r]);
                    const float m_use = m_new == -INFINITY ? 0.f : m_new;
                    alpha[r] = exp2f(m_i[m][r] - m_use);
                    m_i[m][r] = m_new;
                    mx[r] = m_use;
                }
                #pragma unroll
                for (int n = 0; n < 2; n++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float pv = exp2f(s[m][n][e] - mx[e >> 1]);
                        s[m][n][e] = pv;
                        rs[e >> 1] += pv;
                    }
                #pragma unroll
                for (int r = 0; r < 2; r++) l_i[m][r] = l_i[m][r] * alpha[r] + rs[r];
                #pragma unroll
                for (int d = 0; d < HD / 8; d++) {
                    o[m][d][0] *= alpha[0]; o[m][d][1] *= alpha[0]; o[m][d][2] *= alpha[1]; o[m][d][3] *= alpha[1];
                }
                pa[m][0] = pack_bf16(s[m][0][0], s[m][0][1]);
                pa[m][1] = pack_bf16(s[m][0][2], s[m][0][3]);
                pa[m][2] = pack_bf16(s[m][1][0], s[m][1][1]);
                pa[m][3] = pack_bf16(s[m][1][2], s[m][1][3]);
            }
        #pragma unroll
        for (int dp = 0; dp < HD / 16; dp++) {
            uint32_t bfr[4];
            ldsm4t(bfr, vs_ + ((lane & 7) + ((lane >> 3) & 1) * 8) * LD + dp * 16 + (lane >> 4) * 8);
            #pragma unroll
            for (int m = 0; m < MT; m++)
                if (m < n_mt) {
                    mma(o[m][2 * dp], pa[m], bfr[0], bfr[1]);
                    mma(o[m][2 * dp + 1], pa[m], bfr[2], bfr[3]);
                }
        }
        __syncthreads();                                            // everyone is done with this stage
        if (p + NS < p_end) load_page(stage, p + NS);
        cp_commit();
    }
    cp_wait<0>();
    ik_pdl_launch_dependents();
    // the four warps' partial results, merged in warp order (the ring is free now)
    float* sm_o = (float*)Ks;                         // [4][ROWS][HD]
    float* sm_ml = sm_o + 4 * ROWS * HD;              // [4][ROWS][2]
    #pragma unroll
    for (int m = 0; m < MT; m++)
        if (m < n_mt) {
            #pragma unroll
            for (int r = 0; r < 2; r++) {
                float l = l_i[m][r];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int row = warp * ROWS + m * 16 + g + 8 * r;
                #pragma unroll
                for (int d = 0; d < HD / 8; d++) {
                    sm_o[row * HD + d * 8 + 2 * t] = o[m][d][2 * r];
                    sm_o[row * HD + d * 8 + 2 * t + 1] = o[m][d][2 * r + 1];
                }
                if (t == 0) { sm_ml[row * 2] = m_i[m][r]; sm_ml[row * 2 + 1] = l; }
            }
        }
    __syncthreads();
    const int n_splits = cut.n_shared + cut.n_own;
    for (int idx = threadIdx.x; idx < n_rows * HD; idx += 128) {
        const int r = idx / HD, x = idx % HD, rho = first_row + r;
        float mm = -INFINITY;
        #pragma unroll
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, sm_ml[(w * ROWS + r) * 2]);
        const float m_use = mm == -INFINITY ? 0.f : mm;
        float acc = 0.f, ll = 0.f;
        #pragma unroll
        for (int w = 0; w < 4; w++) {
            const float a = exp2f(sm_ml[(w * ROWS + r) * 2] - m_use);
            acc += sm_o[(w * ROWS + r) * HD + x] * a;
            ll += sm_ml[(w * ROWS + r) * 2 + 1] * a;
        }
        const size_t slot = ((size_t)(first_seq + rho / G) * nh + kvh * G + rho % G) * n_splits + split;
        part_o[slot * HD + x] = acc;
        if (x == 0) { part_ml[slot * 2] = mm; part_ml[slot * 2 + 1] = ll; }
    }
}

// Joins a (sequence, head)'s partials: the shared chunks, then its own, then the sink.
__global__ void attn_shared_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, bf16* __restrict__ out,
                                        const int* __restrict__ kv_lens, const int* __restrict__ shared, int table_cols, int nh, int sink,
                                        const float* __restrict__ sink_v, Cut cut) {
    ik_pdl_wait();
    ik_pdl_launch_dependents();
    const int b = blockIdx.x, h = blockIdx.y;
    const int pages = min((max(kv_lens[b], 0) + PAGE - 1) / PAGE, table_cols), together = min(max(shared[b], 0), table_cols);
    const int n_s = chunks_of(together, cut.shared_chunk, cut.n_shared), n_o = chunks_of(pages - min(together, pages), cut.own_chunk, cut.n_own);
    const size_t base = ((size_t)b * nh + h) * (cut.n_shared + cut.n_own);
    const float m_sink = sink ? (sink_v ? sink_v[h] * 1.4426950408889634f : 0.f) : -INFINITY;
    auto at = [&](int i) { return base + (i < n_s ? i : cut.n_shared + i - n_s); };
    float mm = m_sink;
    for (int i = 0; i < n_s + n_o; i++) mm = fmaxf(mm, part_ml[at(i) * 2]);
    const float m_use = mm == -INFINITY ? 0.f : mm;
    for (int x = threadIdx.x; x < HD; x += blockDim.x) {
        float acc = 0.f, ll = sink ? exp2f(m_sink - m_use) : 0.f;
        for (int i = 0; i < n_s + n_o; i++) {
            const float a = exp2f(part_ml[at(i) * 2] - m_use);
            acc += part_o[at(i) * HD + x] * a;
            ll += part_ml[at(i) * 2 + 1] * a;
        }
        out[((size_t)b * nh + h) * HD + x] = __float2bfloat16_rn(mm == -INFINITY ? 0.f : acc / ll);
    }
}

}  // namespace

IK_EXPORT int ik_attn_shared_head_dim() { return HD; }

// part_o: [B, nh, n_shared + n_own, HD] floats, part_ml: [B, nh, n_shared + n_own, 2] floats, both owned by the caller.  starts: [n_groups + 1], shared: [B], on the
// device; max_members: no group is larger (rows beyond it would be left out).
IK_EXPORT int ik_attn_shared(const void* q, const void* k_pages, const void* v_pages, void* out, float* part_o, float* part_ml, const int* kv_lens,
                             const int* table, int table_stride, int table_cols, const int* starts, const int* shared, int n_groups, int max_members, int B,
                             int nh, int nkv, float scale, float softcap, int sink, const float* sink_v, int page_size, int n_pages, int shared_chunk,
                             int n_shared, int own_chunk, int n_own, int* status, cudaStream_t stream) {
    const float sc_a = softcap > 0.f ? scale / softcap : scale * 1.4426950408889634f, sc_b = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
    if (B <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || page_size != PAGE || n_groups < 0 || max_members <= 0 || max_members > B || shared_chunk <= 0 || own_chunk <= 0 ||
        n_shared <= 0 || n_own <= 0 || nkv > 65535 || nh > 65535 || table_cols <= 0 || table_stride < table_cols || n_pages <= 0)
        return IK_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return IK_UNSUPPORTED;
    const int G = nh / nkv, row_tiles = (max_members * G + ROWS - 1) / ROWS;
    const Cut cut{shared_chunk, n_shared, own_chunk, n_own};
    const long long blocks = (long long)n_groups * row_tiles * n_shared + (long long)B * ((G + ROWS - 1) / ROWS) * n_own;
    if (blocks > 0x7fffffff) return IK_UNSUPPORTED;
    const size_t q_bytes = (size_t)ROWS * LD * sizeof(bf16), stage_bytes = (size_t)2 * PAGE * LD * sizeof(bf16);
    const size_t merge_bytes = (size_t)4 * ROWS * (HD + 2) * sizeof(float);
    constexpr int NS = HD <= 64 ? 4 : HD <= 128 ? 2 : 2;
    const size_t smem = q_bytes + (NS * stage_bytes > merge_bytes ? NS * stage_bytes : merge_bytes);
    auto kern = attn_shared_kernel<NS>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    IK_RETURN_IF_ERROR(ik_launch(kern, dim3((unsigned)blocks, nkv), 128, smem, stream, (const bf16*)q, (const bf16*)k_pages, (const bf16*)v_pages, part_o, part_ml,
                                 kv_lens, table, table_stride, table_cols, starts, shared, n_groups, row_tiles, B, nh, nkv, sc_a, sc_b, n_pages, cut, status));
    IK_RETURN_IF_ERROR(ik_launch_family(IK_FAMILY_ATTENTION_MERGE, attn_shared_join_kernel, dim3(B, nh), HD < 128 ? HD : 128, 0, stream, (const float*)part_o,
                                        (const float*)part_ml, (bf16*)out, kv_lens, shared, table_cols, nh, sink, sink_v, cut));
    IK_LAUNCH_STATUS();
}
