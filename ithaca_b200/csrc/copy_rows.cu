// Copies of rows within tensors of a cache, many tensors and many rows in one launch: the pages and states that a forked sequence needs for
// itself.  A job is a tensor [entries, rows, segments, bytes]; a move copies the first `part` bytes of every segment of row src to rows
// dst_0, dst_1, ..., in all entries.  A page of a layer is a row, its kv heads are the segments, and `part` is what the filled positions take;
// a state is one segment, copied whole.  What lies behind `part` in a destination stays as it is.
//
// Sources and destinations of a job are disjoint (the caller checks), so no order among the copies matters.  Bound by memory: every
// source byte is read once for all its destinations and every destination byte is written once.  Job and move lists travel in the kernel's
// parameters: no upload, and a captured launch keeps its own.
//
// A block moves 8 KB of a segment with four 16-byte loads under way per thread.  us in a replayed graph on B200: six sequences with states of 32 MB each become 24, 126
// (814 MB, the copy rate); the begun pages of 16 beams in 32 layers, 136 MB in 8,192 segments of 0.25 to 16 KB, 27 (5.1 TB/s); one page of a small model 1.5.  Blocks of 64 to 512
// threads with 2 to 8 loads: 124-129, 27-37, 1.5-2.2.
#include <string.h>
#define IK_FAMILY 1
#include "common.cuh"

namespace {

constexpr int JOBS = 16, MOVES = 160, DSTS = 320, FAN = 8;             // of one launch; the host cuts longer lists
constexpr int CT = 128, CU = 4;                                        // threads, vectors under way per thread

struct Job {
    char* base;
    long long entry_stride, row_stride, seg_stride;                     // bytes
    int entries, segs, chunks;                                          // chunks: pieces of CT * CU vectors of the longest part
    int width;                                                          // bytes of a vector: 16, 4 or 2
    int first_move, n_moves;
    long long first_block;                                              // of the launch's blocks
};
struct Move { int src, first_dst, n_dst; long long part; };
struct Work {
    int n_jobs;
    Job jobs[JOBS];
    Move moves[MOVES];
    int dst[DSTS];
};

template <typename T>
__device__ __forceinline__ void copy_piece(const char* src, char* base, long long row_stride, const int* dst, int n_dst, long long part, long long at) {
    constexpr int W = sizeof(T);
    const long long n = part / W;
    T x[CU];
    #pragma unroll
    for (int i = 0; i < CU; i++) {
        const long long j = at + i * CT + threadIdx.x;
        if (j < n) x[i] = reinterpret_cast<const T*>(src)[j];
    }
    for (int d = 0; d < n_dst; d++) {
        T* const to = reinterpret_cast<T*>(base + dst[d] * row_stride);
        #pragma unroll
        for (int i = 0; i < CU; i++) {
            const long long j = at + i * CT + threadIdx.x;
            if (j < n) to[j] = x[i];
        }
    }
}

__global__ void __launch_bounds__(CT) copy_rows_kernel(const __grid_constant__ Work w) {
    ik_pdl_wait();
    ik_pdl_launch_dependents();
    int ji = 0;
    while (ji + 1 < w.n_jobs && (long long)blockIdx.x >= w.jobs[ji + 1].first_block) ji++;
    const Job& job = w.jobs[ji];
    int i = (int)((long long)blockIdx.x - job.first_block);
    const int chunk = i % job.chunks; i /= job.chunks;
    const int seg = i % job.segs; i /= job.segs;
    const int mv = i % job.n_moves, entry = i / job.n_moves;
    const Move& move = w.moves[job.first_move + mv];
    char* const base = job.base + entry * job.entry_stride + seg * job.seg_stride;
    const char* const src = base + move.src * job.row_stride;
    const int* const dst = w.dst + move.first_dst;
    const long long at = (long long)chunk * CT * CU;
    if (job.width == 16) {
        copy_piece<uint4>(src, base, job.row_stride, dst, move.n_dst, move.part, at);
        // the rest of a part that is no multiple of 16 bytes
        const long long whole = move.part & ~15ll;
        if (chunk == 0 && threadIdx.x < (int)(move.part - whole) / 2) {
            const unsigned short x = reinterpret_cast<const unsigned short*>(src + whole)[threadIdx.x];
            for (int d = 0; d < move.n_dst; d++) reinterpret_cast<unsigned short*>(base + dst[d] * job.row_stride + whole)[threadIdx.x] = x;
        }
    } else if (job.width == 4) copy_piece<uint32_t>(src, base, job.row_stride, dst, move.n_dst, move.part, at);
    else copy_piece<unsigned short>(src, base, job.row_stride, dst, move.n_dst, move.part, at);
}

}  // namespace

// jobs: per job 10 numbers: base address, entries, entry stride, rows, row stride, segments, segment stride, bytes of a position, first move, number of moves (strides and
// sizes in bytes).  moves: per move src, dst, positions.  The lists are read before the call returns.
IK_EXPORT int ik_copy_rows(const long long* jobs, int n_jobs, const int* moves, int n_moves, cudaStream_t stream) {
    if (n_jobs < 0 || n_moves < 0) return IK_BAD_ARGUMENT;
    constexpr long long BLOCKS = 0x7fffffff;                             // of a launch
    auto width_of = [](const long long* a) {
        const long long all = a[0] | a[2] | a[4] | a[6];
        return all % 16 == 0 ? 16 : (all | a[7]) % 4 == 0 ? 4 : 2;
    };
    auto chunks_of = [&](const long long* a, long long part) { const long long piece = (long long)CT * CU * width_of(a); return (part + piece - 1) / piece; };
    for (int j = 0; j < n_jobs; j++) {
        const long long* a = jobs + 10 * j;
        if (!a[0] || a[1] <= 0 || a[1] > 0x7fffffff || a[3] <= 0 || a[5] <= 0 || a[5] > 0x7fffffff || a[7] <= 0 || (a[7] & 1) || (a[0] & 1) || (a[2] & 1) || (a[4] & 1) || (a[6] & 1) ||
            a[8] < 0 || a[9] < 0 || a[8] + a[9] > n_moves)
            return IK_BAD_ARGUMENT;
        int longest = 0;
        for (long long i = a[8]; i < a[8] + a[9]; i++) {
            const int* m = moves + 3 * i;
            if (m[0] < 0 || m[0] >= a[3] || m[1] < 0 || m[1] >= a[3] || m[0] == m[1] || m[2] < 0) return IK_BAD_ARGUMENT;
            if (m[2] > longest) longest = m[2];
        }
        // a launch takes all entries and segments of a job, so that many blocks have to fit: told here, before anything is copied
        if ((double)chunks_of(a, longest * a[7]) * (double)a[5] * (double)a[1] * (double)(a[9] < MOVES ? a[9] : MOVES) > (double)BLOCKS) return IK_UNSUPPORTED;
    }
    Work w;
    w.n_jobs = 0;
    int used = 0, used_dst = 0;
    long long blocks = 0;
    auto flush = [&]() -> int {
        if (blocks > 0) {
            cudaError_t e = ik_launch(copy_rows_kernel, dim3((unsigned)blocks), CT, 0, stream, w);
            if (e != cudaSuccess) return (int)e;
        }
        w.n_jobs = used = used_dst = 0;
        blocks = 0;
        return IK_OK;
    };
    for (int j = 0; j < n_jobs; j++) {
        const long long* a = jobs + 10 * j;
        long long i = a[8];
        const long long end = a[8] + a[9];
        while (i < end) {
            if (w.n_jobs == JOBS || used == MOVES || used_dst + FAN > DSTS) { int st = flush(); if (st) return st; }
            Job& job = w.jobs[w.n_jobs];
            job.base = (char*)a[0]; job.entries = (int)a[1]; job.entry_stride = a[2]; job.row_stride = a[4]; job.segs = (int)a[5]; job.seg_stride = a[6];
            job.width = width_of(a);
            job.first_move = used; job.first_block = blocks;
            const long long from = i;
            long long most = 0;
            while (i < end && used < MOVES && used_dst + FAN <= DSTS) {
                Move& m = w.moves[used];
                m.src = moves[3 * i]; m.part = moves[3 * i + 2] * a[7]; m.first_dst = used_dst; m.n_dst = 0;
                // neighbours with the same source and length share one reading of it
                const int src = moves[3 * i], rows = moves[3 * i + 2];
                while (i < end && m.n_dst < FAN && moves[3 * i] == src && moves[3 * i + 2] == rows) { w.dst[used_dst++] = moves[3 * i + 1]; m.n_dst++; i++; }
                if (m.part > most) most = m.part;
                used++;
            }
            job.n_moves = used - job.first_move;
            job.chunks = (int)chunks_of(a, most);
            const long long more = (long long)job.chunks * job.segs * job.n_moves * job.entries;
            if (more == 0 || blocks + more > BLOCKS) {                   // nothing to copy, or this job goes into the next launch
                used = job.first_move;
                used_dst = used ? w.moves[used - 1].first_dst + w.moves[used - 1].n_dst : 0;
                if (more) { i = from; int st = flush(); if (st) return st; }
                continue;
            }
            blocks += more;
            w.n_jobs++;
        }
    }
    return flush();
}
