// The best continuations of beam search.  R requests have K beams each; beam b of request r has a sum of log probabilities c[r,b] and a
// row of logits l[r,b,:].  A candidate (b, v) scores c[r,b] + (l[r,b,v] - lse[r,b]) with lse[r,b] = log sum_v exp l[r,b,v]; the n
// largest of a request are wanted in descending order, equal ones by ascending b V + v.
//
// One pass over the logits.  Slices of a row go to blocks of their own (beam_rows_kernel): a block keeps its slice in registers, forms the
// slice's maximum and sum of exponentials, and finds its n largest logits; within a row the order of the logits is the order of the
// scores, so only those can be among a request's n best.  A second kernel (beam_merge_kernel, a block per request) joins the slices' sums into
// the beams' lse and picks from the lists.
//
// Finding the n largest without a sort: of the threads' own largest elements (every thread holds up to 32), the n-th largest, tau, is a lower
// bound of the slice's n-th largest, and only the n threads whose largest is at least tau hold elements >= tau.  So at most 32 n
// elements are gathered, whatever the data, and usually hardly more than n; their ranks are counted.  An element's key is its value (as an integer that
// orders like the value) above its place's complement, so keys are distinct and equal values come by ascending place.  The merge does the same with
// the lists: the n-th largest head is a bound, and only n lists have entries above it.
//
// Scores are formed and compared in 64 bits (two beams' candidates may be closer than a float of their size can tell) and rounded once;
// exponentials are floats, summed in float over 32 terms and in 64 bits beyond.  A logit of -inf or NaN is no candidate; neither is any of a beam
// whose sum is -inf or NaN.  Where a row has logits of +inf, they share the probability.  Places without a candidate: score -inf, beam and token -1.
#include <math.h>
#define IK_FAMILY 16
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int BT = 256, BE = 32, SLICE = BT * BE;                    // threads, elements of a thread and of a block
constexpr int BEAMS = 16, OUT = 32, SLICES = 128;                    // most beams, results and slices of a row

__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ u64 key_of(float v, uint32_t at) { return ((u64)order_key(v) << 32) | (uint32_t)~at; }

__device__ __forceinline__ u64 shfl_xor64(u64 v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }

// A warp's 32 keys in descending order (lane 0 the largest): bitonic.
__device__ __forceinline__ u64 warp_sort_desc(u64 k, int lane) {
    #pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
        #pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const u64 o = shfl_xor64(k, step);
            const bool up = (lane & size) == 0, first = (lane & step) == 0;     // up: descending half
            k = (up == first) ? (k > o ? k : o) : (k < o ? k : o);
        }
    return k;
}
// Of two such lists the 32 largest, in order: the larger of a[i] and b[31 - i] are those, as a bitonic sequence.
__device__ __forceinline__ u64 warp_merge_desc(u64 a, u64 b_reversed, int lane) {
    u64 k = a > b_reversed ? a : b_reversed;
    #pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
        const u64 o = shfl_xor64(k, step);
        k = ((lane & step) == 0) ? (k > o ? k : o) : (k < o ? k : o);
    }
    return k;
}

// scratch: keys [rows][slices][n], then (maximum, sum) [rows][slices] as doubles
__global__ void __launch_bounds__(BT)
beam_rows_kernel(const float* __restrict__ logits, long long ldl, const float* __restrict__ sums, int V, int n, int slices,
                 u64* __restrict__ keys, double2* __restrict__ stats) {
    __shared__ u64 sorted[BT / 32][32];
    __shared__ u64 cand[OUT * BE];
    __shared__ float red_m[BT / 32];
    __shared__ double red_s[BT / 32];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x, slice = blockIdx.y;
    u64* const out = keys + ((size_t)row * slices + slice) * n;
    if (!(sums[row] > -INFINITY)) return;                              // a dead beam: the merge does not look at its lists
    const float* const w = logits + (long long)row * ldl;
    const int per = (V + slices - 1) / slices, lo = slice * per, hi = min(V, lo + per);
    // element e of a thread stands at lo + e BT + tid, whatever the row's alignment: equal rows give equal sums, so that equal candidates stay equal
    float v[BE];
    #pragma unroll
    for (int e = 0; e < BE; e++) v[e] = lo + e * BT + tid < hi ? w[lo + e * BT + tid] : -INFINITY;
    float m = -INFINITY;
    #pragma unroll
    for (int e = 0; e < BE; e++) {
        v[e] = v[e] > -INFINITY ? v[e] : -INFINITY;                    // NaN too
        m = fmaxf(m, v[e]);
    }
    // the thread's largest, the first of equals
    int best = 0;
    #pragma unroll
    for (int e = BE - 1; e >= 0; e--) best = v[e] == m ? e : best;
    auto place = [&](int e) { return (uint32_t)(lo + e * BT + tid); };
    const u64 mine = m > -INFINITY ? key_of(m, place(best)) : 0ull;
    u64 k = warp_sort_desc(mine, lane);
    sorted[warp][lane] = k;
    float mm = m;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    if (lane == 0) red_m[warp] = mm;
    if (tid == 0) n_cand = 0;
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < BT / 32; i++) mm = fmaxf(mm, red_m[i]);
    // the slice's sum of exponentials (elements equal to the maximum count 1, an infinite one too)
    float s = 0.f;
    #pragma unroll
    for (int e = 0; e < BE; e++) s += v[e] == mm ? 1.0f : expf(v[e] - mm);
    double ss = mm > -INFINITY ? (double)s : 0.0;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) red_s[warp] = ss;
    // the 32 largest of the threads' largest
    #pragma unroll
    for (int half = BT / 64; half > 0; half >>= 1) {
        if (warp < half) k = warp_merge_desc(k, sorted[warp + half][31 - lane], lane);
        __syncthreads();
        if (warp < half) sorted[warp][lane] = k;
        __syncthreads();
    }
    if (tid == 0) {
        double t = 0.0;
        for (int i = 0; i < BT / 32; i++) t += red_s[i];
        stats[(size_t)row * slices + slice] = make_double2((double)mm, t);
    }
    const u64 tau = max(sorted[0][n - 1], 1ull);
    if (mine >= tau) {
        #pragma unroll
        for (int e = 0; e < BE; e++)
            if (v[e] > -INFINITY) {
                const u64 c = key_of(v[e], place(e));
                if (c >= tau) cand[atomicAdd(&n_cand, 1)] = c;        // at most n threads come here: never more than n BE
            }
    }
    __syncthreads();
    const int c = n_cand;
    for (int i = tid; i < c; i += BT) {
        const u64 me = cand[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += cand[j] > me;
        if (rank < n) out[rank] = me;
    }
    for (int i = c + tid; i < n; i += BT) out[i] = 0ull;
}

// A candidate of the merge: descending scores, equal ones by ascending place (beam * V + token).
__device__ __forceinline__ bool ahead(double s, uint32_t at, double s2, uint32_t at2) { return s > s2 || (s == s2 && at < at2); }

__global__ void __launch_bounds__(BT)
beam_merge_kernel(const u64* __restrict__ keys, const double2* __restrict__ stats, const float* __restrict__ sums, int K, int V, int n, int slices,
                  float* __restrict__ out_s, int* __restrict__ out_b, int* __restrict__ out_v) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int lists = K * slices;
    double* const head_s = reinterpret_cast<double*>(smem);            // [lists]
    uint32_t* const head_at = reinterpret_cast<uint32_t*>(head_s + lists);
    __shared__ double cand_s[OUT * OUT];
    __shared__ uint32_t cand_at[OUT * OUT];
    __shared__ int picked[OUT];
    __shared__ double lse[BEAMS], base[BEAMS];
    __shared__ int shares[BEAMS];                                      // a beam with infinite logits
    __shared__ int n_picked, n_cand, tau_list;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x;
    for (int b = warp; b < K; b += BT / 32) {
        const float c = sums[r * K + b];
        const bool live = c > -INFINITY;
        double m = -INFINITY, s = 0.0;
        if (live) {
            for (int i = lane; i < slices; i += 32) m = fmax(m, stats[(size_t)(r * K + b) * slices + i].x);
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int i = lane; i < slices; i += 32) {
                const double2 t = stats[(size_t)(r * K + b) * slices + i];
                s += t.x == m ? t.y : t.y * exp(t.x - m);
            }
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) {
            const bool any = live && m > -INFINITY, inf = m == INFINITY;
            base[b] = any ? (double)c : -INFINITY;
            lse[b] = any ? (inf ? log(s) : m + log(s)) : 0.0;
            shares[b] = inf;
        }
    }
    if (tid == 0) { n_picked = n_cand = 0; tau_list = -1; }
    __syncthreads();
    auto score = [&](int b, u64 key) {                                 // -inf: not a candidate
        if (key == 0ull || !(base[b] > -INFINITY)) return -(double)INFINITY;
        double l = (double)order_value((uint32_t)(key >> 32));
        if (shares[b]) { if (l < INFINITY) return -(double)INFINITY; l = 0.0; }
        return base[b] + (l - lse[b]);
    };
    auto place = [&](int b, u64 key) { return (uint32_t)b * (uint32_t)V + (uint32_t)~(uint32_t)key; };
    for (int i = tid; i < lists; i += BT) {
        const int b = i / slices;
        const u64 key = base[b] > -INFINITY ? keys[((size_t)r * lists + i) * n] : 0ull;
        head_s[i] = score(b, key);
        head_at[i] = head_s[i] > -INFINITY ? place(b, key) : 0xffffffffu - i;
    }
    __syncthreads();
    if (lists > n)                                                      // the n-th largest head
        for (int i = tid; i < lists; i += BT) {
            const double s = head_s[i];
            const uint32_t at = head_at[i];
            int rank = 0;
            for (int j = 0; j < lists; j++) rank += ahead(head_s[j], head_at[j], s, at);
            if (rank == n - 1) tau_list = i;
        }
    __syncthreads();
    const double tau_s = tau_list < 0 ? -(double)INFINITY : head_s[tau_list];
    const uint32_t tau_at = tau_list < 0 ? 0xffffffffu : head_at[tau_list];
    for (int i = tid; i < lists; i += BT)
        if (head_s[i] > -INFINITY && !ahead(tau_s, tau_at, head_s[i], head_at[i])) picked[atomicAdd(&n_picked, 1)] = i;
    __syncthreads();
    for (int p = warp; p < n_picked; p += BT / 32) {
        const int i = picked[p], b = i / slices;
        if (lane < n) {
            const u64 key = keys[((size_t)r * lists + i) * n + lane];
            const double s = score(b, key);
            const uint32_t at = place(b, key);
            if (s > -INFINITY && !ahead(tau_s, tau_at, s, at)) {
                const int slot = atomicAdd(&n_cand, 1);
                cand_s[slot] = s;
                cand_at[slot] = at;
            }
        }
    }
    __syncthreads();
    const int c = n_cand;
    for (int i = tid; i < c; i += BT) {
        const double s = cand_s[i];
        const uint32_t at = cand_at[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += ahead(cand_s[j], cand_at[j], s, at);
        if (rank < n) {
            out_s[r * n + rank] = (float)s;
            out_b[r * n + rank] = (int)(at / (uint32_t)V);
            out_v[r * n + rank] = (int)(at % (uint32_t)V);
        }
    }
    for (int i = c + tid; i < n; i += BT) { out_s[r * n + i] = -INFINITY; out_b[r * n + i] = out_v[r * n + i] = -1; }
}

int slices_of(int V) { return (V + SLICE - 1) / SLICE; }

}  // namespace

// Bytes of scratch, or -1 where the sizes are not supported.
IK_EXPORT long long ik_beam_select_scratch(int R, int K, int V, int n) {
    if (R <= 0 || K <= 0 || V <= 0 || n <= 0 || K > BEAMS || n > OUT || slices_of(V) > SLICES || (long long)R * K > 0x7fffffff / 2) return -1;
    return (long long)R * K * slices_of(V) * (n * 8ll + 16);
}

// scratch: ik_beam_select_scratch bytes on 16 bytes.
IK_EXPORT int ik_beam_select(const float* logits, long long ldl, const float* sums, int R, int K, int V, int n, void* scratch, float* out_s,
                             int* out_b, int* out_v, cudaStream_t stream) {
    if (ik_beam_select_scratch(R, K, V, n) < 0 || (ldl < V && R * K > 1) || ((uintptr_t)logits & 3) || ((uintptr_t)scratch & 15)) return IK_BAD_ARGUMENT;
    const int slices = slices_of(V);
    double2* const stats = reinterpret_cast<double2*>(scratch);
    u64* const keys = reinterpret_cast<u64*>(stats + (size_t)R * K * slices);
    IK_RETURN_IF_ERROR(ik_launch(beam_rows_kernel, dim3(R * K, slices), BT, 0, stream, logits, ldl, sums, V, n, slices, keys, stats));
    const size_t smem = (size_t)K * slices * 12;
    IK_RETURN_IF_ERROR(ik_launch(beam_merge_kernel, dim3(R), BT, smem, stream, (const u64*)keys, (const double2*)stats, sums, K, V, n, slices, out_s, out_b, out_v));
    IK_LAUNCH_STATUS();
}
