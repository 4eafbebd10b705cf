// The best continuations of beam search.  R requests have K beams each; beam b of request r has a sum of log probabilities c[r,b] and a
// row of logits l[r,b,:].  A candidate (b, v) scores c[r,b] + (l[r,b,v] - lse[r,b]) with lse[r,b] = log sum_v exp l[r,b,v]; the n
// largest of a request are wanted in descending order, equal ones by ascending b V + v.
//
// One pass over the logits and a second look at small pieces of them, no sort.  beam_tiles_kernel: a warp takes a tile of 1,024 logits of a row and leaves
// the tile's maximum, where it stands, the one behind it, and the sum of exponentials below it.  beam_merge_kernel, a block per request: joins the
// sums into the beams' lse, and with them every tile's maximum into a score.  Of these the n-th largest is a lower bound of the n-th best candidate (n tiles
// have a candidate at least as good), and only tiles that are not below it can hold any of the n best: hardly more than n.  Of a tile whose second largest is below the
// bound the maximum is all that counts; the others are read again (L2 has them) for what is not below it.  What is gathered, usually hardly more than n, is
// ranked by counting.  Where there is more (few tiles, sorted or constant logits), a tile's candidates are held against the n-th best of its lanes' two best each, a tile
// that this does not tell apart gives its n best in sorted lists, and so do all together.  Where many tiles are as good as the bound, the n best are found by exact
// comparisons with their places.
//
// Bound by memory where there are many rows, by the merge's chain of dependent steps where there are few.  us in a replayed graph on B200, tiles + the rest: 32 requests of 16
// beams over 128,256 tokens 42 + 8 (263 MB: the pass runs at the copy rate), 16 of 8 over 50,257 6.3 + 5.2, one of 4 over 128,256 2.6 + 4.6.  A first version that
// took every slice's n best by sorting its threads' maxima in the pass itself: 230, 33, 13.  Without a tile's second largest, every chosen tile was read again:
// 3 to 6 us more.  Both in one launch, a cluster of 8 or 16 blocks to a request: one of 4 12.6 and 9.8 (7.4 here), 16 of 8 19.  Many candidates a tile: one request of
// 16 beams over 1,000 tokens, 32 results 11 (85 with the tile's best one at a time and everything ranked by counting); equal logits, 4 beams over 128,256, 32 results 38 (234).
//
// Scores are formed from float logits, a float sum and the beam's lse in 64 bits, compared so and rounded once: a beam's candidates are in their exact order, whatever its sum.
// The lse comes from float exponentials, summed in float within a tile and in 64 bits beyond: off by less than 3.3e-6 by its error bound, by up to 1.8e-7 as measured (1,000 to
// 128,256 logits).  Candidates of different beams that are closer than that may change places.  A logit of -inf or NaN is no candidate; neither is any of a beam
// whose sum is -inf or NaN, nor one whose score is below what a float holds.  Where a row has logits of +inf, they share the probability.  Places without a candidate: score -inf, beam and token -1.
#include <math.h>
#define IK_FAMILY 16
#include "common.cuh"

namespace {

constexpr int TILE = 1024, PER = TILE / 32;                            // logits of a tile, of a lane
constexpr int RT = 256, MT = 512, MW = MT / 32;                        // threads of the two kernels
constexpr int BEAMS = 16, OUT = 32, TILES = 1024;                      // most beams, results and tiles of a row
constexpr int PICKS = 40;                                              // tiles that the merge takes as they come
constexpr int CANDS = 160;                                             // candidates that are ranked without a second thought

// What a tile leaves: its maximum, the one behind it (equal to it where it stands twice), the sum of exponentials below the maximum; the maximum's place in its row and the
// beam in the upper 12 bits.
struct __align__(16) Tile { float top, second, sum; uint32_t where; };
static_assert(TILES * TILE <= 1 << 20 && BEAMS <= 1 << 12, "a place and a beam share 32 bits");
__device__ __forceinline__ uint32_t place_of(const Tile& t) { return t.where & 0xfffffu; }
__device__ __forceinline__ int beam_of(const Tile& t) { return (int)(t.where >> 20); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A lane's logits of a tile that starts at `lo`; what lies behind the row is -inf.  VEC: rows on 16 bytes of a multiple of four logits.  The order in which a
// tile is summed does not depend on where it lies in memory, so equal rows give equal sums and equal candidates stay equal.
template <bool VEC> __device__ __forceinline__ int place_in(int e, int lane) { return VEC ? (e >> 2) * 128 + lane * 4 + (e & 3) : e * 32 + lane; }
template <bool VEC>
__device__ __forceinline__ void load_tile(float (&v)[PER], const float* __restrict__ w, int lo, int V, int lane) {
    if (VEC) {
        #pragma unroll
        for (int i = 0; i < PER / 4; i++) {
            const int at = lo + place_in<true>(4 * i, lane);
            const float4 x = at < V ? *reinterpret_cast<const float4*>(w + at) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
        }
    } else {
        #pragma unroll
        for (int e = 0; e < PER; e++) v[e] = lo + e * 32 + lane < V ? w[lo + e * 32 + lane] : -INFINITY;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(RT, 5)
beam_tiles_kernel(const float* __restrict__ logits, long long ldl, const float* __restrict__ sums, int K, int V, int tiles, Tile* __restrict__ out) {
    ik_pdl_wait();
    ik_pdl_launch_dependents();
    const int lane = threadIdx.x & 31, row = blockIdx.x, tile = blockIdx.y * (RT / 32) + (threadIdx.x >> 5);
    if (tile >= tiles) return;
    const int lo = tile * TILE, beam = row % K;
    if (!(sums[row] > -INFINITY)) {                                    // a dead beam: not read
        if (lane == 0) out[(size_t)row * tiles + tile] = Tile{-INFINITY, -INFINITY, 0.f, (uint32_t)beam << 20 | (uint32_t)lo};
        return;
    }
    float v[PER];
    load_tile<VEC>(v, logits + (long long)row * ldl, lo, V, lane);
    constexpr int GROUPS = 4, IN = PER / GROUPS;
    float group[GROUPS], top = -INFINITY;
    #pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        group[g] = -INFINITY;
        #pragma unroll
        for (int e = 0; e < IN; e++) group[g] = fmaxf(group[g], v[g * IN + e]);       // (the other operand where one is NaN)
        top = fmaxf(top, group[g]);
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // where the maximum stands first, how often, and what comes behind it: only the groups that have it are looked through
    int first = TILE, times = 0;
    float second = -INFINITY;
    #pragma unroll
    for (int g = GROUPS - 1; g >= 0; g--)
        if (__any_sync(0xffffffffu, group[g] == top)) {
            #pragma unroll
            for (int e = IN - 1; e >= 0; e--) {
                const bool is = v[g * IN + e] == top;
                first = is ? place_in<VEC>(g * IN + e, lane) : first;
                times += is;
                second = fmaxf(second, is ? -INFINITY : v[g * IN + e]);
            }
        } else second = fmaxf(second, group[g]);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) second = fmaxf(second, __shfl_xor_sync(0xffffffffu, second, o));
    if (__reduce_add_sync(0xffffffffu, times) > 1) second = top;
    first = __reduce_min_sync(0xffffffffu, first);
    float s = 0.f;
    if (top < INFINITY) {
        // the difference first, then the factor: a product with -top log2 e inside would carry one rounding error into all terms.  The bound keeps NaN and
        // -inf out of the sum (2^-150 is 0)
        #pragma unroll
        for (int e = 0; e < PER; e++) s += ex2(fmaxf((v[e] - top) * 1.4426950408889634f, -150.f));
    } else {
        #pragma unroll
        for (int e = 0; e < PER; e++) s += v[e] == INFINITY ? 1.f : 0.f;
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) out[(size_t)row * tiles + tile] = Tile{top, second, s, (uint32_t)beam << 20 | (uint32_t)(lo + first)};
}

// A candidate: its score as an integer that orders like it, and its place (beam * V + token); no candidate: 0 and NOWHERE.  Ordered by descending scores, equal ones by
// ascending place.  Compared without branches: a warp that jumps at every comparison takes 190 cycles for one step of a ranking, without jumps a tenth of that.
struct __align__(16) Cand { unsigned long long s; uint32_t at; };
constexpr uint32_t NOWHERE = 0xffffffffu;
__device__ __forceinline__ Cand none() { return Cand{0ull, NOWHERE}; }
__device__ __forceinline__ unsigned long long order_key(double v) {    // more than 0
    const long long b = __double_as_longlong(v);
    return (unsigned long long)(b ^ ((b >> 63) | (long long)0x8000000000000000ull));
}
__device__ __forceinline__ double order_value(unsigned long long k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ bool ahead(const Cand& a, const Cand& b) { return (a.s > b.s) | ((a.s == b.s) & (a.at < b.at)); }
__device__ __forceinline__ Cand shfl_xor(const Cand& c, int m) { return Cand{__shfl_xor_sync(0xffffffffu, c.s, m), __shfl_xor_sync(0xffffffffu, c.at, m)}; }
__device__ __forceinline__ Cand shfl(const Cand& c, int from) { return Cand{__shfl_sync(0xffffffffu, c.s, from), __shfl_sync(0xffffffffu, c.at, from)}; }
__device__ __forceinline__ Cand pick(bool second, const Cand& a, const Cand& b) { return Cand{second ? b.s : a.s, second ? b.at : a.at}; }
__device__ __forceinline__ Cand better(const Cand& a, const Cand& b) { return pick(ahead(b, a), a, b); }

__device__ __forceinline__ float shfl_xor(float c, int m) { return __shfl_xor_sync(0xffffffffu, c, m); }
__device__ __forceinline__ float exchange(bool front, float mine, float other) { return front ? fmaxf(mine, other) : fminf(mine, other); }
__device__ __forceinline__ Cand exchange(bool front, const Cand& mine, const Cand& other) { return pick(front == ahead(other, mine), mine, other); }
__device__ __forceinline__ float better(float a, float b) { return fmaxf(a, b); }

// A warp's 32 candidates (or floats) in order, lane 0 the best: bitonic.
template <typename T>
__device__ __forceinline__ T warp_sort(T k, int lane) {
    #pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
        #pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const T o = shfl_xor(k, step);
            const bool front = ((lane & size) == 0) == ((lane & step) == 0);
            k = exchange(front, k, o);
        }
    return k;
}
// The best 32 of two sorted lists, in order: the better of a[i] and b[31 - i] are those, as a bitonic sequence.
template <typename T>
__device__ __forceinline__ T warp_merge(T a, const T& b_reversed, int lane) {
    a = better(a, b_reversed);
    #pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
        const T o = shfl_xor(a, step);
        const bool front = (lane & step) == 0;
        a = exchange(front, a, o);
    }
    return a;
}

// The best 32 of the block's warps' sorted lists, in order, at the front of `lists`.
__device__ __forceinline__ void block_best(Cand list, Cand* lists, int warp, int lane) {
    lists[warp * 32 + lane] = list;
    #pragma unroll 1
    for (int half = MW / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) list = warp_merge(list, lists[(warp + half) * 32 + 31 - lane], lane);
        __syncthreads();
        if (warp < half) lists[warp * 32 + lane] = list;
    }
    __syncthreads();
}

// How many of a list are ahead of its i-th (a warp).
__device__ __forceinline__ int rank_of(const Cand* list, int count, int i, int lane) {
    const Cand me = list[i];
    int rank = 0;
    for (int j = lane; j < count; j += 32) rank += ahead(list[j], me) ? 1 : 0;
    return __reduce_add_sync(0xffffffffu, rank);
}

// What the merge keeps of a beam: its sum (-inf: nothing to choose), its lse, whether infinite logits share its probability.
struct Beam { double base, lse; int shares; };
__device__ __forceinline__ double score_of(const Beam& b, float l) {
    if (b.shares) l = l < INFINITY ? -INFINITY : 0.f;
    const double s = b.base + ((double)l - b.lse);
    return l > -INFINITY ? s : -(double)INFINITY;                      // (a dead beam's sum is -inf, too)
}
__device__ __forceinline__ Cand cand_of(const Beam& b, float l, uint32_t at) {
    const double s = score_of(b, l);
    return pick((float)s > -INFINITY, none(), Cand{order_key(s), at});
}

template <bool VEC>
__global__ void __launch_bounds__(MT, 1)
beam_merge_kernel(const float* __restrict__ logits, long long ldl, const Tile* __restrict__ tile_of, const float* __restrict__ sums, int K, int V, int n, int tiles,
                  float* __restrict__ out_s, int* __restrict__ out_b, int* __restrict__ out_v) {
    __shared__ Beam beams[BEAMS];
    __shared__ float sorted[2 * MW][32];                               // lists of the merge's levels, one behind the other
    __shared__ Cand cand[PICKS * OUT], picked[OUT * 32];               // candidates; tiles by their maxima
    __shared__ int picked_tile[OUT * 32], chosen[PICKS], order[OUT];
    __shared__ int n_picked, n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x, total = K * tiles;
    if (tid == 0) n_picked = n_cand = 0;
    if (tid < OUT) order[tid] = -1;
    ik_pdl_wait();
    IK_AFTER_WAIT(tile_of);
    IK_AFTER_WAIT(sums);
    IK_AFTER_WAIT(logits);
    const Tile* const mine = tile_of + (size_t)r * total;
    for (int b = warp; b < K; b += MW) {
        const float c = sums[r * K + b];
        const Tile* const row = mine + b * tiles;
        float top = -INFINITY;
        double s = 0.0;
        #pragma unroll 4
        for (int i = lane; i < tiles; i += 32) top = fmaxf(top, row[i].top);
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        #pragma unroll 4
        for (int i = lane; i < tiles; i += 32) s += (double)(row[i].top == top ? row[i].sum : row[i].sum * expf(row[i].top - top));
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
            const bool any = top > -INFINITY, inf = top == INFINITY;
            beams[b] = Beam{any ? (double)c : -(double)INFINITY, any ? (inf ? log(s) : (double)top + log(s)) : 0.0, inf};
        }
    }
    __syncthreads();
    auto tile_cand = [&](int i) {
        const Tile t = mine[i];
        return cand_of(beams[beam_of(t)], t.top, (uint32_t)beam_of(t) * (uint32_t)V + place_of(t));
    };
    // a bound from the threads' best tiles.  Rounded to float the order stays (but for ties), so the n-th largest float is that of the n-th best, and the tiles
    // that are not below it are few: at most n threads have any, unless many are as good as equal
    float best = -INFINITY;
    for (int i = tid; i < total; i += MT) {
        const Tile t = mine[i];
        best = fmaxf(best, (float)score_of(beams[beam_of(t)], t.top));
    }
    float k = warp_sort(best, lane);
    sorted[warp][lane] = k;
    #pragma unroll 1
    for (int half = MW / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            k = warp_merge(k, sorted[2 * MW - 4 * half + warp + half][31 - lane], lane);
            sorted[2 * MW - 2 * half + warp][lane] = k;
        }
    }
    __syncthreads();
    const float bound = sorted[2 * MW - 2][n - 1];
    if (best > -INFINITY && best >= bound)
        for (int i = tid; i < total; i += MT) {
            const Cand c = tile_cand(i);
            if (c.s && (float)order_value(c.s) >= bound) {
                const int at = atomicAdd(&n_picked, 1);
                if (at < PICKS) { picked[at] = c; picked_tile[at] = i; }
            }
        }
    __syncthreads();
    int p = n_picked;
    if (p > PICKS) {                                                   // many equal ones: the bound from the exact order
        Cand mine_best = none();
        for (int i = tid; i < total; i += MT) mine_best = better(mine_best, tile_cand(i));
        __syncthreads();                                               // every thread has read the number that is counted anew
        if (tid == 0) n_picked = 0;
        block_best(warp_sort(mine_best, lane), cand, warp, lane);
        const Cand tau = cand[n - 1];
        if (mine_best.s && !ahead(tau, mine_best))
            for (int i = tid; i < total; i += MT) {
                const Cand c = tile_cand(i);
                if (c.s && !ahead(tau, c)) {
                    const int at = atomicAdd(&n_picked, 1);            // at most n threads with BEAMS * TILES / MT = 32 tiles each
                    picked[at] = c;
                    picked_tile[at] = i;
                }
            }
        __syncthreads();
        p = n_picked;
        for (int i = warp; i < p; i += MW) {
            const int rank = rank_of(picked, p, i, lane);
            if (lane == 0 && rank < n) chosen[rank] = i;
        }
        __syncthreads();
        p = min(p, n);
    } else if (tid < p) chosen[tid] = tid;
    __syncthreads();
    // their candidates that are not below the bound
    for (int t = warp; t < p; t += MW) {
        const int i = picked_tile[chosen[t]];
        const Tile tile = mine[i];
        const int b = beam_of(tile), lo = (i - b * tiles) * TILE;
        const Beam beam = beams[b];
        // a logit below this has a score below the bound: a few roundings of 64 bits and the conversion are within 2^-20 of the sizes
        const double at_least = (double)bound - beam.base + beam.lse;
        const float least = beam.shares ? INFINITY : (float)(at_least - 1e-6 * (fabs(at_least) + fabs((double)bound) + fabs(beam.base) + fabs(beam.lse)));
        if (tile.second < least || tile.second == -INFINITY) {         // usually: the tile's best is its only candidate
            if (lane == 0) cand[atomicAdd(&n_cand, 1)] = picked[chosen[t]];
            continue;
        }
        const float* const w = logits + (long long)(r * K + b) * ldl;
        float v[PER];
        load_tile<VEC>(v, w, lo, V, lane);
        uint32_t in = 0;
        #pragma unroll
        for (int e = 0; e < PER; e++) in |= !(v[e] < least) && v[e] > -INFINITY ? 1u << e : 0u;
        int most_of_tile = max(n, CANDS / p), count = __reduce_add_sync(0xffffffffu, __popc(in));
        if (__builtin_expect(count > most_of_tile, 0)) {                                    // few tiles, or one like no other: the n-th best of the lanes' two best each is a bound, too
            float top = -INFINITY, next = -INFINITY;
            #pragma unroll
            for (int e = 0; e < PER; e++) {
                const float x = in >> e & 1 ? v[e] : -INFINITY;
                next = fmaxf(next, fminf(x, top));
                top = fmaxf(top, x);
            }
            const float next_reversed = __shfl_sync(0xffffffffu, warp_sort(next, lane), 31 - lane);
            const float nth = __shfl_sync(0xffffffffu, warp_merge(warp_sort(top, lane), next_reversed, lane), n - 1);
            const float tight = (float)((double)nth - 1e-6 * (fabs((double)nth) + fabs(beam.base) + fabs(beam.lse)));      // (as above)
            #pragma unroll
            for (int e = 0; e < PER; e++) in &= v[e] < tight ? ~(1u << e) : ~0u;
            count = __reduce_add_sync(0xffffffffu, __popc(in));
            most_of_tile = max(n, PICKS * OUT / p);
        }
        int base = 0;
        if (lane == 0) base = atomicAdd(&n_cand, count <= most_of_tile ? count : n);
        base = __shfl_sync(0xffffffffu, base, 0);
        auto put = [&](int slot, int at) { cand[slot] = cand_of(beam, w[at], (uint32_t)b * (uint32_t)V + (uint32_t)at); };
        if (count <= most_of_tile) {
            int before = __popc(in);
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
            base += before - __popc(in);
            for (; in; in &= in - 1) put(base++, lo + place_in<VEC>(__ffs(in) - 1, lane));
        } else {
            // the n best in order, 32 logits after the other; by their scores: of large sums several logits give the same
            Cand list = none();
            #pragma unroll 1
            for (int e = 0; e < PER; e++) {
                if (!__any_sync(0xffffffffu, in >> e & 1)) continue;
                const int at = lo + place_in<VEC>(e, lane);
                const Cand me = in >> e & 1 ? cand_of(beam, w[at], (uint32_t)b * (uint32_t)V + (uint32_t)at) : none(), last = shfl(list, n - 1);
                if (!__any_sync(0xffffffffu, ahead(me, last))) continue;
                list = warp_merge(list, shfl(warp_sort(me, lane), 31 - lane), lane);
            }
            if (lane < n) cand[base + lane] = list;
        }
    }
    __syncthreads();
    const int c = n_cand;
    if (c > CANDS) {                                                   // by counting, 1,024 of them take 150 us
        Cand list = none();
        for (int i = warp * 32; i < c; i += MT) list = warp_merge(list, shfl(warp_sort(i + lane < c ? cand[i + lane] : none(), lane), 31 - lane), lane);
        __syncthreads();
        block_best(list, cand, warp, lane);
        if (tid < OUT) order[tid] = tid;
    } else for (int i = warp; i < c; i += MW) {                        // (what turned out to be no candidate stands behind all that are)
        const int rank = rank_of(cand, c, i, lane);
        if (lane == 0 && rank < n) order[rank] = i;
    }
    __syncthreads();
    if (tid < n) {
        const Cand me = order[tid] < 0 ? none() : cand[order[tid]];
        const bool is = me.s != 0ull;
        const int b = (int)(me.at / (uint32_t)V);
        const size_t to = (size_t)r * n + tid;
        out_s[to] = is ? (float)order_value(me.s) : -INFINITY;
        out_b[to] = is ? b : -1;
        out_v[to] = is ? (int)(me.at - (uint32_t)b * (uint32_t)V) : -1;
    }
}

}  // namespace

// scratch: 16 bytes for every 1,024 logits of a row, or part of them, on 16 bytes.  At most 16 beams, 32 results, 1,048,576 logits.
IK_EXPORT int ik_beam_select(const float* logits, long long ldl, const float* sums, int R, int K, int V, int n, void* scratch, long long scratch_bytes, float* out_s,
                             int* out_b, int* out_v, cudaStream_t stream) {
    const int tiles = (V + TILE - 1) / TILE;
    if (R <= 0 || K <= 0 || V <= 0 || n <= 0 || K > BEAMS || n > OUT || tiles > TILES || (long long)R * K > 0x3fffffff || scratch_bytes < (long long)R * K * tiles * 16 ||
        (ldl < V && R * K > 1) || ((uintptr_t)logits & 3) || ((uintptr_t)scratch & 15))
        return IK_BAD_ARGUMENT;
    Tile* const t = reinterpret_cast<Tile*>(scratch);
    const dim3 grid(R * K, (tiles + RT / 32 - 1) / (RT / 32));
    const bool vec = V % 4 == 0 && ldl % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    IK_RETURN_IF_ERROR(vec ? ik_launch(beam_tiles_kernel<true>, grid, RT, 0, stream, logits, ldl, sums, K, V, tiles, t)
                           : ik_launch(beam_tiles_kernel<false>, grid, RT, 0, stream, logits, ldl, sums, K, V, tiles, t));
    IK_RETURN_IF_ERROR(vec ? ik_launch_family(IK_FAMILY_ELEMENTWISE, beam_merge_kernel<true>, dim3(R), MT, 0, stream, logits, ldl, (const Tile*)t, sums, K, V, n, tiles, out_s, out_b, out_v)
                           : ik_launch_family(IK_FAMILY_ELEMENTWISE, beam_merge_kernel<false>, dim3(R), MT, 0, stream, logits, ldl, (const Tile*)t, sums, K, V, n, tiles, out_s, out_b, out_v));
    IK_LAUNCH_STATUS();
}
