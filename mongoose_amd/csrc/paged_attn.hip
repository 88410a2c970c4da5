// paged_attn.hip -- attention of each request's new tokens over its pages of the cache.
//
// For a token at position i and a query head h over KV head h / group:
//     s_j = scale * q . k_j;  with a cap s_j = cap * tanh(s_j / cap);  with slopes s_j -= slope_h * |i - j|
//     o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)   over the positions j that i sees (paged_sees), m their greatest s_j
// in one pass: a running maximum m, sum l and output O, the latter two multiplied by exp(m - m') where m grows to m'.  A token that
// sees nothing gets zeros.
//
// A query head's rows and the other heads' of its KV head go together: a tile is 16 or 128 rows (token, head), so that every K and V
// row is read once for all of them.  Scores are computed transposed, S^T = K Q^T, and the output O^T = V^T P^T: the MFMA result of the
// first (a lane: one query row, several positions) is the operand of the second as it stands, and a row's maximum and sum are
// a lane's own but for two exchanges.
#include <float.h>

#include "device_util.h"
#include "paged.h"

namespace mg {

constexpr int PT = 1024;                  // threads of the plan
constexpr int NARROW = 16, WIDE = 128;    // rows of a tile
constexpr int PLAN_LDS_TILES = 4096;      // tiles whose places on the line the plan holds in LDS
// Units a worker has at least where a tile's workers are its own: a narrow unit is as short as a share can be (one request of 500
// positions 8.8 us, with two 10.8); a wide share costs its 64 KB out and in (8B shape, one fresh prompt: 469 rows fp16 29 us, with one 38,
// with five 33; 409 rows fp32 52, with one 73, with two 70, with five 53).
constexpr int LEAST_NARROW = 1, LEAST_WIDE = 3;
constexpr int NARROW_WORKERS = 256;       // workgroups that narrow tiles have at most (a CU each)
constexpr int MERGE_LDS = 8192;           // floats of LDS for the weights of partial results
static_assert(NARROW_WORKERS * NARROW <= MERGE_LDS, "a narrow tile's shares are weighed in one turn");

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef unsigned uint16v_t __attribute__((ext_vector_type(16)));
typedef unsigned uint2_t __attribute__((ext_vector_type(2)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

// Positions of a unit: a narrow tile's four waves take 32 of an fp16 cache or 16 of an fp32 one each, a wide tile's share them.
MG_HD int narrow_keys(int kvHalf) { return kvHalf ? 128 : 64; }
MG_HD int wide_keys(int kvHalf) { return kvHalf ? 64 : 32; }

// Rows a KV head (tokens x group) up to which a request goes to the kernel that waits for memory, with longer ones to the one that waits for
// the matrix units.  8B shape:
//   A batch of up to 256 rows: all narrow, which reads K and V once for 16 rows, but in one launch.  One request of 8, 16, 32 and 64 tokens
//   over 16,000 positions: fp16 33, 41, 64, 112 us, wide 83, 89, 103, 105; fp32 43, 66, 117, 220, wide 338, 380, 401, 317.
//   Larger batches: narrow up to 16 rows.  24 requests of 5, 8, 12 tokens over 500 to 4,000 positions, fp16: 77, 78, 80 us wide, 75, 81, 99
//   narrow, and 96 requests of 5 tokens 208 wide, 304 narrow.  With an fp32 cache narrow tiles would be better there, up to 64 rows (228,
//   204, 385, and with 16 tokens 361 us wide; 169, 141, 249, 276 narrow): its wide tiles wait for the fp32 instructions of rows that are not there.
int paged_narrow_rows(const PagedGeo& g, int rows) {
    return (long long)rows * g.group <= 256 ? 256 : NARROW;
}
int paged_max_tiles(const PagedGeo& g) { return (int)((long long)g.maxRows * g.group / WIDE) + g.maxReqs + 256 / NARROW; }
size_t paged_part_floats(const PagedGeo& g) { return (size_t)((long long)g.maxRows * g.group <= NARROW ? NARROW : WIDE) * (g.headDim + 2); }
// Workgroups, in turns of the KV heads: two a CU for wide tiles; one a CU for narrow ones, though a CU holds two: HBM likes fewer
// streams (8B shape, fp16: 120,001 positions 98 us, with two 113; 48 requests 174 and 182).  Fewer where the batch
// cannot have that many units.
int paged_workers(const PagedGeo& g, int nReqs, int rows, bool wide) {
    const long long tiles = (long long)rows * g.group / NARROW + nReqs, units = tiles * (g.maxLen / 32 + 2);
    const int resident = NARROW_WORKERS * (wide ? 2 : 1);
    const long long most = resident / g.nKVHeads > 0 ? resident / g.nKVHeads : 1;
    return (int)(units < 1 ? 1 : units < most ? units : most);
}

// ---------------------------------------------------------------------------
// The plan (paged_rules.h): one workgroup, a thread a request, then a thread a tile, then a thread a worker.
// ---------------------------------------------------------------------------
// Inclusive sums over the workgroup; `carry` is what came before and becomes the total.
__device__ __forceinline__ unsigned plan_scan(unsigned v, unsigned& carry, unsigned* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = (unsigned)__shfl_up((int)v, d, 64);
        if (lane >= d) v = sat_add(v, o);
    }
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    unsigned before = carry, mine = 0;
    for (int w = 0; w < PT / 64; w++) {
        if (w == wave) mine = before;
        before = sat_add(before, part[w]);
    }
    carry = before;
    return sat_add(mine, v);
}
// A request as the plan takes it: rows inside the call's, a length inside the handle's.
__device__ __forceinline__ int4 plan_request(const PagedPlan& p, int r) {
    const int first = max(0, min(p.rowStart[r], p.rows)), last = max(first, min(p.rowStart[r + 1], p.rows));
    const int len = max(0, min(p.lens[r], p.maxLen));
    return make_int4(first, last - first, len, p.prefixLens ? max(0, min(p.prefixLens[r], len)) : 0);
}
__device__ __forceinline__ void put_tile(PagedTile* at, const PagedTile& t) {
    int4* d = reinterpret_cast<int4*>(at);
    d[0] = make_int4(t.req, t.row0, t.rows, t.len);
    d[1] = make_int4(t.prefix, t.first, t.cost0, t.unit0);
    d[2] = make_int4(t.units, t.worker0, t.worker1, t.index);
    d[3] = make_int4(t.tileRows, t.unitKeys, 0, 0);
}
// Largest i with sums[i] <= x, of n sums
__device__ __forceinline__ int plan_find(const unsigned* sums, int n, unsigned x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}
// One workgroup for the narrow tiles and one for the wide ones
__global__ __launch_bounds__(PT) void paged_plan_kernel(PagedPlan p) {
    const bool wide = blockIdx.x != 0;
    const int tileRows = wide ? WIDE : NARROW, unitKeys = wide ? wide_keys(p.kvHalf) : narrow_keys(p.kvHalf);
    p.tiles += wide ? p.maxTiles : 0;
    p.workers += wide ? p.maxWorkers : 0;
    p.nWorkers = wide ? p.wideWorkers : p.nWorkers;
    if (threadIdx.x == 0 && !wide) *p.made = {p.nReqs, p.rows, p.window, 0};
    __shared__ unsigned tile0[PAGED_MAX_REQS + 1], place[PLAN_LDS_TILES], part[PT / 64];
    __shared__ int4 held[PT];
    const int tid = threadIdx.x;
    unsigned sum = 0;
    if (tid == 0) tile0[0] = 0;
    for (int r0 = 0; r0 < p.nReqs; r0 += PT) {
        const int r = r0 + tid;
        unsigned n = 0;
        if (r < p.nReqs) {
            const int4 rq = plan_request(p, r);
            const long long rows = (long long)rq.y * p.group;
            if (wide == (rows > p.narrowRows)) n = (unsigned)((rows + tileRows - 1) / tileRows);
            if (r < PT) held[r] = rq;
        }
        n = plan_scan(n, sum, part);
        if (r < p.nReqs) tile0[r + 1] = n;
    }
    __syncthreads();
    const int nTiles = (int)min(sum, (unsigned)p.maxTiles);          // (more only where the caller's rows overlap)
    PagedTile t;
    unsigned cost = 0;
    auto make = [&](int i) {
        const int r = plan_find(tile0, p.nReqs, (unsigned)i);
        const int4 rq = r < PT ? held[r] : plan_request(p, r);
        t.req = r; t.row0 = rq.x; t.rows = rq.y; t.len = rq.z; t.prefix = rq.w;
        t.tileRows = tileRows; t.unitKeys = unitKeys;
        t.first = (i - (int)tile0[r]) * tileRows;
        t.index = i;
        paged_units(t, p.window, p.group);
    };
    for (int i0 = 0; i0 < nTiles; i0 += PT) {
        const int i = i0 + tid;
        unsigned c = 0;
        if (i < nTiles) { make(i); c = (unsigned)paged_cost(t); }
        const unsigned end = plan_scan(c, cost, part);
        if (i < nTiles) {
            t.cost0 = (int)(end - c);
            if (i < PLAN_LDS_TILES) place[i] = end - c;
            else p.tiles[i].cost0 = t.cost0;
        }
    }
    __syncthreads();
    const bool few = paged_few(nTiles, p.nWorkers);                  // (512 tiles at most: one round)
    int workers = max(1, min(p.nWorkers, (int)cost)), n = 0;
    if (few) {
        if (tid < nTiles) n = paged_workers_for(t, (int)cost, nTiles, p.nWorkers, wide ? LEAST_WIDE : LEAST_NARROW);
        unsigned all = 0;
        const unsigned end = plan_scan((unsigned)n, all, part);
        workers = (int)all;
        if (tid < nTiles) {
            t.worker0 = (int)end - n;
            t.worker1 = (int)end - 1;
            tile0[tid] = end - n;                                    // (its first use is over: plan_scan has synchronised)
            put_tile(p.tiles + tid, t);
        }
    } else {
        for (int i = tid; i < nTiles; i += PT) {
            const int cost0 = i < PLAN_LDS_TILES ? (int)place[i] : p.tiles[i].cost0;
            if (nTiles > PT) make(i);                                // (else it is still at hand)
            t.cost0 = cost0;
            const int x = cost0 + PAGED_TILE_COST;
            t.worker0 = t.units ? paged_worker_of((int)cost, workers, x) : 0;
            t.worker1 = t.units ? paged_worker_of((int)cost, workers, x + t.units - 1) : 0;
            put_tile(p.tiles + i, t);
        }
    }
    __syncthreads();
    for (int w = tid; w < p.nWorkers; w += PT) {
        int4* d = reinterpret_cast<int4*>(p.workers + w);
        int4 range = make_int4(0, 0, 0, 0);
        if (w < workers && nTiles > 0) {
            int i, a, b;
            if (few) {
                i = plan_find(tile0, nTiles, (unsigned)w);
            } else {
                a = paged_share((int)cost, workers, w);
                b = paged_share((int)cost, workers, w + 1);
                int lo = 0, hi = nTiles;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if ((mid < PLAN_LDS_TILES ? (int)place[mid] : p.tiles[mid].cost0) <= a) lo = mid; else hi = mid;
                }
                i = lo;
            }
            const int4* from = reinterpret_cast<const int4*>(p.tiles + i);
            const int4 x0 = from[0], x1 = from[1], x2 = from[2], x3 = from[3];
            d[0] = x0; d[1] = x1; d[2] = x2; d[3] = x3;
            if (few) {
                PagedTile s;
                s.cost0 = x1.z; s.units = x2.x;
                const int parts = x2.z - x2.y + 1, k = w - x2.y;
                a = paged_part(s, parts, k);
                b = k + 1 < parts ? paged_part(s, parts, k + 1) : s.cost0 + paged_cost(s);
            }
            range = make_int4(a, b, nTiles, 0);
        }
        d[4] = range;
    }
}
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(p.wideWorkers > 0 ? 2 : 1), dim3(PT), 0, s, p);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// cap * tanh(s / cap).  Near zero the odd Taylor polynomial up to x^13, s + s x^2 P(x^2) with x = s / cap: where |x| < 0.45 the next
// term is below 2^-26 of the result.  Beyond, (1 - e^-2x) / (1 + e^-2x).
constexpr float CAP_NEAR = 0.45f;
__device__ __forceinline__ float capped_near(float s, float x2) {
    float t = fmaf(x2, 21844.f / 6081075.f, -1382.f / 155925.f);
    t = fmaf(x2, t, 62.f / 2835.f);
    t = fmaf(x2, t, -17.f / 315.f);
    t = fmaf(x2, t, 2.f / 15.f);
    t = fmaf(x2, t, -1.f / 3.f);
    return fmaf(x2 * t, s, s);
}
__device__ __forceinline__ float capped(float s, float cap, float invCap) {
    const float x = s * invCap, a = fabsf(x);
    const float e = __builtin_amdgcn_exp2f(a * -2.885390081777927f);
    const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
    return a < CAP_NEAR ? capped_near(s, x * x) : cap * far;
}
// The cap on all the scores of a lane: without the far form where no lane of the wave needs it (8B shape, four requests of 345 to
// 467 rows over a window of 1,024, cap 50: 131 us, without this 139)
template <typename T, int N>
__device__ __forceinline__ void cap_all(T (&s)[N], float cap, float invCap) {
    constexpr int M = sizeof(T) / 4;
    auto at = [&](int i) -> float { if constexpr (M == 1) return s[i]; else return s[i / M][i % M]; };
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N * M; i++) most = fmaxf(most, fabsf(at(i)));
    auto all = [&](auto f) {
#pragma unroll
        for (int i = 0; i < N * M; i++) {
            if (i % 8 == 0) __builtin_amdgcn_sched_barrier(0);       // (eight at once: for more there are no registers)
            if constexpr (M == 1) s[i] = f(at(i)); else s[i / M][i % M] = f(at(i));
        }
    };
    if (!__any(!(most * invCap < CAP_NEAR))) all([&](float y) { const float x = y * invCap; return capped_near(y, x * x); });
    else all([&](float y) { return capped(y, cap, invCap); });
}
// 16 bytes through to memory, for a workgroup of another die to read within the launch
__device__ __forceinline__ void store_through(float* p, float4_t v) {
    const uint4_t w = __builtin_bit_cast(uint4_t, v);
    unsigned long long* d = reinterpret_cast<unsigned long long*>(p);
    __hip_atomic_store(d, w[0] | (unsigned long long)w[1] << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(d + 1, w[2] | (unsigned long long)w[3] << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Opens a load into LDS (as MG_SET_M0), with the five wait states that an address from a vector instruction's scalar result needs:
// the compiler keeps no distances to what is inside a string.
#define PAGED_SET_M0 "s_mov_b32 m0, %0\n\ts_nop 4\n\t"
template <int J>
__device__ __forceinline__ int quad_lane(int v) { return dpp_i<J * 0x55>(v); }      // lane J of the quad

// A tile's fields, the same in every lane, in scalar registers
__device__ __forceinline__ PagedTile tile_at(const PagedTile* from) {
    PagedTile t = *from;
    int* x = &t.req;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(PagedTile) / 4); i++) x[i] = __builtin_amdgcn_readfirstlane(x[i]);
    return t;
}
// A value to be worked with anew where it is asked for: what is made of it (addresses, masks) is not worth registers across a loop
__device__ __forceinline__ int anew(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int thread_anew() { return anew(threadIdx.x); }
// What a tile's code needs of its row, on the lane's behalf
struct PagedRow { int token, head, pos; };
__device__ __forceinline__ PagedRow paged_row(const PagedTile& t, int group, int kvh, int row) {
    const int rr = min(t.first + row, t.rows * group - 1), token = rr / group;
    return {token, kvh * group + rr - token * group, t.len - t.rows + token};
}

// Where a position's row of K or V starts (in bytes from the pool), through its page; `zeros` for a position that is out of [begin, end) or gone
__device__ __forceinline__ const char* kv_row(const char* pool, const char* zeros, size_t rowBytes, int key, int page, int begin, int end, int shift) {
    const bool held = (key >= begin) & (key < end) & (page >= 0);          // (no branches: a step has ten of these)
    const unsigned at = held ? ((unsigned)page << shift) + ((unsigned)key & ((1u << shift) - 1)) : 0u;
    return (held ? pool : zeros) + (size_t)at * rowBytes;
}

// Where a worker leaves its share of a tile's result: rows of headDim floats, then the rows' maxima and sums.
__device__ __forceinline__ float* part_of(const PagedAttention& p, const PagedTile& t, int kvh, int w) {
    return p.parts + (((size_t)kvh * p.nWorkers + w) * 2 + (w == t.worker0)) * p.partStride;
}
// After a worker has stored its share (through to memory): whether it is the last one of the tile's to come here.  scratch: LDS
// that nobody reads any more.
__device__ __forceinline__ bool last_to_finish(const PagedAttention& p, const PagedTile& t, int kvh, float* scratch) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned* count = p.arrived + (size_t)kvh * p.maxTiles + t.index;
    unsigned* before = reinterpret_cast<unsigned*>(scratch);
    if (threadIdx.x == 0) *before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool last = *before == (unsigned)(t.worker1 - t.worker0);
    __syncthreads();
    if (!last) return false;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}
// The weights of shares s0 .. s0 + n - 1 in each row's result, wt[s][ROWS], and the rows' sums with them, den[ROWS]; the rows' greatest
// maxima, M[ROWS], where s0 is 0.  Ends with the LDS written.
template <int HD, int ROWS>
__device__ __forceinline__ void merge_weights(const PagedAttention& p, const PagedTile& t, int kvh, int R, int s0, int n, float* M, float* den, float* wt) {
    const int tid = thread_anew(), segs = t.worker1 - t.worker0 + 1;
    auto at = [&](int s, int i) { return part_of(p, t, kvh, t.worker0 + s)[ROWS * HD + i]; };
    if (s0 == 0 && tid < R) {
        float m = -INFINITY;
#pragma unroll 8
        for (int s = 0; s < segs; s++) m = fmaxf(m, at(s, tid));
        M[tid] = m == -INFINITY ? 0.f : m;
        den[tid] = 0.f;
    }
    __syncthreads();                      // (and the weights before these are used up)
    for (int i = tid; i < n * ROWS; i += WG)
        if (i % ROWS < R) wt[i] = __builtin_amdgcn_exp2f(at(s0 + i / ROWS, i % ROWS) - M[i % ROWS]);
    __syncthreads();
    if (tid < R) {
        float d = den[tid];
#pragma unroll 8
        for (int s = 0; s < n; s++) d = fmaf(wt[s * ROWS + tid], at(s0 + s, ROWS + tid), d);
        den[tid] = d;
    }
}
__device__ __forceinline__ float4_t over(float4_t v, float l) { return l == 0.f ? v : v / l; }       // (nothing seen: zeros)

// Values that are no numbers.  Zero times one is no zero, so that one reaches rows that do not see it, and its product with the second
// term of a weight turns an infinity into a NaN.  A tile whose result has elements that are no numbers therefore goes through its
// units three times more, with the maxima of the first time: with ones for +infinity and NaN, zeros for all else, and weights of 1 (or 0
// where they are 0); the same for -infinity and NaN; with zeros for all three.  An element is what the last time gives, plus an
// infinity where the first count is not 0, minus one where the second is not.  Other tiles pay for a look at their result.
enum { PLUS_INFINITE, MINUS_INFINITE, FINITE };
// What stands for the values of a word in a pass
template <bool HALF>
__device__ __forceinline__ unsigned stand_in(unsigned v, int pass) {
    constexpr int BITS = HALF ? 16 : 32;
    constexpr unsigned sign = 1u << (BITS - 1), inf = HALF ? 0x7c00u : 0x7f800000u, one = HALF ? 0x3c00u : 0x3f800000u;
    unsigned out = 0;
#pragma unroll
    for (int at = 0; at < 32; at += BITS) {
        const unsigned x = HALF ? (v >> at) & 0xffffu : v, size = x & (sign - 1);
        const bool counts = size > inf || x == (pass == MINUS_INFINITE ? sign | inf : inf);
        out |= (pass == FINITE ? (size < inf ? x : 0u) : counts ? one : 0u) << at;
    }
    return out;
}
__device__ __forceinline__ float with_infinities(float o, bool plus, bool minus) { return (plus ? o + INFINITY : o) + (minus ? -INFINITY : 0.f); }

// The power of two that a row of q, |q| up to `top`, is scaled by: to 2^14 .. 2^15, or to less where the factor left for its scores would
// fall below 2^-119 and no longer be a normal number (such scores are below 2^-80).
__device__ __forceinline__ int power_up(float top, float scale) {
    return top > 0.f && top < INFINITY ? min(15 - __builtin_amdgcn_frexp_expf(top), 118 + __builtin_amdgcn_frexp_expf(scale)) : 0;
}

// A tile of 16 rows: four waves take a step of KB positions each of every unit, each with its own running maximum, sum and output.
// Bound by HBM: a lane loads its K and V operands from the pages straight into registers, each where the last step's have gone into
// their products, the page numbers two steps ahead; nothing is shared between the waves before the end.  8B shape, fp16, 48 requests
// of 100 to 8,000 positions: 168 us, 5.5 TB/s.
//   K (A operand of S^T): lane l = position l%16, 16 bytes a step of the head dimension.
//   V (A operand of O^T): lane l holds, of four consecutive positions 4(l/16).. a block of 16, the elements l%16 * HD/16 .. of their
//     rows -- whole rows side by side -- and turns them in registers: block e of the output is dimensions l%16 * HD/16 + e.
// fp16 caches: q, scaled by a power of two to 2^14 .. 2^15, and the probabilities, times 2^14, each as two fp16 terms (22 bits;
// what is below 2^-29 of the row's largest |q| or 2^-38 of the largest probability is lost); K and V as they are.
// fp32 caches: fp32 matrix instructions throughout.
template <typename KVT, int HD, bool MOD>
struct NarrowTile {
    static constexpr bool HALF = sizeof(KVT) == 2;
    static constexpr int KB = HALF ? 32 : 16;              // positions of a wave's step
    static constexpr int NB = KB / 16, UK = 4 * KB, EPL = HD / 16;
    static constexpr int KV4 = HALF ? HD / 32 : HD / 16;   // 16-byte pieces a lane holds of a block's K rows
    static constexpr int VW = HALF ? EPL / 2 : EPL;        // words a lane holds of a V row
    static constexpr float SHIFT = HALF ? 14.f : 0.f;      // probabilities are held times 2^SHIFT

    const PagedAttention& p;
    const PagedTile& t;
    int lane, l16, g, wave;
    PagedSpan span;
    PagedRow row;
    const int* pages;
    const char *Kp, *Vp, *zeros;
    size_t rowBytes;
    float c, cap, invCap, slope;
    half8_t qh[HALF ? HD / 32 : 1], ql[HALF ? HD / 32 : 1];
    float4_t qf[HALF ? 1 : HD / 16];
    uint4_t k[NB][KV4];            // the step's K and V, then the next one's
    unsigned v[NB * 4][VW];
    float m, l;
    float4_t o[EPL];

    int here, next;                // page numbers of the step at hand and of the one behind it

    __device__ __forceinline__ NarrowTile(const PagedAttention& p_, const PagedTile& t_, int kvh, int u0, int u1) : p(p_), t(t_) {
        const int tid = thread_anew();
        lane = tid & 63; l16 = lane & 15; g = lane >> 4;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        span = paged_span(t.rows, t.len, t.prefix, p.window, p.g.group, t.first, NARROW);
        row = paged_row(t, p.g.group, kvh, l16);
        pages = p.table + (size_t)t.req * p.g.width;
        rowBytes = (size_t)p.g.kvDim * sizeof(KVT);
        Kp = static_cast<const char*>(p.K) + (size_t)kvh * HD * sizeof(KVT);
        Vp = static_cast<const char*>(p.V) + (size_t)kvh * HD * sizeof(KVT);
        zeros = reinterpret_cast<const char*>(p.zeros);
        here = page_of(u0);
        const float* q = p.q + (size_t)(t.row0 + row.token) * p.ldq + (size_t)row.head * HD;
        float4_t x[HD / 16];                      // the row's elements as the operands want them
#pragma unroll
        for (int i = 0; i < HD / 16; i++) x[i] = *reinterpret_cast<const float4_t*>(q + (HALF ? i / 2 * 32 + g * 8 + i % 2 * 4 : i * 16 + g * 4));
        next = page_of(min(u0 + 1, u1 - 1));
        load_k(u0, here);
        load_v(u0, here);
        cap = p.softcap;
        invCap = MOD && cap > 0.f ? 1.f / cap : 0.f;
        slope = MOD && p.slopes ? p.slopes[row.head] : 0.f;
        c = p.scale;
        if constexpr (HALF) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 16; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) top = fmaxf(top, fabsf(x[i][j]));
            top = rows_max(top);
            const int up = power_up(top, c);
#pragma unroll
            for (int s = 0; s < HD / 32; s++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = ldexpf(x[2 * s + j / 4][j % 4], up);
                    qh[s][j] = (_Float16)y;
                    ql[s][j] = (_Float16)(y - (float)qh[s][j]);
                }
            c = ldexpf(c, -up);
        } else {
#pragma unroll
            for (int s = 0; s < HD / 16; s++) qf[s] = x[s];
        }
        if (!MOD) c *= 1.4426950408889634f;
        c = fminf(c, FLT_MAX);                    // (0 times it is 0)
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; e++) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    __device__ __forceinline__ int base_of(int u) const { return (t.unit0 + u) * UK + wave * KB; }
    // The page of the step's run lane % (KB / 8) of eight positions, -1 where there is none
    __device__ __forceinline__ int page_of(int u) const {
        const int key = min(base_of(u) + (lane & (KB / 8 - 1)) * 8, span.end - 1);
        const int page = pages[max(key, 0) >> p.g.pageShift];
        return page >= 0 && page < p.g.nPages ? page : -1;
    }
    // The page of the positions 16 b .. 16 b + 15 that the lane has to do with: of its upper eight or its lower
    __device__ __forceinline__ int page_in(int mine, int b, bool upper) const {
        const int lo = HALF && b ? quad_lane<2>(mine) : quad_lane<0>(mine), hi = HALF && b ? quad_lane<3>(mine) : quad_lane<1>(mine);
        return upper ? hi : lo;                       // (all lanes take part in both exchanges)
    }
    __device__ __forceinline__ void load_k(int u, int mine) {
        const int base = base_of(u);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const char* at = kv_row(Kp, zeros, rowBytes, base + 16 * b + l16, page_in(mine, b, l16 & 8), span.begin, span.end, p.g.pageShift) + g * 16;
#pragma unroll
            for (int i = 0; i < KV4; i++) k[b][i] = *reinterpret_cast<const uint4_t*>(at + i * 64);
        }
    }
    __device__ __forceinline__ void load_v(int u, int mine) {
        const int base = base_of(u);
#pragma unroll
        for (int j = 0; j < NB * 4; j++) {
            const int page = page_in(mine, j / 4, g & 2);
            const char* at = kv_row(Vp, zeros, rowBytes, base + 16 * (j / 4) + 4 * g + j % 4, page, span.begin, span.end, p.g.pageShift) + l16 * (VW * 4);
            if constexpr (VW == 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(at);
                v[j][0] = x.x; v[j][1] = x.y;
            } else {
#pragma unroll
                for (int e = 0; e < VW; e += 4) {
                    const uint4_t x = *reinterpret_cast<const uint4_t*>(at + e * 4);
#pragma unroll
                    for (int i = 0; i < 4; i++) v[j][e + i] = x[i];
                }
            }
        }
    }
    struct Weights { half8_t hi, lo; float x[NB * 4]; };
    static __device__ __forceinline__ Weights weights(const float (&x)[NB * 4]) {
        Weights w;
        if constexpr (HALF) {
#pragma unroll
            for (int j = 0; j < 8; j++) { w.hi[j] = (_Float16)x[j]; w.lo[j] = (_Float16)(x[j] - (float)w.hi[j]); }
        } else {
#pragma unroll
            for (int j = 0; j < NB * 4; j++) w.x[j] = x[j];
        }
        return w;
    }
    // Block e of V^T P^T on top of `out`
    __device__ __forceinline__ float4_t product(int e, const Weights& w, float4_t out) const {
        if constexpr (HALF) {
            uint4_t a;
#pragma unroll
            for (int j = 0; j < 4; j++) a[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
            out = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), w.hi, out, 0, 0, 0);
            out = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), w.lo, out, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const unsigned x = v[i][e];
                out = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), w.x[i], out, 0, 0, 0);
            }
        }
        return out;
    }
    // Step u, on page numbers `mine`; loads the K rows of the one behind it (if any, on page numbers `next`) where it is done with its own
    template <bool AGAIN>
    __device__ __forceinline__ void compute(int u, int mine, bool more, int next, int pass) {
        const int base = base_of(u);
        float4_t S[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            S[b] = float4_t{0.f, 0.f, 0.f, 0.f};
            if constexpr (HALF) {
#pragma unroll
                for (int i = 0; i < KV4; i++) {
                    S[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, k[b][i]), qh[i], S[b], 0, 0, 0);
                    S[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, k[b][i]), ql[i], S[b], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < KV4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) S[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float4_t, k[b][i])[j], qf[i][j], S[b], 0, 0, 0);
            }
        }
        if constexpr (HALF) {
            // Infinite keys: the second term's product with one may be an infinity of the other sign, or zero times it; the first
            // term's alone is what the formula gives.
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NB * 4; j++) sum += S[j / 4][j % 4];
            if (__any(sum != sum)) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float4_t first{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < KV4; i++) first = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, k[b][i]), qh[i], first, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; j++) S[b][j] = S[b][j] != S[b][j] ? first[j] : S[b][j];
                }
            }
        }
        if (more) load_k(u + 1, next);
        // scores in powers of two; the lane's positions are base + 16 b + 4 g + i
        float x[NB * 4];
#pragma unroll
        for (int j = 0; j < NB * 4; j++) x[j] = S[j / 4][j % 4] * c;
        if constexpr (MOD) {
            if (cap > 0.f) cap_all(x, cap, invCap);
#pragma unroll
            for (int j = 0; j < NB * 4; j++) x[j] = (x[j] - slope * (float)abs(row.pos - (base + 16 * (j / 4) + 4 * g + j % 4))) * 1.4426950408889634f;
        }
        const bool inner = base + KB <= t.prefix || (base + KB - 1 <= span.pos0 && (p.window == 0 || base > span.pos1 - p.window));       // all rows see all of it
        const bool all = inner && __all(mine >= 0);
        if (!all) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const bool held = page_in(mine, b, g & 2) >= 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (!held || !paged_sees(row.pos, base + 16 * b + 4 * g + i, t.len, p.window, t.prefix)) x[4 * b + i] = -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < NB * 4; j++) top = fmaxf(top, x[j]);
        top = fmaxf(m, rows_max(top));
        const float from = top == -INFINITY ? 0.f : top;          // (a score that is a NaN stays one)
        if (__any(top > m)) {
            const float f = __builtin_amdgcn_exp2f(m - from);
            l *= f;
#pragma unroll
            for (int e = 0; e < EPL; e++) o[e] *= f;
            m = top;
        }
#pragma unroll
        for (int j = 0; j < NB * 4; j++) {
            x[j] = __builtin_amdgcn_exp2f(x[j] - from + SHIFT);
            l += x[j];
        }
        if (!inner) {
            bool some = false;
#pragma unroll
            for (int j = 0; j < NB * 4; j++) some |= x[j] != 0.f;
            if (!__any(some)) return;                     // (no row has anything here)
        }
        if constexpr (AGAIN) {
#pragma unroll
            for (int j = 0; j < NB * 4; j++) {
                x[j] = pass == FINITE ? x[j] : x[j] > 0.f ? 1.f : 0.f;
#pragma unroll
                for (int e = 0; e < VW; e++) v[j][e] = stand_in<HALF>(v[j][e], pass);
            }
        }
        const Weights wt = weights(x);
#pragma unroll
        for (int e = 0; e < EPL; e++) o[e] = product(e, wt, o[e]);
    }
    template <bool AGAIN>
    __device__ __forceinline__ void units(int u0, int u1, int pass) {
        for (int u = u0; u < u1; u++) {
            const int behind = page_of(min(u + 2, u1 - 1));
            const bool more = u + 1 < u1;
            compute<AGAIN>(u, here, more, next, pass);
            if (more) load_v(u + 1, next);
            here = next;
            next = behind;
        }
    }
    __device__ __forceinline__ void run(int u0, int u1, int kvh, int, float* lds) {
        units<false>(u0, u1, 0);
        float odd = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) odd = fmaf(o[e][i], 0.f, odd);
        if (__any(odd != odd)) {
            unsigned plus = 0, minus = 0;         // a bit an element
#pragma unroll 1
            for (int pass = PLUS_INFINITE; pass <= FINITE; pass++) {
                here = page_of(u0);
                next = page_of(min(u0 + 1, u1 - 1));
                load_k(u0, here);
                load_v(u0, here);
                l = 0.f;
#pragma unroll
                for (int e = 0; e < EPL; e++) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
                units<true>(u0, u1, pass);
                unsigned counts = 0;
#pragma unroll
                for (int e = 0; e < EPL; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) counts |= (o[e][i] > 0.f ? 1u : 0u) << (4 * e + i);
                if (pass == PLUS_INFINITE) plus = counts;
                if (pass == MINUS_INFINITE) minus = counts;
            }
#pragma unroll
            for (int e = 0; e < EPL; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[e][i] = with_infinities(o[e][i], plus >> (4 * e + i) & 1, minus >> (4 * e + i) & 1);
        }
        join(kvh, lds);
    }
    // The four waves' results as one, at lds (rows of HD + 4 floats) with maxima and sums behind
    static constexpr int FLOATS = 4 * NARROW * (HD + 4) + 8 * NARROW;
    __device__ __forceinline__ void join(int kvh, float* lds) {
        float* wm = lds + 4 * NARROW * (HD + 4);
        float* wl = wm + 4 * NARROW;
        l = rows_sum(l);
        __syncthreads();                          // (the tile before has been written out)
        float* mine = lds + (wave * NARROW + l16) * (HD + 4) + 4 * g * EPL;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < EPL; e += 4) *reinterpret_cast<float4_t*>(mine + i * EPL + e) = float4_t{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
        if (g == 0) { wm[wave * NARROW + l16] = m; wl[wave * NARROW + l16] = l; }
        __syncthreads();
        const int tid = thread_anew();
#pragma unroll
        for (int n = 0; n < NARROW * (HD / 4) / WG; n++) {
            const int i = tid + n * WG, r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            const float M = fmaxf(fmaxf(wm[r], wm[NARROW + r]), fmaxf(wm[2 * NARROW + r], wm[3 * NARROW + r])), from = M == -INFINITY ? 0.f : M;
            float4_t a{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) a += *reinterpret_cast<const float4_t*>(lds + (w * NARROW + r) * (HD + 4) + d) * __builtin_amdgcn_exp2f(wm[w * NARROW + r] - from);
            *reinterpret_cast<float4_t*>(lds + r * (HD + 4) + d) = a;
        }
        float M = 0.f, L = 0.f;
        if (tid < NARROW) {
            M = fmaxf(fmaxf(wm[tid], wm[NARROW + tid]), fmaxf(wm[2 * NARROW + tid], wm[3 * NARROW + tid]));
            const float from = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < 4; w++) L = fmaf(wl[w * NARROW + tid], __builtin_amdgcn_exp2f(wm[w * NARROW + tid] - from), L);
        }
        __syncthreads();
        if (tid < NARROW) { wm[tid] = M; wl[tid] = L; }
        __syncthreads();
    }
    __device__ __forceinline__ void write(int kvh, int w, float* lds) const {
        const float* ms = lds + 4 * NARROW * (HD + 4);
        const float* ls = ms + 4 * NARROW;
        const int tid = thread_anew(), R = min(NARROW, t.rows * p.g.group - t.first);
        const bool whole = t.worker0 == t.worker1;
        float* mine = part_of(p, t, kvh, w);
        for (int i = tid; i < R * (HD / 4); i += WG) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            const float4_t v = *reinterpret_cast<const float4_t*>(lds + r * (HD + 4) + d);
            if (!whole) { store_through(mine + r * HD + d, v); continue; }
            const PagedRow at = paged_row(t, p.g.group, kvh, r);
            *reinterpret_cast<float4_t*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + d) = over(v, ls[r]);
        }
        if (whole) return;
        if (tid < R) { st_agent(mine + NARROW * HD + tid, ms[tid]); st_agent(mine + NARROW * HD + NARROW + tid, ls[tid]); }
        if (last_to_finish(p, t, kvh, lds)) merge(kvh, R, lds);
    }
    // All workers' shares: threads take rows and columns and, where there are fewer of those than threads, shares in turn
    __device__ __forceinline__ void merge(int kvh, int R, float* lds) const {
        float *M = lds, *den = lds + NARROW, *wt = lds + 2 * NARROW;
        constexpr int N = NARROW * HD / 4 / WG > 0 ? NARROW * HD / 4 / WG : 1;
        const int tid = thread_anew(), segs = t.worker1 - t.worker0 + 1, cols = R * (HD / 4), par = max(1, WG / cols);
        float4_t acc[N];
#pragma unroll
        for (int k = 0; k < N; k++) acc[k] = float4_t{0.f, 0.f, 0.f, 0.f};
        merge_weights<HD, NARROW>(p, t, kvh, R, 0, segs, M, den, wt);
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = par > 1 ? tid % cols : tid + k * WG, from = par > 1 ? tid / cols : 0;
            if (i >= cols || from >= par || (par > 1 && k > 0)) continue;
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
#pragma unroll 4
            for (int s = from; s < segs; s += par)
                acc[k] += wt[s * NARROW + r] * *reinterpret_cast<const float4_t*>(part_of(p, t, kvh, t.worker0 + s) + r * HD + d);
        }
        __syncthreads();
        if (par > 1) {                        // the shares of the same columns, in their order
            float4_t* x = reinterpret_cast<float4_t*>(wt);
            if (tid / cols < par) x[tid] = acc[0];
            __syncthreads();
            if (tid < cols)
                for (int k = 1; k < par; k++) acc[0] += x[tid + k * cols];
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = tid + k * WG;
            if (i >= cols) continue;
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            const PagedRow at = paged_row(t, p.g.group, kvh, r);
            *reinterpret_cast<float4_t*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + d) = over(acc[k], den[r]);
        }
    }
};

// A tile of 128 rows: a wave takes 32 of them over all the positions, which go through LDS (two buffers, filled by loads that run a
// unit ahead), so that a K or V row is fetched once for 128 rows.  8B shape, fp16, 2,048 tokens over 16,384 positions: 1,015 us, 1,015
// TFLOP/s with both terms counted.  Bound by the matrix units: 32x32 instructions, two terms a product
// with an fp16 cache (as in NarrowTile), four K = 2 fp32 instructions a 16-byte piece with an fp32 one.
//   K (A operand): lane l = position l%32, 16 bytes at dimensions 16 s + 8 (l/32) (fp16) or 8 s + 4 (l/32) (fp32).
//   V (A operand): dimension l%32 of a block of 32, the positions of the lane's own probabilities -- 4 (l/32) + 0..3 of every eight --
//     fp16 through the transposing LDS read, fp32 word by word.
// A row's 16-byte pieces lie in LDS at piece ^ swz(row), so that neither rows of one piece nor (fp16) four rows of two meet in a bank.
template <typename KVT, int HD, bool MOD>
struct WideTile {
    static constexpr bool HALF = sizeof(KVT) == 2;
    static constexpr int UK = HALF ? 64 : 32, NB = UK / 32, DB = HD / 32;
    static constexpr int ROWB = HD * (int)sizeof(KVT), PR = ROWB / 16;      // bytes and 16-byte pieces of a row
    static constexpr int RI = 64 / PR, NI = UK / RI / 4;                    // rows a load instruction brings, instructions a wave
    static constexpr int TILEB = UK * ROWB, BUFB = 2 * TILEB;               // K, then V
    static constexpr int VOTES = 2 * BUFB / 4;                              // a word of each wave's, behind the buffers
    static constexpr int QS = HALF ? HD / 16 : HD / 8;
    static constexpr float SHIFT = HALF ? 13.f : 0.f;      // probabilities times 2^SHIFT,
    static constexpr float LAZY = HALF ? 2.f : 8.f;        // and up to 2^LAZY more: the maximum is only moved where it grows by more

    const PagedAttention& p;
    const PagedTile& t;
    int lane, n32, hf, wave;
    PagedSpan span;           // the tile's
    int pos0, pos1, begin, end;      // the wave's own rows'
    bool active;
    PagedRow row;
    const int* pages;
    const char *Kp, *Vp, *zeros;
    size_t rowBytes;
    static constexpr unsigned ldsBase = 0;
    unsigned from[NI];      // the lane's offset of every load instruction from its run of eight positions
    float c, cap, invCap, slope;
    half8_t qh[HALF ? QS : 1], ql[HALF ? QS : 1];
    float4_t qf[HALF ? 1 : QS];
    float m, l;
    float16_t o[DB];

    static __device__ __forceinline__ int swz(int r) { return HALF ? ((r & 3) << 1) | ((r >> 2) & 1) : r & 7; }

    int here, next;                  // page numbers of the unit at hand and of the one behind it

    __device__ __forceinline__ WideTile(const PagedAttention& p_, const PagedTile& t_, int kvh, int u0, int u1) : p(p_), t(t_) {
        const int tid = thread_anew();
        lane = tid & 63; n32 = lane & 31; hf = lane >> 5;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        span = paged_span(t.rows, t.len, t.prefix, p.window, p.g.group, t.first, WIDE);
        const int mine = t.first + 32 * wave;
        active = mine < t.rows * p.g.group;
        const PagedSpan own = paged_span(t.rows, t.len, t.prefix, p.window, p.g.group, active ? mine : t.first, 32);
        pos0 = own.pos0; pos1 = own.pos1; begin = own.begin; end = own.end;
        row = paged_row(t, p.g.group, kvh, 32 * wave + n32);
        pages = p.table + (size_t)t.req * p.g.width;
        rowBytes = (size_t)p.g.kvDim * sizeof(KVT);
        Kp = static_cast<const char*>(p.K) + (size_t)kvh * ROWB;
        Vp = static_cast<const char*>(p.V) + (size_t)kvh * ROWB;
        zeros = reinterpret_cast<const char*>(p.zeros);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = (wave * NI + i) * RI + lane / PR;
            from[i] = (unsigned)(r & 7) * (unsigned)rowBytes + (unsigned)((lane % PR) ^ swz(r)) * 16;
        }
        here = page_of(u0);
        const float* q = p.q + (size_t)(t.row0 + row.token) * p.ldq + (size_t)row.head * HD;
        float4_t x[HD / 8];                       // the row's elements as the operands want them, all asked for at once
#pragma unroll
        for (int i = 0; i < HD / 8; i++) x[i] = *reinterpret_cast<const float4_t*>(q + (HALF ? i / 2 * 16 + hf * 8 + i % 2 * 4 : i * 8 + hf * 4));
        next = page_of(min(u0 + 1, u1 - 1));
        __syncthreads();                          // (the tile before is done with the LDS)
        issue(u0, here, 0);
        cap = p.softcap;
        invCap = MOD && cap > 0.f ? 1.f / cap : 0.f;
        slope = MOD && p.slopes ? p.slopes[row.head] : 0.f;
        c = p.scale;
        if constexpr (HALF) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) top = fmaxf(top, fabsf(x[i][j]));
            float other = top;
            row_swap32(top, other);
            top = fmaxf(top, other);
            const int up = power_up(top, c);
#pragma unroll
            for (int s = 0; s < QS; s++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = ldexpf(x[2 * s + j / 4][j % 4], up);
                    qh[s][j] = (_Float16)y;
                    ql[s][j] = (_Float16)(y - (float)qh[s][j]);
                }
            c = ldexpf(c, -up);
        } else {
#pragma unroll
            for (int s = 0; s < QS; s++) qf[s] = x[s];
        }
        if (!MOD) c *= 1.4426950408889634f;
        c = fminf(c, FLT_MAX);                    // (0 times it is 0)
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[b][i] = 0.f;
    }

    __device__ __forceinline__ int base_of(int u) const { return (t.unit0 + u) * UK; }
    // The page of the unit's run lane % (UK / 8) of eight positions, -1 where there is none
    __device__ __forceinline__ int page_of(int u) const {
        const int key = min(base_of(u) + (lane & (UK / 8 - 1)) * 8, span.end - 1);
        const int page = pages[max(key, 0) >> p.g.pageShift];
        return page >= 0 && page < p.g.nPages ? page : -1;
    }
    // Loads a unit into a buffer.  A load instruction's rows are within one run of eight positions.
    __device__ __forceinline__ void issue(int u, int mine, unsigned buf) const {
        const int base = base_of(u);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r0 = (wave * NI + i) * RI, run = r0 >> 3;
            const int page = __builtin_amdgcn_readlane(mine, run), key = base + run * 8;
            const bool inside = page >= 0 && key >= span.begin && key + 8 <= span.end;
            const size_t at = (size_t)(inside ? ((unsigned)page << p.g.pageShift) + ((unsigned)key & (unsigned)(p.g.pageSize - 1)) : 0u) * rowBytes;
            const unsigned dst = ldsBase + buf * BUFB + (unsigned)r0 * ROWB;
            if (inside) {
                asm volatile(PAGED_SET_M0 "global_load_lds_dwordx4 %1, %2" : : "s"(dst), "v"(from[i]), "s"(Kp + at) : "memory");
                asm volatile(PAGED_SET_M0 "global_load_lds_dwordx4 %1, %2" : : "s"(dst + TILEB), "v"(from[i]), "s"(Vp + at) : "memory");
            } else {
                const int r = r0 + lane / PR, piece = ((lane % PR) ^ swz(r)) * 16;
                const char* k = kv_row(Kp, zeros, rowBytes, base + r, page, span.begin, span.end, p.g.pageShift) + piece;
                const char* v = kv_row(Vp, zeros, rowBytes, base + r, page, span.begin, span.end, p.g.pageShift) + piece;
                asm volatile(PAGED_SET_M0 "global_load_lds_dwordx4 %1, off" : : "s"(dst), "v"(k) : "memory");
                asm volatile(PAGED_SET_M0 "global_load_lds_dwordx4 %1, off" : : "s"(dst + TILEB), "v"(v) : "memory");
            }
        }
    }
    static __device__ __forceinline__ uint4_t lds16(unsigned at) { return *reinterpret_cast<__attribute__((address_space(3))) const uint4_t*>(at); }
    // S^T of a unit: element i of block b is position 32 b + 8 (i/4) + 4 hf + i%4.  mends: where a NaN comes from the second term's
    // product with an infinite key, the first term's alone.
    __device__ __forceinline__ void scores(unsigned K, float16_t (&S)[NB], bool mend) const {
        const int r = anew(n32);
        const unsigned at = K + (unsigned)r * ROWB + (unsigned)(hf ^ swz(r)) * 16;
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int i = 0; i < 16; i++) S[b][i] = 0.f;
#pragma unroll
            for (int s = 0; s < QS; s++) {
                if (s % 4 == 0) __builtin_amdgcn_sched_barrier(0);       // (reads for four steps at once; for all, q would not stay in registers)
                const uint4_t k = lds16((at ^ (unsigned)(s * 32)) + b * 32 * ROWB);
                if constexpr (HALF) {
                    S[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, k), qh[s], S[b], 0, 0, 0);
                    S[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, k), ql[s], S[b], 0, 0, 0);
                } else {
                    const float4_t kf = __builtin_bit_cast(float4_t, k);
#pragma unroll
                    for (int j = 0; j < 4; j++) S[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[s][j], S[b], 0, 0, 0);
                }
            }
            if constexpr (HALF)
                if (mend) {
                    float16_t first;
#pragma unroll
                    for (int i = 0; i < 16; i++) first[i] = 0.f;
#pragma unroll
                    for (int s = 0; s < QS; s++) {
                        __builtin_amdgcn_sched_barrier(0);
                        first = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, lds16((at ^ (unsigned)(s * 32)) + b * 32 * ROWB)), qh[s], first, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) S[b][i] = S[b][i] != S[b][i] ? first[i] : S[b][i];
                }
        }
    }
    // Where the lane reads V of a unit at V: position 4 hf (fp32) or 4 hf + its quad's number (fp16), dimension block 0
    __device__ __forceinline__ unsigned v_base(unsigned V) const {
        const int x = anew(lane), h = x >> 5;
        if (HALF) {
            const int i16 = x & 15, a = i16 >> 2;
            return V + (unsigned)(4 * h + a) * ROWB + (unsigned)((2 * ((x >> 4) & 1) + ((i16 & 3) >> 1)) ^ ((a << 1) | h)) * 16 + (unsigned)(i16 & 1) * 8;
        }
        return V + (unsigned)(4 * h) * ROWB + (unsigned)(((x & 31) >> 2) ^ (4 * h)) * 16 + (unsigned)(x & 3) * 4;
    }
    // Block d of V^T P^T on top of `out`
    struct Weights { half8_t hi[HALF ? UK / 16 : 1], lo[HALF ? UK / 16 : 1]; };
    __device__ __forceinline__ float16_t product(unsigned V, int d, const float16_t (&S)[NB], const Weights& w, float16_t out) const {
        if constexpr (HALF) {
            const unsigned at = V ^ (unsigned)(d * 64);
#pragma unroll
            for (int kk = 0; kk < UK / 16; kk++) {
                typedef __attribute__((address_space(3))) short4_t* lp;
                const uint2_t x = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lp>(at + kk * 16 * ROWB)));
                const uint2_t y = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lp>(at + kk * 16 * ROWB + 8 * ROWB)));
                const half8_t v = __builtin_bit_cast(half8_t, uint4_t{x[0], x[1], y[0], y[1]});
                out = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w.hi[kk], out, 0, 0, 0);
                out = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w.lo[kk], out, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float v = *reinterpret_cast<__attribute__((address_space(3))) const float*>((V ^ (unsigned)(i % 4 * 16)) + (unsigned)(8 * (i / 4) + i % 4) * ROWB + (unsigned)d * 128);
                out = __builtin_amdgcn_mfma_f32_32x32x2f32(v, S[0][i], out, 0, 0, 0);
            }
        }
        return out;
    }
    // A unit's values in LDS to what stands for them in a pass (elements side by side: their order does not matter)
    __device__ __forceinline__ void replace(unsigned V, int pass) const {
#pragma unroll 1
        for (int i = thread_anew(); i < TILEB / 16; i += WG) {
            uint4_t x = lds16(V + (unsigned)i * 16);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = stand_in<HALF>(x[j], pass);
            *reinterpret_cast<__attribute__((address_space(3))) uint4_t*>(V + (unsigned)i * 16) = x;
        }
    }
    // Scores to probabilities (times 2^SHIFT, over the maximum mNew); returns the lane's sum of them
    __device__ __forceinline__ float weigh(float16_t (&S)[NB], int base, unsigned long long held, bool all, float& mNew) const {
        const int first = base + 4 * anew(hf);            // the lane's first position
        if constexpr (MOD) {
#pragma unroll
            for (int b = 0; b < NB; b++) S[b] *= c;
            if (cap > 0.f) cap_all(S, cap, invCap);
            if (p.slopes) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) S[b][i] = fmaf(-slope, (float)abs(row.pos - (first + 32 * b + 8 * (i / 4) + i % 4)), S[b][i]);
            }
        }
        const float factor = MOD ? 1.4426950408889634f : c;          // scores to powers of two
        if (!all) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!((held >> (4 * b + i / 4)) & 1) || !paged_sees(row.pos, first + 32 * b + 8 * (i / 4) + i % 4, t.len, p.window, t.prefix)) S[b][i] = -INFINITY;
        }
        float top = S[0][0];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, S[b][i]);
        float other = top;
        row_swap32(top, other);
        top = fmaxf(top, other);
        top = top == -INFINITY ? top : top * factor;
        mNew = top > m + LAZY || m == -INFINITY ? fmaxf(m, top) : m;
        const float shift = SHIFT - (mNew == -INFINITY ? 0.f : mNew);          // (a score that is a NaN stays one)
        float ts = 0.f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                S[b][i] = __builtin_amdgcn_exp2f(fmaf(S[b][i], factor, shift));
                ts += S[b][i];
            }
        return ts;
    }
    // Unit u, of page numbers `here`, in buffer `buf`; asks for the one behind it on the way
    template <bool AGAIN>
    __device__ __forceinline__ void compute(int u, bool more, unsigned buf, int pass) {
        const int base = base_of(u), mine = here;
        if (!active || base >= end || base + UK <= begin) {
            if (more) issue(u + 1, next, buf ^ 1);
            return;
        }
        const unsigned K = ldsBase + buf * BUFB, V = K + TILEB;
        const unsigned long long held = __ballot(mine >= 0);
        constexpr unsigned long long runs = (1ull << (UK / 8)) - 1;
        const bool inner = base + UK <= t.prefix || (base + UK - 1 <= pos0 && (p.window == 0 || base > pos1 - p.window));        // all rows see all of it
        const bool all = inner && (held & runs) == runs;
        float16_t S[NB];
        float mNew;
        scores(K, S, false);
        if (more) issue(u + 1, next, buf ^ 1);
        float ts = weigh(S, base, held, all, mNew);
        if (HALF && __any(ts != ts)) {            // (not a loop: what the masks need would be worked out ahead of it, for every unit)
            scores(K, S, true);
            ts = weigh(S, base, held, all, mNew);
        }
        if (__any(mNew != m)) {
            const float f = mNew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mNew);
            l *= f;
#pragma unroll
            for (int b = 0; b < DB; b++) o[b] *= f;
            m = mNew;
        }
        l += ts;
        if (!inner && !__any(ts != 0.f)) return;          // (no row has anything here)
        if (AGAIN && pass != FINITE) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) S[b][i] = S[b][i] > 0.f ? 1.f : 0.f;
        }
        Weights w;
        if constexpr (HALF) {
#pragma unroll
            for (int kk = 0; kk < UK / 16; kk++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = S[kk / 2][8 * (kk % 2) + i];
                    w.hi[kk][i] = (_Float16)x;
                    w.lo[kk][i] = (_Float16)(x - (float)w.hi[kk][i]);
                }
        }
        const unsigned Vl = v_base(V);
#pragma unroll
        for (int d = 0; d < DB; d++) {
            __builtin_amdgcn_sched_barrier(0);            // (as in scores)
            o[d] = product(Vl, d, S, w, o[d]);
        }
    }
    template <bool AGAIN>
    __device__ __forceinline__ void units(int u0, int u1, int pass) {
        unsigned buf = 0;
        for (int u = u0; u < u1; u++) {
            // this unit's rows have landed; nobody reads the other buffer any more
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const int behind = page_of(min(u + 2, u1 - 1));
            if constexpr (AGAIN) {
                replace(ldsBase + buf * BUFB + TILEB, pass);
                __syncthreads();
            }
            compute<AGAIN>(u, u + 1 < u1, buf, pass);
            here = next;
            next = behind;
            buf ^= 1;
        }
    }
    __device__ __forceinline__ void run(int u0, int u1, int, int, float* lds) {
        units<false>(u0, u1, 0);
        float odd = 0.f;
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) odd = fmaf(o[b][i], 0.f, odd);
        const bool any = __any(odd != odd);
        unsigned* votes = reinterpret_cast<unsigned*>(lds) + VOTES;
        if (lane == 0) votes[wave] = any;
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(votes[0] | votes[1] | votes[2] | votes[3])) {         // all four waves, or none
            unsigned long long plus = 0, minus = 0;       // a bit an element
#pragma unroll 1
            for (int pass = PLUS_INFINITE; pass <= FINITE; pass++) {
                here = page_of(u0);
                next = page_of(min(u0 + 1, u1 - 1));
                issue(u0, here, 0);
                l = 0.f;
#pragma unroll
                for (int b = 0; b < DB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[b][i] = 0.f;
                units<true>(u0, u1, pass);
                unsigned long long counts = 0;
#pragma unroll
                for (int b = 0; b < DB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) counts |= (o[b][i] > 0.f ? 1ull : 0ull) << (16 * b + i);
                if (pass == PLUS_INFINITE) plus = counts;
                if (pass == MINUS_INFINITE) minus = counts;
                __syncthreads();                          // (the last unit's buffer may be the first one's)
            }
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] = with_infinities(o[b][i], plus >> (16 * b + i) & 1, minus >> (16 * b + i) & 1);
        }
        float other = l;
        row_swap32(l, other);
        l += other;
    }
    // A share lies as its registers do -- a wave's block b, rows of four i / 4, then its 64 lanes -- so that stores and loads are whole lines
    __device__ __forceinline__ void write(int kvh, int w, float* lds) {
        const int r = 32 * wave + n32;
        if (t.worker0 != t.worker1) {
            float* part = part_of(p, t, kvh, w);
            if (active) {
#pragma unroll
                for (int b = 0; b < DB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        store_through(part + ((wave * DB + b) * 4 + i) * 256 + lane * 4, float4_t{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]});
                if (hf == 0) { st_agent(part + WIDE * HD + r, m); st_agent(part + WIDE * HD + WIDE + r, l); }
            }
            __syncthreads();                      // (all waves are done with the last unit's LDS)
            if (!last_to_finish(p, t, kvh, lds)) return;
            float *M = lds, *den = lds + WIDE, *wt = lds + 2 * WIDE;
            constexpr int TURN = MERGE_LDS / WIDE;
            const int segs = t.worker1 - t.worker0 + 1, R = min(WIDE, t.rows * p.g.group - t.first);
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] = 0.f;
            for (int s0 = 0; s0 < segs; s0 += TURN) {
                const int n = min(TURN, segs - s0);
                merge_weights<HD, WIDE>(p, t, kvh, R, s0, n, M, den, wt);
                if (!active) continue;
                for (int s = 0; s < n; s++) {
                    const float* from = part_of(p, t, kvh, t.worker0 + s0 + s) + wave * DB * 4 * 256 + lane * 4;
                    const float f = wt[s * WIDE + r];
#pragma unroll
                    for (int b = 0; b < DB; b++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float4_t v = *reinterpret_cast<const float4_t*>(from + (b * 4 + i) * 256);
#pragma unroll
                            for (int j = 0; j < 4; j++) o[b][4 * i + j] = fmaf(f, v[j], o[b][4 * i + j]);
                        }
                }
            }
            __syncthreads();
            l = den[r];
        }
        if (t.first + r >= t.rows * p.g.group) return;
        float* out = p.out + (size_t)(t.row0 + row.token) * p.ldo + (size_t)row.head * HD + 4 * hf;
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<float4_t*>(out + 32 * b + 8 * i) = over(float4_t{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]}, l);
    }
};

template <typename KVT, int HD, bool MOD, template <typename, int, bool> class Tile, int ROWS>
__device__ __forceinline__ void attend(const PagedAttention& p, float* lds) {
    // neighbouring shares on one die, whose L2 then holds the KV head's rows that they have in common
    const int id = (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3));
    const int kvh = id / p.nWorkers, w = id % p.nWorkers;
    if (kvh >= p.g.nKVHeads) return;
    const PagedWorker* k = p.workers + w;
    const int a = __builtin_amdgcn_readfirstlane(k->a), b = __builtin_amdgcn_readfirstlane(k->b), tiles = __builtin_amdgcn_readfirstlane(k->tiles);
    const bool ours = p.made->is(p.plan);             // (asked for together with the share)
    PagedTile t = tile_at(&k->tile);
    if (!ours || a >= b) return;
    for (;;) {
        const int u0 = paged_unit_at(t, a), u1 = paged_unit_at(t, b);
        if (u0 < u1) {
            Tile<KVT, HD, MOD> n(p, t, kvh, u0, u1);
            n.run(u0, u1, kvh, w, lds);
            n.write(kvh, w, lds);
        } else if (t.units == 0 && a <= t.cost0 && t.cost0 < b) {
            for (int i = threadIdx.x; i < min(ROWS, t.rows * p.g.group - t.first) * (HD / 4); i += WG) {
                const PagedRow at = paged_row(t, p.g.group, kvh, i / (HD / 4));
                *reinterpret_cast<float4*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + (i % (HD / 4)) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        if (t.index + 1 >= tiles) break;
        t = tile_at(p.tiles + t.index + 1);
        if (t.cost0 >= b) break;
    }
}
template <typename KVT, int HD, bool MOD>
__global__ __launch_bounds__(WG, 2) void paged_narrow_kernel(PagedAttention p) {
    extern __shared__ __attribute__((aligned(1024))) float lds[];      // (all the LDS there is: it starts at 0)
    attend<KVT, HD, MOD, NarrowTile, NARROW>(p, lds);
}
template <typename KVT, int HD, bool MOD>
__global__ __launch_bounds__(WG, 2) void paged_wide_kernel(PagedAttention p) {
    extern __shared__ __attribute__((aligned(1024))) float lds[];
    attend<KVT, HD, MOD, WideTile, WIDE>(p, lds);
}

static size_t attn_lds(int headDim, bool wide) {
    const size_t tile = wide ? (size_t)2 * 2 * 64 * headDim * 2 + 16 : (size_t)(4 * NARROW * (headDim + 4) + 8 * NARROW) * 4;
    const size_t merge = (size_t)(2 * (wide ? WIDE : NARROW) + MERGE_LDS) * 4;
    return tile > merge ? tile : merge;
}
template <typename F>
static hipError_t with_kernel(const PagedGeo& g, bool mod, bool wide, F f) {
#define PAGED_PICK(KVT, HD, MOD) (wide ? f(paged_wide_kernel<KVT, HD, MOD>) : f(paged_narrow_kernel<KVT, HD, MOD>))
    if (g.kvHalf) {
        if (g.headDim == 64) return mod ? PAGED_PICK(_Float16, 64, true) : PAGED_PICK(_Float16, 64, false);
        return mod ? PAGED_PICK(_Float16, 128, true) : PAGED_PICK(_Float16, 128, false);
    }
    if (g.headDim == 64) return mod ? PAGED_PICK(float, 64, true) : PAGED_PICK(float, 64, false);
    return mod ? PAGED_PICK(float, 128, true) : PAGED_PICK(float, 128, false);
#undef PAGED_PICK
}
hipError_t paged_attention_setup(const PagedGeo& g) {
    for (int i = 0; i < 4; i++) {
        hipError_t e = with_kernel(g, i & 1, i >> 1, [&](auto* k) {
            return hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)attn_lds(g.headDim, i >> 1));
        });
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
hipError_t launch_paged_attention(const PagedAttention& p0, hipStream_t s) {
    for (int wide = p0.wideWorkers > 0; wide >= 0; wide--) {
        PagedAttention p = p0;
        if (wide) p.nWorkers = p.wideWorkers;
        const int groups = (p.nWorkers * p.g.nKVHeads + 7) / 8 * 8;
        p.tiles += wide ? p.maxTiles : 0;
        p.workers += wide ? p.maxWorkers : 0;
        const size_t lds = attn_lds(p.g.headDim, wide);
        hipError_t e = with_kernel(p.g, p.softcap > 0.f || p.slopes, wide, [&](auto* k) {
            hipLaunchKernelGGL(k, dim3(groups), dim3(WG), lds, s, p);
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mg
