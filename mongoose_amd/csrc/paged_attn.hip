// paged_attn.hip -- attention of each request's new tokens over its pages of the cache.
//
// For a token at position i and a query head h over KV head h / group:
//     s_j = scale * q . k_j;  with a cap s_j = cap * tanh(s_j / cap);  with slopes s_j -= slope_h * |i - j|
//     o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)   over the positions j that i sees (paged_sees), m their greatest s_j
// in one pass: a running maximum m, sum l and output O, the latter two multiplied by exp(m - m') where m grows to m'.  A token that
// sees nothing gets zeros.
//
// A query head's rows and the other heads' of its KV head go together: a tile is 16 rows (token, head), so that every K and V row is
// read once for all of them.  Scores are computed transposed, S^T = K Q^T, and the output O^T = V^T P^T: the MFMA result of the
// first (a lane: one query row, several positions) is the operand of the second as it stands, and a row's maximum and sum are
// a lane's own but for two exchanges.
#include "device_util.h"
#include "paged.h"

namespace mg {

constexpr int PT = 1024;                  // threads of the plan
constexpr int NARROW = 16;                // rows of a tile
constexpr int PLAN_LDS_TILES = 4096;      // tiles whose places on the line the plan holds in LDS
constexpr int MERGE_LDS = 8192;           // floats of LDS for the weights of partial results

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));

static int narrow_keys(int kvHalf) { return kvHalf ? 128 : 64; }       // positions of a unit: four waves x a step of 32 or 16
int paged_max_tiles(const PagedGeo& g) { return (int)((long long)g.maxRows * g.group / NARROW) + g.maxReqs; }
size_t paged_part_floats(const PagedGeo& g) { return (size_t)NARROW * (g.headDim + 2); }
// Two workgroups a CU, in turns of the KV heads; fewer where the batch cannot have that many units.
int paged_workers(const PagedGeo& g, int nReqs, int rows) {
    const long long tiles = (long long)rows * g.group / NARROW + nReqs, units = tiles * (g.maxLen / narrow_keys(g.kvHalf) + 2);
    const long long most = 512 / g.nKVHeads > 0 ? 512 / g.nKVHeads : 1;
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
__global__ __launch_bounds__(PT) void paged_plan_kernel(PagedPlan p, int unitKeys) {
    __shared__ unsigned tile0[PAGED_MAX_REQS + 1], place[PLAN_LDS_TILES], part[PT / 64];
    const int tid = threadIdx.x;
    unsigned nTiles = 0;
    if (tid == 0) tile0[0] = 0;
    for (int r0 = 0; r0 < p.nReqs; r0 += PT) {
        const int r = r0 + tid;
        unsigned n = 0;
        if (r < p.nReqs) n = (unsigned)((plan_request(p, r).y * p.group + NARROW - 1) / NARROW);
        n = plan_scan(n, nTiles, part);
        if (r < p.nReqs) tile0[r + 1] = n;
    }
    __syncthreads();
    nTiles = min(nTiles, (unsigned)p.maxTiles);          // (more only where the caller's rows overlap)
    unsigned cost = 0;
    for (unsigned i0 = 0; i0 < nTiles; i0 += PT) {
        const unsigned i = i0 + tid;
        PagedTile t{};
        unsigned c = 0;
        if (i < nTiles) {
            int lo = 0, hi = p.nReqs;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (tile0[mid] <= i) lo = mid; else hi = mid;
            }
            const int4 rq = plan_request(p, lo);
            t.req = lo; t.row0 = rq.x; t.rows = rq.y; t.len = rq.z; t.prefix = rq.w;
            t.first = (int)(i - tile0[lo]) * NARROW;
            t.index = (int)i;
            t.tileRows = NARROW; t.unitKeys = unitKeys; t.weight = 1;
            paged_units(t, p.window, p.group);
            c = (unsigned)(PAGED_TILE_COST + t.units * t.weight);
        }
        const unsigned end = plan_scan(c, cost, part);
        if (i < nTiles) {
            t.cost0 = (int)(end - c);
            if (i < PLAN_LDS_TILES) place[i] = end - c;
            p.tiles[i] = t;
        }
    }
    __syncthreads();
    const int workers = max(1, min(p.nWorkers, (int)cost));
    for (unsigned i = tid; i < nTiles; i += PT) {
        PagedTile* t = p.tiles + i;
        const int x = t->cost0 + PAGED_TILE_COST;
        t->worker0 = t->units ? paged_worker_of((int)cost, workers, x) : 0;
        t->worker1 = t->units ? paged_worker_of((int)cost, workers, x + (t->units - 1) * t->weight) : 0;
    }
    __syncthreads();
    for (int w = tid; w < p.nWorkers; w += PT) {
        PagedWorker k{};
        if (w < workers && nTiles > 0) {
            k.a = paged_share((int)cost, workers, w);
            k.b = paged_share((int)cost, workers, w + 1);
            unsigned lo = 0, hi = nTiles;
            while (hi - lo > 1) {
                const unsigned mid = (lo + hi) >> 1;
                if ((mid < PLAN_LDS_TILES ? place[mid] : (unsigned)p.tiles[mid].cost0) <= (unsigned)k.a) lo = mid; else hi = mid;
            }
            k.tile = p.tiles[lo];
            k.tiles = (int)nTiles;
        }
        p.workers[w] = k;
    }
}
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(PT), 0, s, p, narrow_keys(p.kvHalf));
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// cap * tanh(x / cap): the odd Taylor polynomial up to x^13 where |x / cap| < 0.45 (the next term is below 2^-26 of the result),
// (1 - e^-2x) / (1 + e^-2x) beyond.
__device__ __forceinline__ float capped(float s, float cap, float invCap) {
    const float x = s * invCap, a = fabsf(x), x2 = x * x;
    float t = fmaf(x2, 21844.f / 6081075.f, -1382.f / 155925.f);
    t = fmaf(x2, t, 62.f / 2835.f);
    t = fmaf(x2, t, -17.f / 315.f);
    t = fmaf(x2, t, 2.f / 15.f);
    t = fmaf(x2, t, -1.f / 3.f);
    t = fmaf(x * x2, t, x);
    const float e = __builtin_amdgcn_exp2f(a * -2.885390081777927f);
    const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
    return cap * (a < 0.45f ? t : far);
}
// 16 bytes through to memory, for a workgroup of another die to read within the launch
__device__ __forceinline__ void store_through(float* p, float4_t v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1" : : "v"(p), "v"(v) : "memory");
}
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

// The workgroup's result of a tile: row r at o + r * HD (LDS), maxima and sums behind; written out, or as a partial result with the
// last worker to finish putting the tile together.
template <int HD, int ROWS>
__device__ __forceinline__ void finish(const PagedAttention& p, const PagedTile& t, int kvh, int w, const float* o, const float* ms, const float* ls, float* scratch) {
    const int tid = threadIdx.x, R = min(ROWS, t.rows * p.g.group - t.first);
    if (t.worker0 == t.worker1) {
        for (int i = tid; i < R * (HD / 4); i += WG) {
            const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
            const float l = ls[row];
            const float4 v = *reinterpret_cast<const float4*>(o + row * (HD + 4) + d);
            const PagedRow at = paged_row(t, p.g.group, kvh, row);
            *reinterpret_cast<float4*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + d) =
                l == 0.f ? v : make_float4(v.x / l, v.y / l, v.z / l, v.w / l);       // (nothing seen: zeros)
        }
        return;
    }
    constexpr size_t stride = (size_t)ROWS * (HD + 2);
    float* parts = p.parts + (size_t)kvh * p.nWorkers * 2 * stride;
    float* mine = parts + ((size_t)w * 2 + (w == t.worker0)) * stride;
    for (int i = tid; i < R * (HD / 4); i += WG) {
        const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
        store_through(mine + row * HD + d, *reinterpret_cast<const float4_t*>(o + row * (HD + 4) + d));
    }
    for (int i = tid; i < R; i += WG) { st_agent(mine + ROWS * HD + i, ms[i]); st_agent(mine + ROWS * HD + ROWS + i, ls[i]); }
    __shared__ unsigned before;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int segs = t.worker1 - t.worker0 + 1;
    unsigned* count = p.arrived + (size_t)kvh * p.maxTiles + t.index;
    if (tid == 0) before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (before + 1 != (unsigned)segs) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Rows' greatest maxima and sums first, into `scratch` beside every partial result's weight; then the outputs, the workgroup's
    // threads sharing out rows, columns and, where there are few of those, partial results.
    auto part_of = [&](int s) { return parts + ((size_t)(t.worker0 + s) * 2 + (s == 0)) * stride; };
    float* M = scratch;                   // [ROWS]
    float* den = scratch + ROWS;          // [ROWS]
    float* wt = scratch + 2 * ROWS;       // [segs in turn][R]
    const int perTurn = MERGE_LDS / ROWS;
    const int cols = R * (HD / 4), par = max(1, WG / cols);
    if (tid < R) {
        float m = -INFINITY;
#pragma unroll 8
        for (int s = 0; s < segs; s++) m = fmaxf(m, part_of(s)[ROWS * HD + tid]);
        M[tid] = m == -INFINITY ? 0.f : m;
        den[tid] = 0.f;
    }
    float4 acc[(ROWS * HD / 4 + WG - 1) / WG];
#pragma unroll
    for (auto& a : acc) a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < segs; s0 += perTurn) {
        const int n = min(perTurn, segs - s0);
        __syncthreads();
        for (int i = tid; i < n * R; i += WG) wt[i] = __builtin_amdgcn_exp2f(part_of(s0 + i / R)[ROWS * HD + i % R] - M[i % R]);
        __syncthreads();
        if (tid < R) {
            float d = den[tid];
#pragma unroll 8
            for (int s = 0; s < n; s++) d = fmaf(wt[s * R + tid], part_of(s0 + s)[ROWS * HD + ROWS + tid], d);
            den[tid] = d;
        }
#pragma unroll
        for (int k = 0; k < (int)(sizeof(acc) / sizeof(acc[0])); k++) {
            const int i = par > 1 ? tid % cols : tid + k * WG, from = par > 1 ? tid / cols : 0;
            if (i >= cols || from >= par || (par > 1 && k > 0)) continue;
            const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
#pragma unroll 4
            for (int s = from; s < n; s += par) {
                const float4 v = *reinterpret_cast<const float4*>(part_of(s0 + s) + row * HD + d);
                const float f = wt[s * R + row];
                acc[k].x = fmaf(f, v.x, acc[k].x); acc[k].y = fmaf(f, v.y, acc[k].y); acc[k].z = fmaf(f, v.z, acc[k].z); acc[k].w = fmaf(f, v.w, acc[k].w);
            }
        }
    }
    __syncthreads();
    if (par > 1) {                        // the shares of the same columns, in their order
        float4* x = reinterpret_cast<float4*>(wt);
        if (tid / cols < par) x[tid] = acc[0];
        __syncthreads();
        if (tid < cols)
            for (int k = 1; k < par; k++) {
                const float4 v = x[tid + k * cols];
                acc[0].x += v.x; acc[0].y += v.y; acc[0].z += v.z; acc[0].w += v.w;
            }
    }
#pragma unroll
    for (int k = 0; k < (int)(sizeof(acc) / sizeof(acc[0])); k++) {
        const int i = tid + k * WG;
        if (i >= cols) continue;
        const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
        const float l = den[row];
        const PagedRow at = paged_row(t, p.g.group, kvh, row);
        *reinterpret_cast<float4*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + d) =
            l == 0.f ? acc[k] : make_float4(acc[k].x / l, acc[k].y / l, acc[k].z / l, acc[k].w / l);
    }
}

// A tile of 16 rows: four waves take a step of KB positions each of every unit, each with its own running maximum, sum and output.
// Bound by HBM: a lane loads its K and V operands from the pages straight into registers, a step ahead and the page numbers two
// steps ahead; nothing is shared between the waves before the end.
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

    __device__ __forceinline__ NarrowTile(const PagedAttention& p_, const PagedTile& t_, int kvh) : p(p_), t(t_) {
        const int tid = threadIdx.x;
        lane = tid & 63; l16 = lane & 15; g = lane >> 4;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        span = paged_span(t.rows, t.len, t.prefix, p.window, p.g.group, t.first, NARROW);
        row = paged_row(t, p.g.group, kvh, l16);
        pages = p.table + (size_t)t.req * p.g.width;
        rowBytes = (size_t)p.g.kvDim * sizeof(KVT);
        Kp = static_cast<const char*>(p.K) + (size_t)kvh * HD * sizeof(KVT);
        Vp = static_cast<const char*>(p.V) + (size_t)kvh * HD * sizeof(KVT);
        zeros = reinterpret_cast<const char*>(p.zeros);
        cap = p.softcap;
        invCap = MOD && cap > 0.f ? 1.f / cap : 0.f;
        slope = MOD && p.slopes ? p.slopes[row.head] : 0.f;
        const float* q = p.q + (size_t)(t.row0 + row.token) * p.ldq + (size_t)row.head * HD;
        c = p.scale;
        if constexpr (HALF) {
            float x[HD / 32][8], top = 0.f;
#pragma unroll
            for (int s = 0; s < HD / 32; s++) {
                const float4 a = *reinterpret_cast<const float4*>(q + s * 32 + g * 8), b = *reinterpret_cast<const float4*>(q + s * 32 + g * 8 + 4);
                x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w; x[s][4] = b.x; x[s][5] = b.y; x[s][6] = b.z; x[s][7] = b.w;
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[s][j]));
            }
            top = rows_max(top);
            const int up = top > 0.f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
            for (int s = 0; s < HD / 32; s++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = ldexpf(x[s][j], up);
                    qh[s][j] = (_Float16)v;
                    ql[s][j] = (_Float16)(v - (float)qh[s][j]);
                }
            c = ldexpf(c, -up);
        } else {
#pragma unroll
            for (int s = 0; s < HD / 16; s++) qf[s] = *reinterpret_cast<const float4_t*>(q + s * 16 + g * 4);
        }
        if (!MOD) c *= 1.4426950408889634f;
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
    // Block e of V^T P^T on top of `out`; keep: all ones for the lane's positions that count
    template <bool MASKED>
    __device__ __forceinline__ float4_t product(int e, const Weights& w, const unsigned (&keep)[NB * 4], float4_t out) const {
        auto word = [&](int j, int i) { return MASKED ? v[j][i] & keep[j] : v[j][i]; };
        if constexpr (HALF) {
            uint4_t a;
#pragma unroll
            for (int j = 0; j < 4; j++) a[j] = __builtin_amdgcn_perm(word(2 * j + 1, e / 2), word(2 * j, e / 2), e & 1 ? 0x07060302u : 0x05040100u);
            out = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), w.hi, out, 0, 0, 0);
            out = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), w.lo, out, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) out = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, word(i, e)), w.x[i], out, 0, 0, 0);
        }
        return out;
    }
    static __device__ __forceinline__ bool not_finite(unsigned v) {
        if (HALF) return ((v & 0x7fffu) >= 0x7c00u) | ((v & 0x7fff0000u) >= 0x7c000000u);
        return (v & 0x7fffffffu) >= 0x7f800000u;
    }
    // Step u, on page numbers `mine`; loads the K rows of the one behind it (if any, on page numbers `next`) where it is done with its own
    __device__ __forceinline__ void compute(int u, int mine, bool more, int next) {
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
        for (int j = 0; j < NB * 4; j++) {
            x[j] = S[j / 4][j % 4] * c;
            if (MOD) {
                if (cap > 0.f) x[j] = capped(x[j], cap, invCap);
                x[j] = (x[j] - slope * (float)abs(row.pos - (base + 16 * (j / 4) + 4 * g + j % 4))) * 1.4426950408889634f;
            }
        }
        const bool all = __all(mine >= 0) && (base + KB <= t.prefix || (base + KB - 1 <= span.pos0 && (p.window == 0 || base > span.pos1 - p.window)));
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
        bool odd = false;
        if (!all && span.pos0 != span.pos1) {
#pragma unroll
            for (int j = 0; j < NB * 4; j++)
#pragma unroll
                for (int e = 0; e < VW; e++) odd |= not_finite(v[j][e]);
        }
        const Weights wt = weights(x);
        unsigned keep[NB * 4];
        if (!__any(odd)) {
#pragma unroll
            for (int e = 0; e < EPL; e++) o[e] = product<false>(e, wt, keep, o[e]);
            return;
        }
        // Values that are no numbers at positions that not every token sees, and zero times them is no zero: token by token, with
        // the positions that it does not see taken out.
#pragma unroll 1
        for (int pos = span.pos0; pos <= span.pos1; pos++) {
#pragma unroll
            for (int j = 0; j < NB * 4; j++) keep[j] = paged_sees(pos, base + 16 * (j / 4) + 4 * g + j % 4, t.len, p.window, t.prefix) ? ~0u : 0u;
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                const float4_t part = product<true>(e, wt, keep, float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int i = 0; i < 4; i++) o[e][i] = row.pos == pos ? o[e][i] + part[i] : o[e][i];
            }
        }
    }
    __device__ __forceinline__ void run(int u0, int u1) {
        int here = page_of(u0), next = page_of(min(u0 + 1, u1 - 1));
        load_k(u0, here);
        load_v(u0, here);
        for (int u = u0; u < u1; u++) {
            const int behind = page_of(min(u + 2, u1 - 1));
            const bool more = u + 1 < u1;
            compute(u, here, more, next);
            if (more) load_v(u + 1, next);
            here = next;
            next = behind;
        }
    }
    // The four waves' results as one, at lds (rows of HD + 4 floats) with maxima and sums behind
    static constexpr int FLOATS = 4 * NARROW * (HD + 4) + 8 * NARROW;
    __device__ __forceinline__ void join(float* lds) {
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
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = tid; i < NARROW * (HD / 4); i += WG) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
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
};

template <typename KVT, int HD, bool MOD>
__global__ __launch_bounds__(WG, 2) void paged_attn_kernel(PagedAttention p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    // neighbouring shares on one die, whose L2 then holds the KV head's rows that they have in common
    const int id = (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3));
    const int kvh = id / p.nWorkers, w = id % p.nWorkers;
    if (kvh >= p.g.nKVHeads) return;
    const PagedWorker* k = p.workers + w;
    const int a = __builtin_amdgcn_readfirstlane(k->a), b = __builtin_amdgcn_readfirstlane(k->b), tiles = __builtin_amdgcn_readfirstlane(k->tiles);
    if (a >= b) return;
    PagedTile t = tile_at(&k->tile);
    for (;;) {
        const int u0 = paged_unit_at(t, a), u1 = paged_unit_at(t, b);
        if (u0 < u1) {
            NarrowTile<KVT, HD, MOD> n(p, t, kvh);
            n.run(u0, u1);
            n.join(lds);
            finish<HD, NARROW>(p, t, kvh, w, lds, lds + 4 * NARROW * (HD + 4), lds + 4 * NARROW * (HD + 4) + 4 * NARROW, lds);
        } else if (t.units == 0 && a <= t.cost0 && t.cost0 < b) {
            for (int i = threadIdx.x; i < min(NARROW, t.rows * p.g.group - t.first) * (HD / 4); i += WG) {
                const PagedRow at = paged_row(t, p.g.group, kvh, i / (HD / 4));
                *reinterpret_cast<float4*>(p.out + (size_t)(t.row0 + at.token) * p.ldo + (size_t)at.head * HD + (i % (HD / 4)) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        if (t.index + 1 >= tiles) break;
        t = tile_at(p.tiles + t.index + 1);
        if (t.cost0 >= b) break;
    }
}

static size_t attn_lds(int headDim) {
    const int tile = 4 * NARROW * (headDim + 4) + 8 * NARROW, merge = 2 * NARROW + MERGE_LDS;
    return (size_t)(tile > merge ? tile : merge) * 4;
}
template <typename F>
static hipError_t with_kernel(const PagedGeo& g, bool mod, F f) {
    if (g.kvHalf) {
        if (g.headDim == 64) return mod ? f(paged_attn_kernel<_Float16, 64, true>) : f(paged_attn_kernel<_Float16, 64, false>);
        return mod ? f(paged_attn_kernel<_Float16, 128, true>) : f(paged_attn_kernel<_Float16, 128, false>);
    }
    if (g.headDim == 64) return mod ? f(paged_attn_kernel<float, 64, true>) : f(paged_attn_kernel<float, 64, false>);
    return mod ? f(paged_attn_kernel<float, 128, true>) : f(paged_attn_kernel<float, 128, false>);
}
hipError_t paged_attention_setup(const PagedGeo& g) {
    for (bool mod : {false, true}) {
        hipError_t e = with_kernel(g, mod, [&](auto* k) {
            return hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)attn_lds(g.headDim));
        });
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t s) {
    const int groups = (p.nWorkers * p.g.nKVHeads + 7) / 8 * 8;
    return with_kernel(p.g, p.softcap > 0.f || p.slopes, [&](auto* k) {
        hipLaunchKernelGGL(k, dim3(groups), dim3(WG), attn_lds(p.g.headDim), s, p);
        return hipGetLastError();
    });
}

}  // namespace mg
