// paged.hip -- a KV cache in pages that several requests share: the handle (mg_paged_*), block tables and slot maps from
// request lengths, and rotary positions with the K/V rows stored by slot.  The attention that reads the pages is in paged_attn.hip.
#include "paged.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <string>

#include "../../include/mongoose_hip.h"
#include "fused_infer.h"
#include "kernels.h"

namespace mg {

// ---------------------------------------------------------------------------
// Block tables and slot maps
//
// With P(x) = ceil(x / page), request r takes P(len + new) - P(len) pages, or gives P(len) back when it has ended (new = -1).
// Three exclusive sums over the requests -- rows, pages taken, pages given back -- place everything else: row i of the step
// belongs to the request whose rows cover it (a binary search in the sums), a page taken is the free ring's entry head + its
// number, a page given back goes to entry head + count + its number.  Only pages free before the call are taken, so the entries
// read and the entries written never meet.  Every workgroup makes the sums for itself (at most 4,096 requests: four rounds of
// 1,024 threads), which costs less than a launch that makes them for all.  Bound by latency: loads, sums, a search, a page's id
// (64 requests of a token each 4.3 us).
// ---------------------------------------------------------------------------
constexpr int TB = 1024;
constexpr int TABLE_ROWS = 1024;      // rows a workgroup maps

struct TableSums { unsigned rows, taken, given; };
__device__ __forceinline__ TableSums add(TableSums a, TableSums b) {
    return {sat_add(a.rows, b.rows), sat_add(a.taken, b.taken), sat_add(a.given, b.given)};
}
// Largest r with sums[r] <= i (sums[0] = 0 <= i < sums[n]): requests without rows are passed over
__device__ __forceinline__ int find(const unsigned* sums, int n, unsigned i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// commit: 0 = no workgroup writes the state a following call starts from (lensOut, ringStateOut, rowStart, counts), 1 = the
// first one does, after its own reads, 2 = nothing but that
__global__ __launch_bounds__(TB) void paged_tables_kernel(PagedTables p, int commit) {
    extern __shared__ unsigned sums[];
    unsigned *start = sums, *took = sums + p.nReqs + 1, *gave = took + p.nReqs + 1;
    __shared__ TableSums part[TB / 64];
    __shared__ int sFlags;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int head = p.ringState[0], count = p.ringState[1];
    if (tid == 0) { sFlags = 0; start[0] = took[0] = gave[0] = 0; }
    TableSums carry{0, 0, 0};
    for (int r0 = 0; r0 < p.nReqs; r0 += TB) {
        const int r = r0 + tid;
        TableSums v{0, 0, 0};
        int bad = 0;
        if (r < p.nReqs) {
            int len = p.lens[r], add = p.newLens[r];
            if (len < 0 || len > p.maxLen || add < -1 || add > p.maxLen || (add > 0 && len + add > p.maxLen)) { bad = 1; len = 0; add = 0; }
            const unsigned held = (unsigned)paged_pages(len, p.pageShift);
            if (add < 0) v.given = held;
            else { v.rows = (unsigned)add; v.taken = (unsigned)paged_pages(len + add, p.pageShift) - held; }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const TableSums o{(unsigned)__shfl_up((int)v.rows, d, 64), (unsigned)__shfl_up((int)v.taken, d, 64), (unsigned)__shfl_up((int)v.given, d, 64)};
            if (lane >= d) v = add(o, v);
        }
        __syncthreads();                                  // (part and sFlags of the round before are read, or set up)
        if (lane == 63) part[wave] = v;
        if (bad) atomicOr(&sFlags, PAGED_BAD_LENGTH);
        __syncthreads();
        TableSums before = carry;
        const int waves = min(TB, p.nReqs - r0 + 63) >> 6;    // (waves past the requests have nothing)
        for (int w = 0; w < waves; w++) {
            if (w == wave) v = add(before, v);
            before = add(before, part[w]);
        }
        carry = before;
        if (r < p.nReqs) { start[r + 1] = v.rows; took[r + 1] = v.taken; gave[r + 1] = v.given; }
    }
    __syncthreads();
    int flags = sFlags;
    if (head < 0 || head >= p.nPages || count < 0 || count > p.nPages || carry.given > (unsigned)(p.nPages - max(0, min(count, p.nPages)))) flags |= PAGED_BAD_RING;
    if (carry.taken > (unsigned)max(count, 0)) flags |= PAGED_NO_PAGES;
    if (carry.rows > (unsigned)p.rows) flags |= PAGED_NO_ROWS;

    if (commit != 2) {
        for (int i = blockIdx.x * TABLE_ROWS + tid; i < min(p.rows, (int)(blockIdx.x + 1) * TABLE_ROWS); i += TB) {
            int slot = -1, pos = -1;
            if (!flags && (unsigned)i < carry.rows) {
                const int r = find(start, p.nReqs, (unsigned)i);
                const int len = p.lens[r];
                pos = len + i - (int)start[r];
                const int entry = pos >> p.pageShift, held = paged_pages(len, p.pageShift);
                int* at = p.table + (size_t)r * p.width + entry;
                int page;
                if (entry < held) page = *at;
                else {
                    long long e = (long long)head + took[r] + (unsigned)(entry - held);      // (below 2^32)
                    if (e >= p.nPages) e -= p.nPages;
                    page = p.ring[e];
                    if ((pos & ((1 << p.pageShift) - 1)) == 0) *at = page;
                }
                if (page >= 0 && page < p.nPages) slot = (page << p.pageShift) + (pos & ((1 << p.pageShift) - 1));
            }
            p.slots[i] = slot;
            p.positions[i] = pos;
        }
        if (!flags)
            for (unsigned i = blockIdx.x * TB + tid; i < carry.given; i += gridDim.x * TB) {
                const int r = find(gave, p.nReqs, i);
                long long e = (long long)head + count + i;
                while (e >= p.nPages) e -= p.nPages;
                p.ring[e] = p.table[(size_t)r * p.width + (i - gave[r])];
            }
    }
    if (commit == 0 || blockIdx.x != 0) return;
    __syncthreads();                        // every thread of this workgroup has read what lensOut and ringStateOut may go over
    for (int r = tid; r < p.nReqs; r += TB) {
        const int len = p.lens[r], add = p.newLens[r];
        p.lensOut[r] = flags ? len : add < 0 ? 0 : len + add;
    }
    for (int r = tid; r <= p.nReqs; r += TB) p.rowStart[r] = flags ? 0 : (int)start[r];
    if (tid == 0) {
        long long h = (long long)head + carry.taken;
        if (h >= p.nPages) h -= p.nPages;
        p.ringStateOut[0] = flags ? head : (int)h;
        p.ringStateOut[1] = flags ? count : count - (int)carry.taken + (int)carry.given;
        p.counts[0] = flags ? 0 : (int)carry.rows;
        p.counts[1] = flags ? 0 : (int)carry.taken;
        p.counts[2] = flags ? 0 : (int)carry.given;
        p.counts[3] = flags;
    }
}
hipError_t launch_paged_tables(const PagedTables& p, hipStream_t s) {
    const int groups = p.rows > TABLE_ROWS ? (p.rows + TABLE_ROWS - 1) / TABLE_ROWS : 1;
    const size_t lds = (size_t)(p.nReqs + 1) * 3 * sizeof(unsigned);
    // With one workgroup, or outputs apart from the inputs, the state is written by the launch that reads it; else by a second.
    const bool apart = p.lensOut + p.nReqs <= p.lens || p.lens + p.nReqs <= p.lensOut;
    const bool one = groups == 1 || (apart && (p.ringStateOut + 2 <= p.ringState || p.ringState + 2 <= p.ringStateOut));
    hipLaunchKernelGGL(paged_tables_kernel, dim3(groups), dim3(TB), lds, s, p, one ? 1 : 0);
    if (!one) hipLaunchKernelGGL(paged_tables_kernel, dim3(1), dim3(TB), lds, s, p, 2);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Rotary positions and K/V rows into their slots
//
// A workgroup a row: pairs (j, j + headDim/2) of q and k turned by the table row of the row's position, four pairs a thread, K and V
// rounded once to the cache's format (to nearest even).  Bound by HBM: every element is read once and written once (4,096 rows of
// the 8B shape, fp16: 28.9 us, 6.5 TB/s).
// ---------------------------------------------------------------------------
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void put4(float* d, float4 v) { *reinterpret_cast<float4*>(d) = v; }
__device__ __forceinline__ void put4(_Float16* d, float4 v) {
    half4_t h = {(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    *reinterpret_cast<half4_t*>(d) = h;
}
template <typename KVT>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedStore p) {
    const int t = blockIdx.x, pos = p.positions[t], slot = p.slots[t];
    if (pos < 0 || pos >= p.tableRows) return;
    const bool store = slot >= 0 && slot < p.nSlots;
    const int quarter = p.headDim / 8, kvDim = p.nKVHeads * p.headDim;       // groups of four pairs a head
    const float* c = p.cosTab + (size_t)pos * (p.headDim / 2);
    const float* s = p.sinTab + (size_t)pos * (p.headDim / 2);
    KVT* Kr = static_cast<KVT*>(p.K) + (size_t)(store ? slot : 0) * kvDim;
    KVT* Vr = static_cast<KVT*>(p.V) + (size_t)(store ? slot : 0) * kvDim;
    const int nq = p.nHeads * quarter, nk = p.nKVHeads * quarter;
    for (int i = threadIdx.x; i < nq + (store ? nk : 0); i += 256) {
        const int h = (i < nq ? i : i - nq) / quarter, j = ((i < nq ? i : i - nq) % quarter) * 4;
        const float* x = (i < nq ? p.q + (size_t)t * p.ldq : p.k + (size_t)t * p.ldk) + (size_t)h * p.headDim + j;
        const float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + p.headDim / 2);
        const float4 cc = *reinterpret_cast<const float4*>(c + j), ss = *reinterpret_cast<const float4*>(s + j);
        const float4 y = make_float4(a.x * cc.x - b.x * ss.x, a.y * cc.y - b.y * ss.y, a.z * cc.z - b.z * ss.z, a.w * cc.w - b.w * ss.w);
        const float4 z = make_float4(a.x * ss.x + b.x * cc.x, a.y * ss.y + b.y * cc.y, a.z * ss.z + b.z * cc.z, a.w * ss.w + b.w * cc.w);
        if (i < nq) {
            float* o = p.qOut + (size_t)t * p.ldqOut + (size_t)h * p.headDim + j;
            put4(o, y);
            put4(o + p.headDim / 2, z);
        } else {
            put4(Kr + (size_t)h * p.headDim + j, y);
            put4(Kr + (size_t)h * p.headDim + j + p.headDim / 2, z);
        }
    }
    if (store)
        for (int i = threadIdx.x; i < kvDim / 4; i += 256) put4(Vr + 4 * i, *reinterpret_cast<const float4*>(p.v + (size_t)t * p.ldv + 4 * i));
}
hipError_t launch_paged_store(const PagedStore& p, hipStream_t s) {
    if (p.rows <= 0) return hipSuccess;
    if (p.kvHalf) hipLaunchKernelGGL(paged_store_kernel<_Float16>, dim3(p.rows), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(paged_store_kernel<float>, dim3(p.rows), dim3(256), 0, s, p);
    return hipGetLastError();
}

// The device a handle's memory is on, for the duration of a call
struct OnDevice {
    int before = -1, want;
    hipError_t err;
    explicit OnDevice(int device) : want(device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != want) err = hipSetDevice(want);
    }
    ~OnDevice() { if (before >= 0 && before != want) (void)hipSetDevice(before); }
};

}  // namespace mg

struct mg_paged {
    mg::PagedGeo g;
    int device;
    char* mem;             // one allocation: zeros, what the plan is for, arrival counts, tiles, workers, partial results
    float* zeros;
    mg::PagedPlanFor* made;
    mg::PagedTile* tiles;
    mg::PagedWorker* workers;
    unsigned* arrived;
    float* parts;
    int maxTiles, maxWorkers;
    mg::PagedPlanFor plan;                     // the last plan asked for (nReqs < 0: none yet)
    int planWorkers, planWideWorkers;
};

namespace {
int refuse(const char* call, const char* why) {
    mg::set_error(std::string(call) + ": " + why);
    return MG_E_ARG;
}
int launched(const char* call, hipError_t e) {
    if (e == hipSuccess) return MG_OK;
    mg::set_error(std::string(call) + ": " + hipGetErrorString(e));
    (void)hipGetLastError();
    return MG_E_HIP;
}
}  // namespace

#define PAGED(h, call)                                                                     \
    if (!(h)) { mg::set_error(call ": NULL handle"); return MG_E_NOT_BUILT; }              \
    mg::OnDevice guard((h)->device);                                                       \
    if (guard.err != hipSuccess) return launched(call, guard.err)

extern "C" {

mg_paged* mg_paged_create(int nHeads, int nKVHeads, int headDim, int pageSize, int nPages, int kvFormat, int maxReqs, int maxRows, int maxLen) {
    mg::set_error("");
    mg::PagedGeo g{};
    if (const char* why = mg::paged_geo(g, nHeads, nKVHeads, headDim, pageSize, nPages, kvFormat, maxReqs, maxRows, maxLen)) {
        refuse("mg_paged_create", why);
        return nullptr;
    }
    int n = 0, device = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0 || hipGetDevice(&device) != hipSuccess) {
        (void)hipGetLastError();
        mg::set_error("mg_paged_create: no HIP device");
        return nullptr;
    }
    mg_paged* h = new (std::nothrow) mg_paged{};
    if (!h) { mg::set_error("mg_paged_create: out of host memory"); return nullptr; }
    h->g = g;
    h->device = device;
    h->plan.nReqs = -1;
    const size_t tiles = (size_t)mg::paged_max_tiles(g), workers = (size_t)std::max(mg::paged_workers(g, g.maxReqs, g.maxRows, false), mg::paged_workers(g, g.maxReqs, g.maxRows, true)), heads = (size_t)g.nKVHeads;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    const size_t oZeros = take((size_t)g.headDim * 4), oMade = take(sizeof(mg::PagedPlanFor)), oArrived = take(heads * tiles * 4), clear = at;      // (the part that starts as zeros)
    const size_t oTiles = take(2 * tiles * sizeof(mg::PagedTile)), oWorkers = take(2 * workers * sizeof(mg::PagedWorker));
    const size_t oParts = take(heads * workers * 2 * mg::paged_part_floats(g) * 4);
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&h->mem), at);
    if (e == hipSuccess) e = mg::launch_fill_zero(h->mem, clear, nullptr);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
    if (e == hipSuccess) e = mg::paged_attention_setup(g);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        mg::set_error("mg_paged_create: " + std::to_string(at) + " bytes of workspace: " + hipGetErrorString(e));
        mg_paged_destroy(h);
        return nullptr;
    }
    h->maxTiles = (int)tiles;
    h->maxWorkers = (int)workers;
    h->zeros = reinterpret_cast<float*>(h->mem + oZeros);
    h->made = reinterpret_cast<mg::PagedPlanFor*>(h->mem + oMade);
    h->arrived = reinterpret_cast<unsigned*>(h->mem + oArrived);
    h->tiles = reinterpret_cast<mg::PagedTile*>(h->mem + oTiles);
    h->workers = reinterpret_cast<mg::PagedWorker*>(h->mem + oWorkers);
    h->parts = reinterpret_cast<float*>(h->mem + oParts);
    return h;
}
void mg_paged_destroy(mg_paged* h) {
    if (!h) return;
    {
        mg::OnDevice guard(h->device);
        if (h->mem) (void)hipFree(h->mem);
    }
    delete h;
}
int mg_paged_table_width(const mg_paged* h) { return h ? h->g.width : 0; }

int mg_paged_tables(mg_paged* h, const int* newLens, int nReqs, const int* lens, int* lensOut, int* table, int* ring, const int* ringState,
                    int* ringStateOut, int rows, int* rowStart, int* slots, int* positions, int* counts, void* stream) {
    PAGED(h, "mg_paged_tables");
    if (const char* why = mg::paged_tables_refusal(h->g, newLens, nReqs, lens, lensOut, table, ring, ringState, ringStateOut, rows, rowStart, slots, positions, counts))
        return refuse("mg_paged_tables", why);
    if (const char* why = mg::paged_tables_overlap(h->g, newLens, nReqs, lens, lensOut, table, ring, ringState, ringStateOut, rows, rowStart, slots, positions, counts))
        return refuse("mg_paged_tables", why);
    mg::PagedTables p{newLens, lens, ringState, lensOut, table, ring, ringStateOut, rowStart, slots, positions, counts,
                      nReqs, rows, h->g.nPages, h->g.pageShift, h->g.width, h->g.maxLen};
    return launched("mg_paged_tables", mg::launch_paged_tables(p, static_cast<hipStream_t>(stream)));
}
int mg_paged_store(mg_paged* h, const float* q, const float* k, const float* v, int ldq, int ldk, int ldv, float* qOut, int ldqOut, void* K,
                   void* V, const int* slots, const int* positions, int rows, const float* cosTab, const float* sinTab, int tableRows, void* stream) {
    PAGED(h, "mg_paged_store");
    if (const char* why = mg::paged_store_refusal(h->g, q, k, v, ldq, ldk, ldv, qOut, ldqOut, K, V, slots, positions, rows, cosTab, sinTab, tableRows))
        return refuse("mg_paged_store", why);
    if (const char* why = mg::paged_store_overlap(h->g, q, k, v, ldq, ldk, ldv, qOut, ldqOut, K, V, rows)) return refuse("mg_paged_store", why);
    mg::PagedStore p{q, k, v, cosTab, sinTab, qOut, K, V, slots, positions, ldq, ldk, ldv, ldqOut, rows, tableRows,
                     h->g.nHeads, h->g.nKVHeads, h->g.headDim, h->g.kvHalf, h->g.nPages * h->g.pageSize};
    return launched("mg_paged_store", mg::launch_paged_store(p, static_cast<hipStream_t>(stream)));
}
int mg_paged_plan(mg_paged* h, const int* rowStart, const int* lens, int nReqs, int rows, int window, const int* prefixLens, void* stream) {
    PAGED(h, "mg_paged_plan");
    if (const char* why = mg::paged_plan_refusal(h->g, rowStart, lens, nReqs, rows, window, prefixLens)) return refuse("mg_paged_plan", why);
    const mg::PagedGeo& g = h->g;
    window = mg::paged_window(window, g.maxLen);
    const int workers = mg::paged_workers(g, nReqs, rows, false), narrow = mg::paged_narrow_rows(g, rows);
    const int wide = (long long)rows * g.group > narrow ? mg::paged_workers(g, nReqs, rows, true) : 0;
    mg::PagedPlan p{rowStart, lens, prefixLens, h->made, h->tiles, h->workers, nReqs, rows, window, g.maxLen, g.group, g.kvHalf, h->maxTiles, h->maxWorkers, workers, wide, narrow};
    const int rc = launched("mg_paged_plan", mg::launch_paged_plan(p, static_cast<hipStream_t>(stream)));
    if (rc == MG_OK) {
        h->plan = {nReqs, rows, window, 0}; h->planWorkers = workers; h->planWideWorkers = wide;
    }
    return rc;
}
int mg_paged_attention(mg_paged* h, const float* q, int ldq, const void* K, const void* V, const int* table, float* out, int ldo, float scale,
                       float softcap, const float* slopes, void* stream) {
    PAGED(h, "mg_paged_attention");
    if (h->plan.nReqs < 0) { mg::set_error("mg_paged_attention: no plan yet (mg_paged_plan)"); return MG_E_STATE; }
    if (h->plan.nReqs == 0 || h->plan.rows == 0) return MG_OK;
    if (const char* why = mg::paged_attention_refusal(h->g, q, ldq, K, V, table, out, ldo, scale, softcap, slopes)) return refuse("mg_paged_attention", why);
    if (const char* why = mg::paged_attention_overlap(h->g, q, ldq, K, V, out, ldo, h->plan.rows)) return refuse("mg_paged_attention", why);
    const mg::PagedGeo& g = h->g;
    mg::PagedAttention p{q, slopes, K, V, table, out, h->made, h->tiles, h->workers, h->parts, h->arrived, h->zeros, mg::paged_part_floats(g),
                         scale == 0.f ? 1.0f / std::sqrt((float)g.headDim) : scale, softcap, h->plan, ldq, ldo, h->plan.window, h->maxTiles, h->maxWorkers, h->planWorkers, h->planWideWorkers, g};
    return launched("mg_paged_attention", mg::launch_paged_attention(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
