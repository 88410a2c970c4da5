// paged.h -- a KV cache in pages that several requests share: the handle behind mg_paged and the launchers of its kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "paged_rules.h"

namespace mg {

struct PagedTables {
    const int *newLens, *lens, *ringState;
    int *lensOut, *table, *ring, *ringStateOut, *rowStart, *slots, *positions, *counts;
    int nReqs, rows, nPages, pageShift, width, maxLen;
};
hipError_t launch_paged_tables(const PagedTables& p, hipStream_t s);

struct PagedStore {
    const float *q, *k, *v, *cosTab, *sinTab;
    float* qOut;
    void *K, *V;
    const int *slots, *positions;
    int ldq, ldk, ldv, ldqOut, rows, tableRows, nHeads, nKVHeads, headDim, kvHalf, nSlots;
};
hipError_t launch_paged_store(const PagedStore& p, hipStream_t s);

// A worker's share [a, b) of the line, and the tile that it starts in
struct PagedWorker { PagedTile tile; int a, b, tiles, pad[13]; };
static_assert(sizeof(PagedTile) == 64 && sizeof(PagedWorker) == 128, "read as 16-byte words");

// What a plan was made for.  The places and numbers of its tiles and workers follow from these: an attention call works on the plan that is
// in the handle's memory only where they are its own (a graph's replay may have left another one there, or it was captured and has not run).
struct PagedPlanFor {
    int nReqs, rows, window, pad;
    MG_HD bool is(const PagedPlanFor& o) const { return ((nReqs ^ o.nReqs) | (rows ^ o.rows) | (window ^ o.window)) == 0; }      // (no branch between the loads)
};

// The plan that a step's attention calls share.
struct PagedPlan {
    const int *rowStart, *lens, *prefixLens;      // the caller's
    PagedPlanFor* made;                           // the handle's
    PagedTile* tiles;                             // maxTiles of them, for narrow tiles and again for wide ones,
    PagedWorker* workers;                         // and maxWorkers of these
    int nReqs, rows, window, maxLen, group, kvHalf, maxTiles, maxWorkers, nWorkers, wideWorkers, narrowRows;      // wideWorkers 0: no wide tiles
};
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s);

struct PagedAttention {
    const float *q, *slopes;
    const void *K, *V;
    const int* table;
    float* out;
    const PagedPlanFor* made;
    const PagedTile* tiles;    // narrow tiles' and wide ones', maxTiles and maxWorkers apart, as in the plan
    const PagedWorker* workers;
    float* parts;              // partial results: two of every worker and KV head
    unsigned* arrived;         // how many workers are done with a tile, [KV head][tile]; zeros between calls
    const float* zeros;        // headDim zeros: what a position outside a tile's, or on a page that is gone, is read from
    size_t partStride;
    float scale, softcap;
    PagedPlanFor plan;
    int ldq, ldo, window, maxTiles, maxWorkers, nWorkers, wideWorkers;
    PagedGeo g;
};
size_t paged_part_floats(const PagedGeo& g);
int paged_max_tiles(const PagedGeo& g);
int paged_workers(const PagedGeo& g, int nReqs, int rows, bool wide);       // workers a KV head
int paged_narrow_rows(const PagedGeo& g, int rows);              // requests of up to so many rows a KV head have narrow tiles
hipError_t paged_attention_setup(const PagedGeo& g);
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t s);

}  // namespace mg
