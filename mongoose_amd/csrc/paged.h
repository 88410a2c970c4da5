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
    int ldq, ldk, ldv, ldqOut, rows, tableRows, nHeads, nKVHeads, headDim, kvFormat, nSlots, pageShift;
};
hipError_t launch_paged_store(const PagedStore& p, hipStream_t s);

struct PagedLoad {
    const void *K, *V;
    const int *table, *rowStart, *lens;
    float *kOut, *vOut;
    int nReqs, rows, ldk, ldv;
    int row0;                  // a launch's first row
    PagedGeo g;
};
hipError_t launch_paged_load(const PagedLoad& p, hipStream_t s);

// A worker's share [a, b) of the line, and the tile that it starts in
struct PagedWorker { PagedTile tile; int a, b, tiles, pad[13]; };
static_assert(sizeof(PagedTile) == 64 && sizeof(PagedWorker) == 128, "read as 16-byte words");

// The plan that a step's attention calls share.
struct PagedPlan {
    const int *rowStart, *lens, *prefixLens;      // the caller's
    const int4* given;                            // or, with shared prefixes, what paged_groups_kernel has made of them
    const int* groupOf;                           // ... and the requests' groups,
    int* groupTile;                               // or, where `given` are groups: takes each one's first tile, and behind the last how many there are
    PagedPlanFor* made;                           // the handle's
    PagedTile* tiles;                             // maxTiles of them, for narrow tiles and again for wide ones,
    PagedWorker* workers;                         // and maxWorkers of these
    int nReqs, rows, window, maxLen, group, kvFormat, maxTiles, maxWorkers, nWorkers, wideWorkers, narrowRows;      // wideWorkers 0: no wide tiles
    PagedPlanFor plan;
};
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s);

// Groups of requests with the same first positions: what the two plans (the groups' shared positions, and every request's own) go by.
struct PagedGroups {
    const int *rowStart, *lens, *groupStart, *sharedLens;      // the caller's
    int4* reqs;          // of every request: first row, rows, length, first position of its own
    int* groupOf;        // its group
    int4* groups;        // of every group: first row, rows, shared positions, the request whose pages are read
    int nReqs, rows, nGroups, maxLen;
};
hipError_t launch_paged_plan_shared(const PagedGroups& g, const PagedPlan& shared, const PagedPlan& own, hipStream_t s);

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
    // Shared prefixes: a call's first pass leaves its workers' shares of the groups' tiles as they are, and its second one, over the requests' own
    // positions, takes those of its rows in.
    int pass;                  // 0: no prefix is shared; 1, 2
    const int4 *reqs, *groups; // as in PagedGroups
    const int* groupTile;
    const PagedTile* sharedTiles;
    const float* sharedParts;
    int sharedPlaces, sharedRows;        // of the first pass: shares a KV head (paged_place), rows of a tile
    int ldq, ldo, window, maxTiles, maxWorkers, nWorkers, wideWorkers;
    PagedGeo g;
};
size_t paged_part_floats(const PagedGeo& g);
int paged_max_tiles(const PagedGeo& g);
int paged_max_tiles_shared(const PagedGeo& g);
bool paged_shared_twice(const PagedGeo& g, int nReqs, int rows, bool groups);
int paged_workers(const PagedGeo& g, int nReqs, int rows, bool wide, bool twice = false);       // workers a KV head
hipError_t paged_attention_setup(const PagedGeo& g);
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t s);

}  // namespace mg
