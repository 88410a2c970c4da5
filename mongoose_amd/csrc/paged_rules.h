// paged_rules.h -- what the calls on a paged KV cache accept and which positions a token sees.  Plain C++, shared by the host
// side, the kernels and the CPU tests.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define MG_HD __host__ __device__ __forceinline__
#else
#define MG_HD inline
#endif

namespace mg {

// Limits of a handle: the block-table kernel holds three sums a request in LDS (48 KB); a distance between positions is exact in
// fp32; a page holds whole runs of eight positions, the finest run that the attention looks up a page for.
constexpr int PAGED_MAX_REQS = 4096, PAGED_MAX_LEN = 1 << 24, PAGED_MAX_ROWS = 1 << 20, PAGED_MIN_PAGE = 8, PAGED_MAX_PAGE = 4096, PAGED_MAX_GROUP = 128;

// Formats of a cache: fp32, fp16, or Q8 -- an int8 an element and an fp32 scale a KV head's row (the row's greatest size / 127).  A Q8
// pool holds its int8 rows [slots, kvDim], then the scales [pages, KV heads, pageSize]: those of a KV head's positions lie side by side,
// as the attention reads them.
enum { PAGED_F32 = 0, PAGED_F16 = 1, PAGED_Q8 = 8 };

struct PagedGeo {
    int nHeads, nKVHeads, headDim, pageSize, nPages, kvFormat, maxReqs, maxRows, maxLen;
    int group;        // query heads a KV head
    int kvDim;        // elements of a position's K (or V) row
    int pageShift;    // log2(pageSize)
    int width;        // entries of a request's row of the block table
};

// nullptr, or why there is no such handle
inline const char* paged_geo(PagedGeo& g, int nHeads, int nKVHeads, int headDim, int pageSize, int nPages, int kvFormat, int maxReqs,
                             int maxRows, int maxLen) {
    if (headDim != 64 && headDim != 128) return "headDim must be 64 or 128";
    if (nKVHeads <= 0 || nHeads <= 0 || nHeads % nKVHeads != 0) return "nHeads must be a positive multiple of nKVHeads";
    if (nHeads / nKVHeads > PAGED_MAX_GROUP || nHeads > 65536) return "at most 128 query heads a KV head and 65536 in all";
    if (pageSize < PAGED_MIN_PAGE || pageSize > PAGED_MAX_PAGE || (pageSize & (pageSize - 1))) return "pageSize must be a power of two from 8 to 4096";
    if (nPages <= 0 || (long long)nPages * pageSize > 0x7fffffffll) return "nPages must be positive and nPages * pageSize below 2^31";
    if (kvFormat != PAGED_F32 && kvFormat != PAGED_F16 && kvFormat != PAGED_Q8) return "kvFormat must be 0 (fp32), 1 (fp16) or 8 (Q8)";
    if (maxReqs <= 0 || maxReqs > PAGED_MAX_REQS) return "maxReqs must be between 1 and 4096";
    if (maxRows <= 0 || maxRows > PAGED_MAX_ROWS) return "maxRows must be between 1 and 2^20";
    if (maxLen <= 0 || maxLen > PAGED_MAX_LEN) return "maxLen must be between 1 and 2^24";
    if ((long long)maxRows * (nHeads / nKVHeads) > (1ll << 40) / maxLen) return "maxRows * (nHeads / nKVHeads) * maxLen must be at most 2^40";
    if ((long long)maxReqs * maxLen > (1ll << 34)) return "maxReqs * maxLen must be at most 2^34";
    g.nHeads = nHeads; g.nKVHeads = nKVHeads; g.headDim = headDim; g.pageSize = pageSize; g.nPages = nPages; g.kvFormat = kvFormat;
    g.maxReqs = maxReqs; g.maxRows = maxRows; g.maxLen = maxLen;
    g.group = nHeads / nKVHeads;
    g.kvDim = nKVHeads * headDim;
    g.pageShift = 0;
    while ((1 << g.pageShift) < pageSize) g.pageShift++;
    g.width = (maxLen + pageSize - 1) / pageSize;
    return nullptr;
}

inline bool paged_aligned(const void* p, size_t a) { return p != nullptr && ((uintptr_t)p & (a - 1)) == 0; }

// The arguments of the calls: nullptr, or what is wrong with them.
inline const char* paged_tables_refusal(const PagedGeo& g, const void* newLens, int nReqs, const void* lens, const void* lensOut,
                                        const void* table, const void* ring, const void* ringState, const void* ringStateOut, int rows,
                                        const void* rowStart, const void* slots, const void* positions, const void* counts) {
    if (nReqs < 0 || nReqs > g.maxReqs) return "nReqs is negative or above the handle's maxReqs";
    if (rows < 0 || rows > g.maxRows) return "rows is negative or above the handle's maxRows";
    const void* always[] = {ring, ringState, ringStateOut, rowStart, counts};
    for (const void* p : always) if (!paged_aligned(p, 4)) return "a pointer is NULL or not aligned to 4 bytes";
    if (nReqs > 0) {
        const void* reqs[] = {newLens, lens, lensOut, table};
        for (const void* p : reqs) if (!paged_aligned(p, 4)) return "a pointer is NULL or not aligned to 4 bytes";
        if (newLens == lensOut) return "newLens and lensOut are the same array";
    }
    if (rows > 0 && (!paged_aligned(slots, 4) || !paged_aligned(positions, 4))) return "a pointer is NULL or not aligned to 4 bytes";
    return nullptr;
}
inline const char* paged_store_refusal(const PagedGeo& g, const void* q, const void* k, const void* v, int ldq, int ldk, int ldv,
                                       const void* qOut, int ldqOut, const void* K, const void* V, const void* slots,
                                       const void* positions, int rows, const void* cosTab, const void* sinTab, int tableRows) {
    if (rows < 0 || rows > g.maxRows) return "rows is negative or above the handle's maxRows";
    if (rows == 0) return nullptr;
    const void* wide[] = {q, k, v, qOut, K, V, cosTab, sinTab};
    for (const void* p : wide) if (!paged_aligned(p, 16)) return "a pointer is NULL or not aligned to 16 bytes";
    if (!paged_aligned(slots, 4) || !paged_aligned(positions, 4)) return "a pointer is NULL or not aligned to 4 bytes";
    if (ldq < g.nHeads * g.headDim || ldqOut < g.nHeads * g.headDim || ldk < g.kvDim || ldv < g.kvDim) return "a row stride is smaller than the row";
    if ((ldq | ldk | ldv | ldqOut) & 3) return "a row stride is not a multiple of 4";
    if (tableRows <= 0) return "the rotary tables have no rows";
    if (K == V) return "K and V are the same array";
    return nullptr;
}
// What the block-table kernel writes while others of its workgroups still read: nullptr, or that two of its arrays overlap.  The lengths
// and the ring's state may be updated in place.
inline const char* paged_tables_overlap(const PagedGeo& g, const int* newLens, int nReqs, const int* lens, const int* lensOut, const int* table,
                                        const int* ring, const int* ringState, const int* ringStateOut, int rows, const int* rowStart,
                                        const int* slots, const int* positions, const int* counts) {
    const struct { const int* p; long long n; } a[] = {
        {lensOut, nReqs}, {ringStateOut, 2}, {table, (long long)nReqs * g.width}, {ring, g.nPages}, {rowStart, nReqs + 1}, {slots, rows},
        {positions, rows}, {counts, 4}, {newLens, nReqs}, {lens, nReqs}, {ringState, 2}};
    for (int i = 0; i < 8; i++)             // (the first eight are written)
        for (int j = i + 1; j < 11; j++) {
            if (a[i].p == a[j].p && ((i == 0 && j == 9) || (i == 1 && j == 10))) continue;
            if (a[i].n > 0 && a[j].n > 0 && (uintptr_t)a[i].p < (uintptr_t)(a[j].p + a[j].n) && (uintptr_t)a[j].p < (uintptr_t)(a[i].p + a[i].n))
                return "arrays overlap (lensOut may be lens, ringStateOut ringState)";
        }
    return nullptr;
}
// Arrays of `rows` rows of `width` floats, `ld` floats apart (a row no longer than that): whether they have a float in common.  Rows of
// one stride may lie between each other (columns of one projection); of two strides, anything between the first and last float counts.
inline bool paged_rows_meet(const void* a, int lda, int wa, const void* b, int ldb, int wb, int rows) {
    const long long d = ((long long)(intptr_t)b - (long long)(intptr_t)a) / 4;        // (both are aligned to 16 bytes)
    if (rows <= 0) return false;
    if (lda != ldb) return d < (long long)(rows - 1) * lda + wa && -d < (long long)(rows - 1) * ldb + wb;
    // rows k apart meet where -wb < d + k ld < wa, -rows < k < rows; of the numbers d + k ld only those within ld of 0 can
    long long r = d % lda;                       // (as d / lda, towards 0)
    const long long k = -(d / lda);
    for (int i = -1; i <= 1; i++) {
        const long long at = r + (long long)i * lda;
        if (at < wa && -at < wb && k + i > -rows && k + i < rows) return true;
    }
    return false;
}
// Whether `bytes` at p and the floats of such rows have memory in common
inline bool paged_pool_meets(const void* p, size_t bytes, const void* a, int ld, int width, int rows) {
    const uintptr_t x = (uintptr_t)p, y = (uintptr_t)a;
    return rows > 0 && x < y + ((size_t)(rows - 1) * ld + width) * 4 && y < x + bytes;
}
inline size_t paged_element_bytes(int kvFormat) { return kvFormat == PAGED_F32 ? 4 : kvFormat == PAGED_F16 ? 2 : 1; }
inline size_t paged_pool_bytes(const PagedGeo& g) {
    const size_t slots = (size_t)g.nPages * g.pageSize;
    return slots * g.kvDim * paged_element_bytes(g.kvFormat) + (g.kvFormat == PAGED_Q8 ? slots * g.nKVHeads * 4 : 0);
}
// What a call writes while others of its workgroups still read it: nullptr, or which of its arguments overlap (those that
// paged_store_refusal has passed).
inline const char* paged_store_overlap(const PagedGeo& g, const void* q, const void* k, const void* v, int ldq, int ldk, int ldv,
                                       const void* qOut, int ldqOut, const void* K, const void* V, int rows) {
    if (rows == 0) return nullptr;
    const int qw = g.nHeads * g.headDim;
    if (!(q == qOut && (ldq == ldqOut || rows == 1)) && paged_rows_meet(q, ldq, qw, qOut, ldqOut, qw, rows)) return "qOut overlaps q, and is not q with the same stride";
    if (paged_rows_meet(k, ldk, g.kvDim, qOut, ldqOut, qw, rows) || paged_rows_meet(v, ldv, g.kvDim, qOut, ldqOut, qw, rows)) return "qOut overlaps k or v";
    const size_t bytes = paged_pool_bytes(g);
    if ((uintptr_t)K < (uintptr_t)V + bytes && (uintptr_t)V < (uintptr_t)K + bytes) return "K and V overlap";
    const void* pools[] = {K, V};
    for (const void* p : pools)
        if (paged_pool_meets(p, bytes, q, ldq, qw, rows) || paged_pool_meets(p, bytes, k, ldk, g.kvDim, rows) ||
            paged_pool_meets(p, bytes, v, ldv, g.kvDim, rows) || paged_pool_meets(p, bytes, qOut, ldqOut, qw, rows)) return "K or V overlaps the rows";
    return nullptr;
}
inline const char* paged_load_refusal(const PagedGeo& g, const void* K, const void* V, const void* table, const void* rowStart, const void* lens,
                                      int nReqs, int rows, const void* kOut, int ldk, const void* vOut, int ldv) {
    if (nReqs < 0 || nReqs > g.maxReqs) return "nReqs is negative or above the handle's maxReqs";
    if (rows < 0) return "rows is negative";
    if (nReqs == 0 || rows == 0) return nullptr;
    const void* wide[] = {K, V, kOut, vOut};
    for (const void* p : wide) if (!paged_aligned(p, 16)) return "a pointer is NULL or not aligned to 16 bytes";
    const void* ints[] = {table, rowStart, lens};
    for (const void* p : ints) if (!paged_aligned(p, 4)) return "a pointer is NULL or not aligned to 4 bytes";
    if (ldk < g.kvDim || ldv < g.kvDim) return "a row stride is smaller than the row";
    if ((ldk | ldv) & 3) return "a row stride is not a multiple of 4";
    return nullptr;
}
// What mg_paged_load writes while others of its workgroups still read
inline const char* paged_load_overlap(const PagedGeo& g, const void* K, const void* V, const void* table, const void* rowStart, const void* lens, int nReqs,
                                      int rows, const void* kOut, int ldk, const void* vOut, int ldv) {
    if (nReqs == 0 || rows == 0) return nullptr;
    if (paged_rows_meet(kOut, ldk, g.kvDim, vOut, ldv, g.kvDim, rows)) return "kOut overlaps vOut";
    const size_t bytes = paged_pool_bytes(g);
    const struct { const void* p; size_t n; } in[] = {{K, bytes}, {V, bytes}, {table, (size_t)nReqs * g.width * 4}, {rowStart, ((size_t)nReqs + 1) * 4}, {lens, (size_t)nReqs * 4}};
    for (auto& a : in)
        if (paged_pool_meets(a.p, a.n, kOut, ldk, g.kvDim, rows) || paged_pool_meets(a.p, a.n, vOut, ldv, g.kvDim, rows)) return "kOut or vOut overlaps what is read";
    return nullptr;
}
inline const char* paged_plan_refusal(const PagedGeo& g, const void* rowStart, const void* lens, int nReqs, int rows, int window,
                                      const void* prefixLens) {
    if (nReqs < 0 || nReqs > g.maxReqs) return "nReqs is negative or above the handle's maxReqs";
    if (rows < 0 || rows > g.maxRows) return "rows is negative or above the handle's maxRows";
    if (window < 0) return "window is negative";
    if (!paged_aligned(rowStart, 4) || (nReqs > 0 && !paged_aligned(lens, 4))) return "a pointer is NULL or not aligned to 4 bytes";
    if (prefixLens && !paged_aligned(prefixLens, 4)) return "prefixLens is not aligned to 4 bytes";
    return nullptr;
}
inline const char* paged_plan_shared_refusal(const PagedGeo& g, const void* rowStart, const void* lens, int nReqs, int rows, int mostNew,
                                             const void* groupStart, const void* sharedLens, int nGroups) {
    if (const char* why = paged_plan_refusal(g, rowStart, lens, nReqs, rows, 0, nullptr)) return why;
    if (mostNew < 0) return "mostNew is negative";
    if (nGroups < 0 || nGroups > g.maxReqs) return "nGroups is negative or above the handle's maxReqs";
    if (nGroups > 0 && (!paged_aligned(groupStart, 4) || !paged_aligned(sharedLens, 4))) return "a pointer is NULL or not aligned to 4 bytes";
    return nullptr;
}
inline const char* paged_attention_refusal(const PagedGeo& g, const void* q, int ldq, const void* K, const void* V, const void* table,
                                           const void* out, int ldo, float scale, float softcap, const void* slopes) {
    const void* wide[] = {q, K, V, out};
    for (const void* p : wide) if (!paged_aligned(p, 16)) return "a pointer is NULL or not aligned to 16 bytes";
    if (!paged_aligned(table, 4) || (slopes && !paged_aligned(slopes, 4))) return "a pointer is NULL or not aligned to 4 bytes";
    if (ldq < g.nHeads * g.headDim || ldo < g.nHeads * g.headDim) return "a row stride is smaller than the row";
    if ((ldq | ldo) & 3) return "a row stride is not a multiple of 4";
    // (beyond these the scale in powers of two, or the cap's reciprocal, is no normal fp32 number; the power of two that an fp16 cache's
    // rows of q take besides is kept from making it one: power_up)
    if (!(scale == 0.f || (scale >= 1e-30f && scale <= 1e30f))) return "scale must be between 1e-30 and 1e30, or 0 for 1 / sqrt(headDim)";
    if (!(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f))) return "softcap must be between 1e-30 and 1e30, or 0 for none";
    if (q == out) return "q and out are the same array";
    return nullptr;
}

inline const char* paged_attention_overlap(const PagedGeo& g, const void* q, int ldq, const void* K, const void* V, const void* out, int ldo, int rows) {
    const int w = g.nHeads * g.headDim;
    if (paged_rows_meet(q, ldq, w, out, ldo, w, rows)) return "out overlaps q";
    const size_t bytes = paged_pool_bytes(g);
    if (paged_pool_meets(K, bytes, out, ldo, w, rows) || paged_pool_meets(V, bytes, out, ldo, w, rows)) return "out overlaps K or V";
    return nullptr;
}

// Sums that stop at 2^31 - 1 instead of wrapping (still associative): an overflowing total is only ever compared with a limit.
MG_HD unsigned sat_add(unsigned a, unsigned b) {
    const unsigned s = a + b;            // both below 2^31
    return s > 0x7fffffffu ? 0x7fffffffu : s;
}
MG_HD int paged_pages(int len, int pageShift) { return (int)(((unsigned)len + (1u << pageShift) - 1) >> pageShift); }
// A window as the calls below take it: none is wider than all positions (a difference from a row's position, which is negative where a
// request has more rows than positions, stays a number).
MG_HD int paged_window(int window, int maxLen) { return window < maxLen ? window : maxLen; }
// Whether the token at position i of a request of `len` positions sees position j.
MG_HD bool paged_sees(int i, int j, int len, int window, int prefix) {
    return (j < len) & (((j <= i) & ((window == 0) | (j > i - window))) | (j < prefix));
}

// Whether any token at positions first .. last may see any of the positions [begin, end)
MG_HD bool paged_some_see(int first, int last, int begin, int end, int window, int prefix) {
    return begin < prefix || (begin <= last && (window == 0 || end > first - window + 1));
}

// ---------------------------------------------------------------------------
// The plan of an attention call.  The rows of a request under one KV head (its new tokens x the head group, token by token) are cut
// into tiles of tileRows, the positions a tile sees into units of unitKeys.  All tiles of a batch, one behind the other, make a line
// of cost: PAGED_TILE_COST for a tile's own start and end, then 1 for each of its units.  Workers get shares [a, b) of the line, the same
// for every KV head.  Where there are many tiles the shares are equal and pass over from tile to tile: any mix of long, short, one
// and many requests keeps every CU busy to the end.  Where there are few, every tile has workers of its own, as many as its part of
// the cost asks for, so that none has the start and the end of two tiles behind each other.  A tile with several workers
// is put together by the last of them to finish.
// ---------------------------------------------------------------------------
constexpr int PAGED_TILE_COST = 1;
constexpr int PAGED_NARROW = 16, PAGED_WIDE = 128;        // rows of a tile

struct PagedTile {
    int req, row0, rows, len, prefix;   // the request, its first row and number of rows in the batch, its length and prefix
    int first;                          // the tile's first row among the request's rows x group
    int cost0;                          // where the tile starts on the line
    int unit0, units;                   // the units it sees
    int worker0, worker1;               // the first and last worker that have some of them
    int index;                          // its number
    int tileRows, unitKeys;             // its kind
    int from, group;                    // the first position that is its own -- those before are shared --, and the group that shares them
};

// The positions [begin, end) that rows first .. first + tileRows - 1 of a request see some of, and the positions of its first and last token.
struct PagedSpan { int begin, end, pos0, pos1; };
MG_HD PagedSpan paged_span(int rows, int len, int prefix, int window, int group, int first, int tileRows, int from = 0) {
    const int all = rows * group;
    const int last = (first + tileRows < all ? first + tileRows : all) - 1;
    PagedSpan s;
    s.pos0 = len - rows + first / group;
    s.pos1 = len - rows + last / group;
    s.end = s.pos1 + 1 > prefix ? s.pos1 + 1 : prefix;
    s.begin = window > 0 && prefix == 0 && s.pos0 - window + 1 > 0 ? s.pos0 - window + 1 : 0;
    if (s.begin < from) s.begin = from;
    return s;
}
MG_HD void paged_units(PagedTile& t, int window, int group) {
    const PagedSpan s = paged_span(t.rows, t.len, t.prefix, window, group, t.first, t.tileRows, t.from);
    t.unit0 = s.begin / t.unitKeys;
    t.units = s.end > s.begin ? (s.end + t.unitKeys - 1) / t.unitKeys - t.unit0 : 0;
}
MG_HD int paged_cost(const PagedTile& t) { return PAGED_TILE_COST + t.units; }
// Many tiles: where worker w's share of a line of `cost` starts, and the worker whose share x is in (workers <= cost, so that no
// share is empty).
MG_HD int paged_share(int cost, int workers, int w) { return (int)((long long)cost * w / workers); }
MG_HD int paged_worker_of(int cost, int workers, int x) { return (int)((((long long)x + 1) * workers - 1) / cost); }
// Few tiles: how many workers a tile has -- at least one, together at most `workers`, and units of `least` and more each -- and where
// the share of its i-th of n starts.
// (Half as many tiles as workers at most.  Up to as many would spare more tiles a second owner -- 8B shape, four of 345 to 467 rows, window,
// cap: 131 us, with that 113; fresh prompts of 340, 359, 316 rows fp16 51 and 33, of 1,512 and 1,576 rows 134 and 139 -- a quarter is the same
// but for 12 requests, three of 165 to 235 rows: 92 us, 94.)
MG_HD bool paged_few(int tiles, int workers) { return 2 * tiles <= workers; }
MG_HD int paged_workers_for(const PagedTile& t, int cost, int tiles, int workers, int least) {
    const int most = t.units / least > 1 ? t.units / least : 1;
    const int n = 1 + (int)((long long)(workers - tiles) * paged_cost(t) / cost);
    return n < most ? n : most;
}
MG_HD int paged_part(const PagedTile& t, int n, int i) {
    return i == 0 ? t.cost0 : t.cost0 + PAGED_TILE_COST + (int)((long long)t.units * i / n);
}
// The share that worker w leaves of a group's tile i, of those that a KV head has.  With shared prefixes every worker leaves one of every tile
// that it has part of, the only one of a tile as well, so that there may be any number of a worker's.  Along the line either the tile or the
// worker steps on from a share to the next, so no two have the same sum of their numbers.
MG_HD int paged_place(int tile, int worker) { return tile + worker; }
// The tiles that groups' rows may have (wide: one a group more than there are whole ones; narrow: for up to 256 rows): a group that shares
// anything has two requests with rows.
inline int paged_group_tiles(const PagedGeo& g) {
    const int requests = g.maxReqs < g.maxRows ? g.maxReqs : g.maxRows;
    return (int)((long long)g.maxRows * g.group / PAGED_WIDE) + 256 / PAGED_NARROW + requests / 2;
}
// The first unit of a tile that starts at `a` on the line or behind.
MG_HD int paged_unit_at(const PagedTile& t, int a) {
    const int u = a - (t.cost0 + PAGED_TILE_COST);
    return u <= 0 ? 0 : u < t.units ? u : t.units;
}

// Rows a KV head (tokens x group) up to which a request goes to the kernel that waits for memory, with longer ones to the one that waits for
// the matrix units.  8B shape:
//   A batch of up to 256 rows: all narrow, which reads K and V once for 16 rows, but in one launch.  One request of 8, 16, 32 and 64 tokens
//   over 16,000 positions: fp16 33, 41, 64, 112 us, wide 83, 89, 103, 105; fp32 43, 66, 117, 220, wide 338, 380, 401, 317.
//   Larger batches: narrow up to 16 rows.  24 requests of 5, 8, 12 tokens over 500 to 4,000 positions, fp16: 77, 78, 80 us wide, 75, 81, 99
//   narrow, and 96 requests of 5 tokens 208 wide, 304 narrow.  With an fp32 cache narrow tiles would be better there, up to 64 rows (228,
//   204, 385, and with 16 tokens 361 us wide; 169, 141, 249, 276 narrow): its wide tiles wait for the fp32 instructions of rows that are not there.
//   Q8: a wide tile also has its rows turned to halves for rows that are not there, so narrow ones go further: 24 requests of 5, 8, 12, 16 tokens
//   as above 98, 90, 104, 113 us wide, 59, 55, 69, 90 narrow; 1.1B shape, 5 tokens 62 and 41.  With many requests, whose wide tiles fill the
//   CUs, up to 32 rows: 96 requests of 5, 8, 16 tokens 233, 231, 299 and 203, 209, 405; 1.1B shape, 8 tokens 115 and 138.
constexpr int NARROW_Q8_FEW = 64, NARROW_Q8 = 32, Q8_FEW_ROWS = 4096;
inline int paged_narrow_rows(const PagedGeo& g, int rows) {
    const long long all = (long long)rows * g.group;
    if (all <= 256) return 256;
    return g.kvFormat != PAGED_Q8 ? PAGED_NARROW : all <= Q8_FEW_ROWS ? NARROW_Q8_FEW : NARROW_Q8;
}
// The same with shared prefixes, for groups (0: all groups have wide tiles; up to 256 rows, as above: 64 requests behind 8,001 positions 98 us, with
// wide ones 133) and for requests, of which the caller may know that none adds more than mostNew rows.  What requests have of their own is short, so
// narrow tiles go further while the wide ones would not fill the CUs (80 requests, 378 rows in all, up to 40 each, Q8: 210 us a call, so 163; 32 of
// 40 rows each, more rows than that: 219 and 235).
inline int paged_narrow_rows_shared(const PagedGeo& g, int rows, int mostNew, bool groups) {
    constexpr int ALL = PAGED_MAX_ROWS * PAGED_MAX_GROUP;
    if ((long long)rows * g.group <= 256) return ALL;
    if (groups) return 0;
    const int narrow = (long long)rows * g.group <= 4096 ? 256 : paged_narrow_rows(g, rows);
    return mostNew > 0 && (long long)mostNew * g.group <= narrow ? ALL : narrow;
}
// What a plan was made for.  The places, numbers and kinds of its tiles and workers follow from these: an attention call works on the plan that is
// in the handle's memory only where they are its own (a graph's replay may have left another one there, or it was captured and has not run).
struct PagedPlanFor {
    int nReqs, rows, window, groups;
    int narrowRows;        // requests of up to so many rows a KV head have narrow tiles: what the caller knows of the rows is in it
    MG_HD bool is(const PagedPlanFor& o) const {
        return ((nReqs ^ o.nReqs) | (rows ^ o.rows) | (window ^ o.window) | (groups ^ o.groups) | (narrowRows ^ o.narrowRows)) == 0;      // (no branch between the loads)
    }
};

// Why mg_paged_tables changes nothing
enum { PAGED_NO_PAGES = 1, PAGED_NO_ROWS = 2, PAGED_BAD_LENGTH = 4, PAGED_BAD_RING = 8 };

}  // namespace mg
