// Attention of new tokens over a paged cache: the problem as its kernels see
// it, and how a workgroup finds its share of it.
//
// Sequence b holds `len` tokens of which the last n are new; token i of them
// is at position p = len - n + i.  Its keys are p - t d, t < K (all of 0..p
// without a window).  With a dilation d, tokens i, i + d, ... are one class:
// their positions share a residue c mod d, and in class coordinates
// u = (j - c) / d a window is the run [w - K + 1, w], w the query's own
// coordinate.  Rows of work are (member of a class, query head of the kv
// head's group), members slowest; a tile is M consecutive rows of one class,
// so its keys are one run of u, staged once for all its rows.
//
// Few rows and long caches: the run of a tile is cut into chunks, one
// workgroup each, joined by k_paged_join.  The lengths are on the device
// only, so each workgroup works out the cut itself (`find_share`): the key
// blocks of all tiles over the workgroups aimed at give the chunk.
#pragma once

#include "na_launch.h"

namespace na {

namespace {

constexpr int kPagedThreads = 256;

struct PagedArgs {
    const void* q;
    void* out;
    float* lse;
    const void *k, *v;
    Lay lq, lo, ll;  // b, s2 (token), h
    long long kp, ks, kh, vp, vs, vh;
    const int *table, *lens, *news;
    long long table_stride;
    int width, pages, page_size;
    FastDiv fpage;
    int B, L, Hq, Hkv, rep, Dqk, Dv;
    FastDiv frep;
    int K, dil;  // K 0: no window
    FastDiv fdil;
    float scale;
    int M, KT;           // rows of a tile, keys of a block
    int tile_slots;      // tiles of a (sequence, kv head) at most
    int direct;          // every tile whole: slot = tile, nothing to work out
    int target;          // workgroups aimed at when tiles are few
    int least;           // key blocks of a chunk at least
    int xcd_run;         // consecutive shares of one XCD (0: as dealt)
    FastDiv fslots, fkv, frun;
    // split tiles: header (count of tiles), a record per tile, m and l, O
    int* count;
    struct PagedTile* tiles;
    float* ml;    // [share][M][2]
    float* part;  // [share][M][Dv]
};

// A split tile: where its parts are, and which rows it holds.
struct PagedTile {
    int first, step, parts;  // parts first, first + step, ...
    int b, h, cls, row0, rows;
};

struct SeqGeo {
    int n, len, classes, tiles, blocks;  // tiles: of all its classes, one kv head
};

// ceil(a / b) of a >= 0 for any b >= 1 (a dilation may be as large as an int).
__device__ __forceinline__ int ceil_div(int a, int b) { return a > 0 ? (a - 1) / b + 1 : 0; }

__device__ __forceinline__ SeqGeo seq_geo(const PagedArgs& a, int b) {
    SeqGeo g;
    g.n = a.news ? imin(imax(a.news[b], 0), a.L) : a.L;
    g.len = imax(a.lens[b], 0);
    g.classes = imin(g.n, a.dil);
    const int members = ceil_div(g.n, a.dil);
    const int per_class = ceil_div(members * a.rep, a.M);
    g.tiles = g.classes * per_class;
    const long long cap = static_cast<long long>(a.width) * a.page_size;
    long long keys = (g.len < cap ? g.len : cap) / a.dil + 1;
    if (a.K) {
        const long long span = static_cast<long long>(a.K) + imin(members, a.M / a.rep + 2) - 1;
        if (span < keys) keys = span;
    }
    g.blocks = static_cast<int>((keys + a.KT - 1) / a.KT);
    return g;
}

// A workgroup's share: keys [u_lo, u_hi] (class coordinates) of one tile.
struct Share {
    int b, h, cls, c;         // class: its first token, its residue
    int row0, rows;
    int w0;                   // class coordinate of member 0
    int u_lo, u_hi;           // empty when u_hi < u_lo
    int n, index;             // index: of the part
    bool split;
};

// Sum over the workgroup; `red` has 4 entries per call site's use.
__device__ __forceinline__ long long block_sum(long long v, long long* red) {
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    lds_publish_barrier();
    return red[0] + red[1] + red[2] + red[3];
}

struct ShareScratch {
    long long red[4];
    int found[8];
};

__device__ __forceinline__ bool find_share(const PagedArgs& a, ShareScratch& sh, Share& r) {
    const int tid = threadIdx.x;
    int want = blockIdx.x;
    if (a.xcd_run) {
        // workgroups are dealt to the 8 XCDs in turn: give each XCD runs of
        // consecutive shares, whose tiles read the same keys
        const int slot = want >> 3, run = fdiv(slot, a.frun);
        want = (run * 8 + (want & 7)) * a.xcd_run + (slot - run * a.xcd_run);
    }
    int b, rem, parts = 1, chunk = 0, tiles, first = 0;
    SeqGeo g;
    if (a.direct) {
        const int bh = fdiv(want, a.fslots);
        rem = want - bh * a.tile_slots;
        b = fdiv(bh, a.fkv);
        if (b >= a.B) return false;
        r.h = bh - b * a.Hkv;
        g = seq_geo(a, b);
        if (rem >= g.tiles) return false;
        tiles = g.tiles;
        r.split = false;
        r.index = 0;
    } else {
        // tiles and key blocks of the whole batch
        long long work = 0, all = 0;
        for (int i = tid; i < a.B; i += kPagedThreads) {
            const SeqGeo s = seq_geo(a, i);
            all += static_cast<long long>(s.tiles) * a.Hkv;
            work += static_cast<long long>(s.tiles) * a.Hkv * s.blocks;
        }
        all = block_sum(all, sh.red);
        work = block_sum(work, sh.red);
        chunk = 0x7fffffff;
        if (all < a.target) {
            const long long c = (work + a.target - 1) / a.target;
            chunk = static_cast<int>(c > a.least ? c : a.least);
        }
        if (blockIdx.x == 0 && tid == 0) *a.count = all < a.target ? static_cast<int>(all) : 0;
        // the sequence whose shares hold `want`: running sums, 256 at a time
        if (tid == 0) sh.found[0] = -1;
        long long base = 0, tile_base = 0;
        for (int i0 = 0; i0 < a.B; i0 += kPagedThreads) {
            const int i = i0 + tid;
            int mine = 0, mine_tiles = 0, ns = 1;
            if (i < a.B) {
                const SeqGeo s = seq_geo(a, i);
                ns = chunk == 0x7fffffff ? 1 : (s.blocks + chunk - 1) / chunk;
                mine_tiles = s.tiles * a.Hkv;
                mine = mine_tiles * ns;
            }
            int run = mine, run_tiles = mine_tiles;
            for (int m = 1; m < 64; m <<= 1) {
                const int x = __shfl_up(run, m), y = __shfl_up(run_tiles, m);
                if ((tid & 63) >= m) {
                    run += x;
                    run_tiles += y;
                }
            }
            __syncthreads();
            if ((tid & 63) == 63) sh.red[tid >> 6] = (static_cast<long long>(run_tiles) << 32) | static_cast<uint32_t>(run);
            lds_publish_barrier();
            long long lo = base, tlo = tile_base;
            for (int w = 0; w < 4; ++w) {
                const int items = static_cast<int>(sh.red[w] & 0xffffffff), tl = static_cast<int>(sh.red[w] >> 32);
                if (w < (tid >> 6)) {
                    lo += items;
                    tlo += tl;
                }
                base += items;
                tile_base += tl;
            }
            lo += run - mine;
            if (want >= lo && want < lo + mine) {
                sh.found[0] = i;
                sh.found[1] = want - static_cast<int>(lo);
                sh.found[2] = ns;
                sh.found[3] = static_cast<int>(lo);
                sh.found[4] = static_cast<int>(tlo + run_tiles - mine_tiles);
            }
            if (base > want) break;
        }
        lds_publish_barrier();
        b = sh.found[0];
        if (b < 0) return false;
        rem = sh.found[1];
        parts = sh.found[2];
        first = sh.found[3];
        g = seq_geo(a, b);
        tiles = g.tiles;
        // order: kv head, part, tile
        const int per_head = parts * tiles;
        r.h = rem / per_head;
        rem -= r.h * per_head;
        r.split = parts > 1;
        r.index = want;
    }
    const int part = rem / tiles, slot = rem - part * tiles;
    const int per_class = tiles / g.classes;
    r.b = b;
    r.n = g.n;
    r.cls = slot / per_class;
    // the last tiles have the most keys: first
    const int t = per_class - 1 - (slot - r.cls * per_class);
    const int members = ceil_div(g.n - r.cls, a.dil);
    r.row0 = t * a.M;
    r.rows = imin(a.M, members * a.rep - r.row0);
    const int x = g.len - g.n + r.cls;  // position of member 0
    r.w0 = x >= 0 ? fdiv(x, a.fdil) : -((-x - 1) / a.dil + 1);
    r.c = x - r.w0 * a.dil;
    r.u_lo = 0;
    r.u_hi = -1;
    if (r.rows > 0) {
        const int wf = r.w0 + fdiv(r.row0, a.frep), wl = r.w0 + fdiv(r.row0 + r.rows - 1, a.frep);
        r.u_lo = a.K ? imax(0, wf - a.K + 1) : 0;
        const long long cap = static_cast<long long>(a.width) * a.page_size - 1 - r.c;
        const long long last = cap < 0 ? -1 : cap / a.dil;
        r.u_hi = wl < last ? wl : static_cast<int>(last);
    }
    if (r.split) {
        if (part == 0 && tid == 0) {
            PagedTile& p = a.tiles[sh.found[4] + r.h * tiles + slot];
            p.first = want;
            p.step = tiles;
            p.parts = parts;
            p.b = b;
            p.h = r.h;
            p.cls = r.cls;
            p.row0 = r.row0;
            p.rows = r.rows;
        }
        const long long from = r.u_lo + static_cast<long long>(part) * chunk * a.KT;
        const long long to = from + static_cast<long long>(chunk) * a.KT - 1;
        if (from > r.u_hi) r.u_hi = r.u_lo - 1;
        else {
            r.u_lo = static_cast<int>(from);
            if (to < r.u_hi) r.u_hi = static_cast<int>(to);
        }
    } else if (!a.direct && tid == 0 && sh.found[4] + r.h * tiles + slot < a.target) {
        a.tiles[sh.found[4] + r.h * tiles + slot].parts = 1;
    }
    return true;
}

// Where key u of class residue c is: false when no page of the cache holds it.
__device__ __forceinline__ bool key_at(const PagedArgs& a, const int* table, int c, int u, int u_hi, int& page,
                                       int& slot) {
    if (u > u_hi) return false;
    const int j = c + u * a.dil;
    const int pg = fdiv(j, a.fpage);
    slot = j - pg * a.page_size;
    page = table[pg];
    return page >= 0 && page < a.pages;
}

}  // namespace

}  // namespace na
