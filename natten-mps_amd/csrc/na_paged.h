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
    int cap, pages, page_size;  // cap: positions of the table, an int at most
    FastDiv fpage;
    int B, L, Hq, Hkv, rep, Dqk, Dv;
    FastDiv frep, flen, fdv;
    int K, dil;  // K 0: no window
    FastDiv fdil;
    float scale;
    int M, log_m, log_kt;  // rows of a tile, keys of a block
    int tile_slots;        // tiles of a (sequence, kv head) at most
    int direct;            // every tile whole: slot = tile, nothing to work out
    int log_target;        // workgroups aimed at when tiles are few
    int least;             // key blocks of a chunk at least
    int xcd_run;           // consecutive shares of one XCD (0: as dealt)
    FastDiv fslots, fkv, frun;
    int per_wave;          // tokens of the batch that a wave looks at for padding
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

// Divisions are by invariants (FastDiv) or powers of two: an emulated 64-bit
// one costs half a microsecond of a call's latency.
struct SeqGeo {
    int n, len, classes, per_class, tiles, blocks;  // tiles: of all its classes, one kv head
};

// ceil(n / d) of 0 <= n
__device__ __forceinline__ int ceil_fdiv(int n, const FastDiv& d) { return n > 0 ? fdiv(n - 1, d) + 1 : 0; }

__device__ __forceinline__ SeqGeo seq_geo(const PagedArgs& a, int n, int len) {
    SeqGeo g;
    g.n = imin(imax(n, 0), a.L);
    g.len = imax(len, 0);
    g.classes = imin(g.n, a.dil);
    const int members = ceil_fdiv(g.n, a.fdil);
    g.per_class = (members * a.rep + a.M - 1) >> a.log_m;
    g.tiles = g.classes * g.per_class;
    int keys = fdiv(imin(g.len, a.cap), a.fdil) + 1;
    if (a.K) {
        const uint32_t span = static_cast<uint32_t>(a.K) + imin(members, fdiv(a.M, a.frep) + 2) - 1;
        if (span < static_cast<uint32_t>(keys)) keys = static_cast<int>(span);
    }
    g.blocks = ((keys - 1) >> a.log_kt) + 1;
    return g;
}

// First key (class coordinates) of the window of the query at w: K - 1 keys
// behind it, not below 0.  w may lie before the sequence (down to -2^27) and
// K be any int, whose difference passes 32 bits: compared, not subtracted.
__device__ __forceinline__ int first_key(const PagedArgs& a, int w) {
    return a.K && w >= a.K ? w - a.K + 1 : 0;
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

// Inclusive running sums over the wave's lanes (DPP shifts inside 16-lane
// rows, then the rows' last lanes to the rows after them).
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_or_zero(T v) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_or_zero<0x111, 0xf>(v);
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);
    v += dpp_or_zero<0x143, 0xc>(v);
    return v;
}

template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Every wave works the cut out for itself, lanes on sequences, 64 at a time:
// no barriers, and what comes out is uniform.
__device__ __forceinline__ bool find_share(const PagedArgs& a, Share& r) {
    const int lane = threadIdx.x & 63, target = 1 << a.log_target;
    int want = wide_block();
    if (a.xcd_run) {
        // workgroups are dealt to the 8 XCDs in turn: give each XCD runs of
        // consecutive shares, whose tiles read the same keys
        const int slot = want >> 3, run = fdiv(slot, a.frun);
        want = (run * 8 + (want & 7)) * a.xcd_run + (slot - run * a.xcd_run);
    }
    int b, rem, parts = 1, chunk = 0, tile_first = 0, n, len;
    r.h = 0;
    r.split = false;
    r.index = 0;
    if (a.direct) {
        const int bh = fdiv(want, a.fslots);
        rem = want - bh * a.tile_slots;
        b = fdiv(bh, a.fkv);
        if (b >= a.B) return false;
        r.h = bh - b * a.Hkv;
        n = a.news ? a.news[b] : a.L;
        len = a.lens[b];
    } else {
        // tiles and key blocks of the whole batch; the sum of blocks in fp32,
        // so that the chunk from it is one more than rounding can lose
        int all = 0;
        float work = 0.f;
        int n0 = 0, len0 = 0;  // of the first 64 sequences
        for (int i0 = 0; i0 < a.B; i0 += 64) {
            const int i = i0 + lane;
            int ni = 0, li = 0;
            if (i < a.B) {
                ni = a.news ? a.news[i] : a.L;
                li = a.lens[i];
            }
            if (i0 == 0) {
                n0 = ni;
                len0 = li;
            }
            const SeqGeo s = seq_geo(a, ni, li);
            const int tiles = s.tiles * a.Hkv;
            all += lane_value(wave_scan(tiles), 63);
            work += lane_value(wave_scan(static_cast<float>(tiles) * static_cast<float>(s.blocks)), 63);
        }
        const bool cut = all < target;
        chunk = imax(static_cast<int>(__builtin_ldexpf(work, -a.log_target)) + 1, a.least);
        if (want == 0 && threadIdx.x == 0) *a.count = cut ? all : 0;
        // the sequence whose shares hold `want`.  Where keys are cut there are
        // fewer than 2^9 tiles and 2^10 shares, summed together.
        int base = 0, owner = -1, lo = 0, ns = 1;
        int i0 = 0;
        for (; i0 < a.B; i0 += 64) {
            const int i = i0 + lane;
            int ni = n0, li = len0;
            if (i0) {
                ni = li = 0;
                if (i < a.B) {
                    ni = a.news ? a.news[i] : a.L;
                    li = a.lens[i];
                }
                n0 = ni;
                len0 = li;
            }
            const SeqGeo s = seq_geo(a, ni, li);
            ns = cut ? static_cast<int>(static_cast<uint32_t>(s.blocks + chunk - 1) / static_cast<uint32_t>(chunk)) : 1;
            const int tiles = s.tiles * a.Hkv;
            const int sum = wave_scan(cut ? (tiles << 16) + tiles * ns : tiles);
            lo = base + sum - (cut ? (tiles << 16) + tiles * ns : tiles);
            const int mine = cut ? lo & 0xffff : lo;
            const unsigned long long hit = __ballot(i < a.B && want >= mine && want < mine + tiles * ns);
            if (hit) {
                owner = __ffsll(hit) - 1;
                // parts of one tile as even as whole blocks allow
                chunk = ns == 1 ? 0 : static_cast<int>(static_cast<uint32_t>(s.blocks + ns - 1) / static_cast<uint32_t>(ns));
                break;
            }
            base += lane_value(sum, 63);
        }
        if (owner < 0) return false;
        b = i0 + owner;
        n = lane_value(n0, owner);
        len = lane_value(len0, owner);
        parts = lane_value(ns, owner);
        chunk = lane_value(chunk, owner);
        const int at = lane_value(lo, owner);
        rem = want - (cut ? at & 0xffff : at);
        tile_first = cut ? at >> 16 : at;
        r.split = parts > 1;
        r.index = want;
    }
    const SeqGeo g = seq_geo(a, __builtin_amdgcn_readfirstlane(n), __builtin_amdgcn_readfirstlane(len));
    if (a.direct) {
        if (rem >= g.tiles) return false;
    } else {
        // order: kv head, part, tile
        const int per_head = parts * g.tiles;
        r.h = static_cast<int>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(per_head));
        rem -= r.h * per_head;
    }
    int part = 0, slot = rem;
    if (parts > 1) {
        part = static_cast<int>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(g.tiles));
        slot = rem - part * g.tiles;
    }
    r.b = b;
    r.n = g.n;
    r.cls = g.classes == 1 ? 0 : static_cast<int>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(g.per_class));
    // the last tiles have the most keys: first
    const int t = g.per_class - 1 - (slot - r.cls * g.per_class);
    const int members = ceil_fdiv(g.n - r.cls, a.fdil);
    r.row0 = t << a.log_m;
    r.rows = imin(a.M, members * a.rep - r.row0);
    const int x = g.len - g.n + r.cls;  // position of member 0
    r.w0 = x >= 0 ? fdiv(x, a.fdil) : -(fdiv(-x - 1, a.fdil) + 1);
    r.c = x - r.w0 * a.dil;
    r.u_lo = 0;
    r.u_hi = -1;
    if (r.rows > 0) {
        const int wf = r.w0 + fdiv(r.row0, a.frep), wl = r.w0 + fdiv(r.row0 + r.rows - 1, a.frep);
        r.u_lo = first_key(a, wf);
        r.u_hi = imin(wl, r.c < a.cap ? fdiv(a.cap - 1 - r.c, a.fdil) : -1);
    }
    if (r.split) {
        if (part == 0 && threadIdx.x == 0) {
            PagedTile& p = a.tiles[tile_first + r.h * g.tiles + slot];
            p.first = want;
            p.step = g.tiles;
            p.parts = parts;
            p.b = b;
            p.h = r.h;
            p.cls = r.cls;
            p.row0 = r.row0;
            p.rows = r.rows;
        }
        const int keys = chunk << a.log_kt;
        const long long from = r.u_lo + static_cast<long long>(part) * keys;
        if (from > r.u_hi) {
            r.u_hi = r.u_lo - 1;
        } else {
            r.u_lo = static_cast<int>(from);
            if (from + keys - 1 < r.u_hi) r.u_hi = static_cast<int>(from + keys - 1);
        }
    } else if (!a.direct && threadIdx.x == 0 && tile_first + r.h * g.tiles + slot < target) {
        a.tiles[tile_first + r.h * g.tiles + slot].parts = 1;
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
