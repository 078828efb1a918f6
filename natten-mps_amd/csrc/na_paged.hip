// Attention of new tokens over a paged cache: the serving form of causal 1-D
// neighbourhood attention (natten_hip_paged_forward).  Tiles, classes and the
// cut of long key runs are described in na_paged.h.
//
//   s_j = scale q . k_j,  m = max_j s_j,  out = sum_j e^(s_j - m) v_j / l,
//   l = sum_j e^(s_j - m),  lse = m + ln l,
// in one pass over the keys with the running m and l in fp32 (base 2 inside:
// the scale carries log2 e).
//
// k_paged_rows  any type, head dims to 256, any alignment: a wave per row.
// k_paged_few   16-bit, head dim 32/64/96/128: 16 rows a workgroup on MFMA,
//               its four waves on different keys.  The cache is read once, so
//               HBM bounds it.
// k_paged_join  joins the parts of tiles whose keys were cut.
#include <type_traits>

#include "na_paged.h"
#include "na_tile.h"

namespace na {

namespace {

// Rows of padding tokens: zeros, and -inf.  The workgroups of the grid share
// the batch's tokens.
template <typename T>
__device__ __forceinline__ void clear_padding(const PagedArgs& a) {
    if (!a.news) return;
    const int tokens = a.B * a.L;
    for (int t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int b = t / a.L, i = t - b * a.L;
        if (i < a.news[b]) continue;
        T* const o = static_cast<T*>(a.out) + b * a.lo.b + i * a.lo.s2;
        for (int e = threadIdx.x; e < a.Hq * a.Dv; e += kPagedThreads) {
            const int h = e / a.Dv;
            o[h * a.lo.h + (e - h * a.Dv)] = from_f<T>(0.f);
        }
        for (int h = threadIdx.x; h < a.Hq; h += kPagedThreads)
            a.lse[b * a.ll.b + i * a.ll.s2 + h * a.ll.h] = -INFINITY;
    }
}

// Token and query head of row r of a tile.
__device__ __forceinline__ void row_token(const PagedArgs& a, int cls, int h, int r, int& i, int& hq) {
    const int m = fdiv(r, a.frep);
    i = cls + m * a.dil;
    hq = h * a.rep + (r - m * a.rep);
}

// lse of a row from its running maximum (base 2) and sum.
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2; }

// ---------------------------------------------------------------------------
// any type and alignment
// ---------------------------------------------------------------------------

// A wave per row; lanes take 64 keys for the scores, then 64 head dims for
// the products.  `VEC` elements of a key are read at once.
template <typename T, int VEC>
__global__ __launch_bounds__(kPagedThreads) void k_paged_rows(PagedArgs a) {
    __shared__ ShareScratch sh;
    __shared__ float qs[4][256];
    clear_padding<T>(a);
    Share r;
    if (!find_share(a, sh, r)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (wave >= r.rows) return;
    int i, hq;
    row_token(a, r.cls, r.h, r.row0 + wave, i, hq);
    const float sc2 = a.scale * kLog2e;
    const T* const q = static_cast<const T*>(a.q) + r.b * a.lq.b + i * a.lq.s2 + hq * a.lq.h;
    for (int d = lane; d < a.Dqk; d += 64) qs[wave][d] = to_f(q[d]);
    // the wave reads its own part of qs only
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int w = r.w0 + fdiv(r.row0 + wave, a.frep);
    const int lo = imax(r.u_lo, a.K ? w - a.K + 1 : 0), hi = imin(r.u_hi, w);
    const int* const table = a.table + r.b * a.table_stride;
    const T* const kb = static_cast<const T*>(a.k) + r.h * a.kh;
    const T* const vb = static_cast<const T*>(a.v) + r.h * a.vh;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int u0 = lo; u0 <= hi; u0 += 64) {
        int page = 0, slot = 0;
        const bool ok = key_at(a, table, r.c, u0 + lane, hi, page, slot);
        float s = -INFINITY;
        if (ok) {
            const T* const k = kb + page * a.kp + slot * a.ks;
            float dot = 0.f;
            for (int d = 0; d < a.Dqk; d += VEC) {
                T x[VEC];
                if constexpr (VEC == 1)
                    x[0] = k[d];
                else
                    *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(k + d);
#pragma unroll
                for (int e = 0; e < VEC; ++e) dot = fmaf(qs[wave][d + e], to_f(x[e]), dot);
            }
            s = dot * sc2;
        }
        float top = s;
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float m2 = fmaxf(m, top), ref = m2 == -INFINITY ? 0.f : m2;
        const float keep = __builtin_amdgcn_exp2f(m - ref);
        const float p = ok ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
        m = m2;
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= keep;
        const long long off = page * a.vp + slot * a.vs;
        const unsigned long long live = __ballot(ok);
        for (int j = 0; j < 64; ++j) {
            if (!((live >> j) & 1)) continue;
            const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j));
            const uint32_t lo32 = __builtin_amdgcn_readlane(static_cast<uint32_t>(off), j);
            const uint32_t hi32 = __builtin_amdgcn_readlane(static_cast<uint32_t>(off >> 32), j);
            const T* const v = vb + static_cast<long long>((static_cast<uint64_t>(hi32) << 32) | lo32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < a.Dv) acc[e] = fmaf(pj, to_f(v[lane + 64 * e]), acc[e]);
        }
    }
    for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x);
    if (r.split) {
        const long long row = static_cast<long long>(r.index) * a.M + wave;
        if (lane == 0) {
            a.ml[2 * row] = m;
            a.ml[2 * row + 1] = l;
        }
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < a.Dv) a.part[row * a.Dv + lane + 64 * e] = acc[e];
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* const o = static_cast<T*>(a.out) + r.b * a.lo.b + i * a.lo.s2 + hq * a.lo.h;
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.Dv) o[lane + 64 * e] = from_f<T>(acc[e] * inv);
    if (lane == 0) a.lse[r.b * a.ll.b + i * a.ll.s2 + hq * a.ll.h] = row_lse(m, l);
}

// ---------------------------------------------------------------------------
// joining parts
// ---------------------------------------------------------------------------

// A workgroup per row of a cut tile: 64 lanes on the head dims (in fours),
// groups of lanes on different parts, joined through LDS in a fixed order.
template <typename T>
__global__ __launch_bounds__(kPagedThreads) void k_paged_join(PagedArgs a) {
    __shared__ float o[kPagedThreads][5];
    const int tile = blockIdx.x;
    if (tile >= *a.count) return;
    const PagedTile t = a.tiles[tile];
    const int row = blockIdx.y;
    if (t.parts <= 1 || row >= t.rows) return;
    const int tid = threadIdx.x;
    float m = -INFINITY;
    for (int s = tid; s < t.parts; s += kPagedThreads)
        m = fmaxf(m, a.ml[2 * ((static_cast<long long>(t.first) + static_cast<long long>(s) * t.step) * a.M + row)]);
    for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    if ((tid & 63) == 0) o[tid >> 6][0] = m;
    lds_publish_barrier();
    m = fmaxf(fmaxf(o[0][0], o[1][0]), fmaxf(o[2][0], o[3][0]));
    const float ref = m == -INFINITY ? 0.f : m;
    __syncthreads();
    // quads of head dims on consecutive threads, the parts over the rest
    const int quads = (a.Dv + 3) / 4, groups = kPagedThreads / quads;
    const int d = 4 * (tid % quads), g = tid / quads;
    float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (g < groups) {
        for (int s = g; s < t.parts; s += groups) {
            const long long at = (static_cast<long long>(t.first) + static_cast<long long>(s) * t.step) * a.M + row;
            const float ms = a.ml[2 * at];
            if (ms == -INFINITY && a.ml[2 * at + 1] == 0.f) continue;  // a part without keys
            const float w = __builtin_amdgcn_exp2f(ms - ref);
            l = fmaf(w, a.ml[2 * at + 1], l);
            const float* const p = a.part + at * a.Dv + d;
            if (a.Dv % 4 == 0) {
                const float4 x = *reinterpret_cast<const float4*>(p);
                acc[0] = fmaf(w, x.x, acc[0]);
                acc[1] = fmaf(w, x.y, acc[1]);
                acc[2] = fmaf(w, x.z, acc[2]);
                acc[3] = fmaf(w, x.w, acc[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < a.Dv) acc[e] = fmaf(w, p[e], acc[e]);
            }
        }
    }
    for (int e = 0; e < 4; ++e) o[tid][e] = acc[e];
    o[tid][4] = l;
    lds_publish_barrier();
    if (g != 0) return;
    for (int s = 1; s < groups; ++s) {
        for (int e = 0; e < 4; ++e) acc[e] += o[s * quads + tid][e];
        l += o[s * quads + tid][4];
    }
    int i, hq;
    row_token(a, t.cls, t.h, t.row0 + row, i, hq);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* const out = static_cast<T*>(a.out) + t.b * a.lo.b + i * a.lo.s2 + hq * a.lo.h;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < a.Dv) out[d + e] = from_f<T>(acc[e] * inv);
    if (tid == 0) a.lse[t.b * a.ll.b + i * a.ll.s2 + hq * a.ll.h] = row_lse(m, l);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Workgroups aimed at when the tiles are few: two a compute unit.
constexpr int kTarget = 512;

struct PagedPlan {
    int M, KT, least, xcd_run;
    long long tiles;  // tile slots of the batch
    int slots;        // of a (sequence, kv head)
    bool split;       // some tile's keys may be cut
    long long grid;
    size_t bytes;     // workspace
};

long long padded(long long bytes) { return (bytes + 255) & ~255ll; }

PagedPlan plan(const PagedCall& c) {
    PagedPlan p{};
    p.M = 4;
    p.KT = 64;
    p.least = 4;
    p.xcd_run = 0;
    const long long rep = c.heads_q / c.heads_kv;
    const long long dil = c.dilation, classes = c.tokens < dil ? c.tokens : dil;
    const long long members = (c.tokens + dil - 1) / dil;
    const long long slots = classes * ((members * rep + p.M - 1) / p.M);
    p.slots = static_cast<int>(slots < 0x7fffffff ? slots : 0x7fffffff);
    p.tiles = slots * c.batch * c.heads_kv;
    const long long cap = static_cast<long long>(c.cache.width) * c.cache.page_size;
    long long keys = cap / dil + 1;
    if (c.kernel) {
        const long long span = static_cast<long long>(c.kernel) + p.M / rep + 1;
        if (span < keys) keys = span;
    }
    // cutting pays where a workgroup has more than the least chunk to read
    // and the tiles leave compute units idle
    p.split = keys > static_cast<long long>(p.least) * p.KT && p.tiles < 8ll * kTarget;
    p.grid = p.tiles;
    if (p.split) {
        const long long most = p.tiles < kTarget ? kTarget + p.tiles : 2ll * kTarget;
        if (p.grid < most) p.grid = most;
        p.bytes = padded(sizeof(int)) + padded(sizeof(PagedTile) * kTarget) +
                  padded(sizeof(float) * 2 * p.M * 2 * kTarget) + sizeof(float) * c.cache.dim_v * p.M * 2 * kTarget;
    }
    return p;
}

template <typename T>
hipError_t launch_rows(const PagedArgs& a, const PagedPlan& p, bool vec, hipStream_t s) {
    constexpr int kVec = 16 / sizeof(T);
    if (vec)
        NA_LAUNCH("na_paged_rows", (k_paged_rows<T, kVec>), dim3(p.grid), dim3(kPagedThreads), 0, s, a);
    else
        NA_LAUNCH("na_paged_rows", (k_paged_rows<T, 1>), dim3(p.grid), dim3(kPagedThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.split) return e;
    NA_LAUNCH("na_paged_join", (k_paged_join<T>), dim3(p.tiles < kTarget ? p.tiles : kTarget, p.M),
              dim3(kPagedThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

size_t paged_workspace(const PagedCall& c) { return plan(c).bytes; }

hipError_t paged_forward(const PagedCall& c, hipStream_t s) {
    const PagedPlan p = plan(c);
    PagedArgs a{};
    a.q = c.q;
    a.out = c.out;
    a.lse = c.lse;
    a.k = c.cache.k;
    a.v = c.cache.v;
    a.lq = c.lq;
    a.lo = c.lo;
    a.ll = c.ll;
    a.kp = c.cache.ks[0];
    a.ks = c.cache.ks[1];
    a.kh = c.cache.ks[2];
    a.vp = c.cache.vs[0];
    a.vs = c.cache.vs[1];
    a.vh = c.cache.vs[2];
    a.table = c.cache.table;
    a.lens = c.cache.lens;
    a.news = c.cache.news;
    a.table_stride = c.cache.table_stride;
    a.width = c.cache.width;
    a.pages = c.cache.pages;
    a.page_size = c.cache.page_size;
    a.fpage = make_fastdiv(a.page_size);
    a.B = c.batch;
    a.L = c.tokens;
    a.Hq = c.heads_q;
    a.Hkv = c.heads_kv;
    a.rep = c.heads_q / c.heads_kv;
    a.Dqk = c.dim_qk;
    a.Dv = c.cache.dim_v;
    a.frep = make_fastdiv(a.rep);
    a.K = c.kernel;
    a.dil = c.dilation;
    a.fdil = make_fastdiv(a.dil);
    a.scale = c.scale;
    a.M = p.M;
    a.KT = p.KT;
    a.tile_slots = p.slots;
    a.direct = p.split ? 0 : 1;
    a.target = kTarget;
    a.least = p.least;
    a.xcd_run = p.xcd_run;
    a.frun = make_fastdiv(imax(p.xcd_run, 1));
    a.fslots = make_fastdiv(p.slots);
    a.fkv = make_fastdiv(a.Hkv);
    if (p.split) {
        char* w = static_cast<char*>(c.work);
        a.count = reinterpret_cast<int*>(w);
        w += padded(sizeof(int));
        a.tiles = reinterpret_cast<PagedTile*>(w);
        w += padded(sizeof(PagedTile) * kTarget);
        a.ml = reinterpret_cast<float*>(w);
        w += padded(sizeof(float) * 2 * p.M * 2 * kTarget);
        a.part = reinterpret_cast<float*>(w);
    }
    if (c.dtype == NATTEN_F32) return launch_rows<float>(a, p, c.vec, s);
    if (c.dtype == NATTEN_F16) return launch_rows<f16>(a, p, c.vec, s);
    return launch_rows<bf16>(a, p, c.vec, s);
}

}  // namespace na
