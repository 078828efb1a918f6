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
// k_paged_few   head dims 32/64/96/128, aligned: 16 to 64 rows a workgroup on
//               MFMA, its four waves on different keys.  With few rows the
//               cache is read once and HBM bounds it.  fp32 takes it for any
//               number of rows.
// k_paged_chunk 16-bit, many rows: 128 or 256 rows a workgroup on MFMA, keys
//               and values staged in LDS for all its waves.
// k_paged_join  joins the parts of tiles whose keys were cut.
#include <type_traits>

#include "na_paged.h"
#include "na_tile.h"

namespace na {

namespace {

// Rows of padding tokens: zeros, and -inf.  The grid's waves share the batch's
// tokens evenly, a lane looks whether one is padding, then the wave clears
// those that are.
template <typename T>
__device__ __forceinline__ void clear_padding(const PagedArgs& a) {
    if (!a.news) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(wide_block() * (kPagedThreads / 64) + static_cast<int>(threadIdx.x >> 6));
    const int first = wave * a.per_wave, end = imin(first + a.per_wave, a.B * a.L);
    for (int t0 = first; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        bool pad = false;
        if (t < end) {
            const int b = fdiv(t, a.flen);
            pad = t - b * a.L >= a.news[b];
        }
        for (unsigned long long left = __ballot(pad); left; left &= left - 1) {
            const int x = t0 + __ffsll(left) - 1, b = fdiv(x, a.flen), i = x - b * a.L;
            T* const o = static_cast<T*>(a.out) + b * a.lo.b + i * a.lo.s2;
            for (int e = lane; e < a.Hq * a.Dv; e += 64) {
                const int h = fdiv(e, a.fdv);
                o[h * a.lo.h + (e - h * a.Dv)] = from_f<T>(0.f);
            }
            for (int h = lane; h < a.Hq; h += 64) a.lse[b * a.ll.b + i * a.ll.s2 + h * a.ll.h] = -INFINITY;
        }
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
// the products.  `VEC` elements of a key are read at once.  Head dims and
// alignments that the MFMA kernels do not take; a row's keys are read once a
// query head and token, and address arithmetic bounds it: one token of each of
// 16 requests of 8192 keys, 32/8 heads of 80, 1640 us (k_paged_few at 96: 93),
// 512 tokens over 4096 keys, 16/4 heads of 80, 3830 us (k_paged_chunk at 96:
// 53); fp32, 257 tokens in a window of 63, 4 heads of 32, 19 (k_paged_few 11).
template <typename T, int VEC>
__global__ __launch_bounds__(kPagedThreads) void k_paged_rows(PagedArgs a) {
    __shared__ float qs[4][256];
    clear_padding<T>(a);
    Share r;
    if (!find_share(a, r)) return;
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
    const int lo = imax(r.u_lo, first_key(a, w)), hi = imin(r.u_hi, w);
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
// on MFMA
// ---------------------------------------------------------------------------

// Elements of an LDS row of head dim D, and the swizzle of its 16-byte pieces:
// the 16 rows x 32 bytes of a transposing read, and the rows that 8 lanes
// write, lie on distinct banks.
template <int D>
constexpr int row_elems() {
    return D == 96 ? 128 : D;
}

template <int D>
__device__ __forceinline__ int piece_swz(int row) {
    constexpr int LD = row_elems<D>();
    const int odd = (row >> 3) & 1;
    if constexpr (LD == 128) return ((row & 7) << 1) | odd;
    else if constexpr (LD == 64) return (((row >> 1) & 3) << 1) | odd;
    else return (((row >> 2) & 1) << 1) | odd;
}

// A row's running maximum is raised, and what was summed scaled down, only
// where the scores pass it by this many powers of two: early keys seldom hold
// the maximum, and exponentials up to 2^8 lose nothing (a sum in fp32 of 2^31
// of them is far from its limit).
constexpr float kSlack = 8.f;

// 16-bit probabilities are rounded once for the product with the values, the
// matrix operands' type; sums and results stay in fp32.  A half step of the
// type on each, against the one on the result, takes errors against 64 bits
// to 1.2 to 1.4 times those of the 32-bit form; a second term would double
// the products.  fp16 ones carry a factor of 2^7 (running values are relative
// to the maximum less 7): with the slack they end at 2^15, and it is those
// below 2^-32 of the largest that vanish, 2^-15 of the weight over 2^17 keys,
// not those below 2^-25.  bf16 has fp32's range.
template <typename T>
constexpr float kCarry = std::is_same<T, f16>::value ? 7.f : 0.f;

// The scale's sign goes into the queries (exact), a scale of zero makes them
// zero, so that scores times `sc2` > 0 order as the logits do.
struct ScaleParts {
    float sc2;
    uint32_t flip, keep;  // of a word: one element, or two 16-bit ones
};

template <typename T>
__device__ __forceinline__ ScaleParts scale_parts(float scale) {
    ScaleParts r;
    r.sc2 = scale == 0.f ? 1.f : __builtin_fabsf(scale) * kLog2e;
    r.flip = scale < 0.f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
    r.keep = scale == 0.f ? 0u : 0xffffffffu;
    return r;
}

__device__ __forceinline__ uint4 scaled(uint4 x, const ScaleParts& s) {
    return make_uint4((x.x & s.keep) ^ s.flip, (x.y & s.keep) ^ s.flip, (x.z & s.keep) ^ s.flip,
                      (x.w & s.keep) ^ s.flip);
}

// A product adds 0 times the values that a row does not attend to, which is
// NaN where such a value is not finite.  Rows with a NaN are summed again
// (redo_rows), in walks whose products meet finite values only; an infinity
// in a result is the row's own.
enum RedoWalk {
    kFinite,  // values that are not finite count as 0
    kPlus,    // +infinity and NaN as 1, the rest as 0, keys attended to as 1
    kMinus,   // -infinity and NaN
    kWalks
};

// The elements of a vector of values as a walk takes them.
template <typename T>
__device__ __forceinline__ uint4 walk_values(uint4 x, int walk) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr uint32_t kOne = F32 ? 0x3F800000u : Mma<typename std::conditional<F32, bf16, T>::type>::kOnes & 0xffffu;
    constexpr uint32_t kSign = F32 ? 0x80000000u : 0x8000u;
    constexpr uint32_t kInf = F32 ? 0x7F800000u : std::is_same<T, f16>::value ? 0x7C00u : 0x7F80u;
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t r = 0;
#pragma unroll
        for (int sh = 0; sh < 32; sh += 8 * static_cast<int>(sizeof(T))) {
            const uint32_t e = F32 ? w[i] : (w[i] >> sh) & 0xffffu, mag = e & (kSign - 1);
            const bool plus = mag > kInf || e == kInf, minus = mag > kInf || e == (kInf | kSign);
            const uint32_t v = walk == kFinite ? (mag < kInf ? e : 0u) : (walk == kPlus ? plus : minus) ? kOne : 0u;
            r |= v << sh;
        }
        w[i] = r;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 NB rows, the four waves on different keys, 32 at a time each.
//
// Scores as S^T = K Q^T (v_mfma 16x16x32): a lane then holds one query (its
// column) and keys 4g..4g+3 of each 16-key block (g its 16-lane row), so the
// softmax of a query is in-lane but for two lane exchanges, and the packed
// probabilities are at once the B operand of O^T = V^T P^T, whose k slots are
// those keys.  K goes straight from the pages to registers in the A layout
// (lane: key `col`, 16-byte pieces g, g + 4, ..); V, read the same way, is
// written to the wave's own LDS and read back transposed.
//
// Each key is read once per kv head and nothing else is big, so HBM bounds
// it: the next keys' loads are issued as soon as the registers are free, and
// page numbers one step before that.  32 requests of 1 to 16385 tokens, 32/8
// heads of 128, one new token each: 1.08 GB in 231 to 240 us (4.6 TB/s; a
// large copy moves 5.2 to 5.4), in fp32 440 us (4.9 TB/s).  One request of
// 131070 tokens and 5 new ones, 8/1 heads of 64: 34 MB in 18 us, of which 11 are
// there with 600 tokens too: latency of lengths, pages, keys and parts.
//
// fp32 takes v_mfma 16x16x4, 16 keys at a time: element e of the 16-byte
// pieces is one product's k slot (both operands permuted alike), and a lane's
// four keys of a block are the k slots of four products with V, whose operand
// needs no transposition.
constexpr int kFewRows = 16;
template <typename T>
constexpr int few_keys() {
    return sizeof(T) == 4 ? 16 : 32;
}

typedef float f32x4v_t __attribute__((ext_vector_type(4)));

// Swizzle of a row's 16-byte pieces in k_paged_few's LDS.
template <typename T, int D>
__device__ __forceinline__ int few_swz(int row) {
    if constexpr (sizeof(T) == 4) return row & (D == 32 ? 7 : 15);
    else return piece_swz<D>(row);
}

// Waves a SIMD that leave the kernel its registers.
template <typename T>
constexpr int few_waves(int dim, int blocks) {
    if (sizeof(T) == 4) return blocks == 1 ? (dim > 64 ? 2 : 4) : dim > 96 ? 1 : 2;
    return blocks > 1 || dim > 96 ? 2 : dim > 64 ? 3 : 4;
}

// Where a row's results go: a part, or the output with its sum.
template <typename T>
__device__ __forceinline__ void put_four(const PagedArgs& a, const Share& r, int row, int d, f32x4_t x, float l) {
    if (r.split) {
        *reinterpret_cast<f32x4_t*>(a.part + (static_cast<long long>(r.index) * a.M + row) * a.Dv + d) = x;
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    int i, hq;
    row_token(a, r.cls, r.h, r.row0 + row, i, hq);
    T* const out = static_cast<T*>(a.out) + r.b * a.lo.b + i * a.lo.s2 + hq * a.lo.h + d;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<f32x4_t*>(out) = x * inv;
    else
        *reinterpret_cast<uint2*>(out) = make_uint2(Mma<T>::pack(x[0] * inv, x[1] * inv),
                                                    Mma<T>::pack(x[2] * inv, x[3] * inv));
}

// Rows of the tile that are summed again, 16 at a time, the waves on
// different keys as in k_paged_few: `again(row, m, l)` says which, and gives
// their maximum and sum (the scores do not depend on the values, so both hold
// as they are).  A walk over the finite values gives the sums, two more
// whether the row attends to infinities of either sign or NaN.  Three walks
// for 16 rows, whatever the values hold: latency bounds them, since one
// workgroup redoes its tile alone and loads nothing ahead.  A pass with finite
// values / a NaN at the newest token / one that all rows attend to, heads of
// 128, us: 4 tokens over 2000 keys 18 / 49 / 49, 512 tokens 60 / 480 / 1720,
// 4096 tokens over 32096 keys 2250 / 39400 / 65800.
// All of the workgroup's threads come here, the tile's own LDS is free.
template <typename T, int D, class Again>
__device__ __forceinline__ void redo_rows(const Share& r, unsigned char* lds, const Again& again) {
    const PagedArgs& a = *static_cast<const PagedArgs*>(kernargs());  // read afresh: nothing is kept for this path
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int E = 16 / sizeof(T), C = D / (4 * E);
    constexpr int LD = row_elems<D>(), DB = D / 16, KS = few_keys<T>(), KB = KS / 16;
    constexpr int kQuads = D / 4, kItems = (16 * kQuads + kPagedThreads - 1) / kPagedThreads;
    const int tid = opaque(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const ScaleParts sp = scale_parts<T>(a.scale);
    const int* const table = a.table + r.b * a.table_stride;
    const T* const kb = static_cast<const T*>(a.k) + r.h * a.kh + E * g;
    const T* const vb = static_cast<const T*>(a.v) + r.h * a.vh + E * g;
    T* const X = reinterpret_cast<T*>(lds) + wave * (KS * LD);
    float* const parts = reinterpret_cast<float*>(lds);  // [4][16][D]
    const uint32_t reach = a.K ? a.K - 1 : 0x7fffffffu;
    lds_publish_barrier();
#pragma unroll 1
    for (int row0 = 0; row0 < r.rows; row0 += 16) {
        const int last = imin(row0 + 15, r.rows - 1), row = imin(row0 + col, last);
        float m, l;
        if (!__ballot(again(row, m, l))) continue;  // the same in every wave
        const float ref = m == -INFINITY ? 0.f : m;
        int qi, qh;
        row_token(a, r.cls, r.h, r.row0 + row, qi, qh);
        const T* const q = static_cast<const T*>(a.q) + r.b * a.lq.b + qi * a.lq.s2 + qh * a.lq.h;
        uint4 qf[C];
#pragma unroll
        for (int c = 0; c < C; ++c) qf[c] = scaled(*reinterpret_cast<const uint4*>(q + E * (4 * c + g)), sp);
        const int hi = r.w0 + fdiv(r.row0 + row, a.frep);
        const int lo_u = imax(r.u_lo, first_key(a, r.w0 + fdiv(r.row0 + row0, a.frep)));
        const int hi_u = imin(r.u_hi, r.w0 + fdiv(r.row0 + last, a.frep));
        f32x4_t sum[kItems];
        uint32_t plus[kItems];
#pragma unroll 1
        for (int walk = kFinite; walk < kWalks; ++walk) {
            f32x4_t o[DB];
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int ub = lo_u + wave * KS; ub <= hi_u; ub += 4 * KS) {
                f32x4_t s[KB];
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    int page = 0, slot = 0;
                    const bool ok = key_at(a, table, r.c, ub + 16 * b + col, hi_u, page, slot);
                    // keys that are not there: the pool's first slot, masked below
                    const int pg = ok ? page : 0, sl = ok ? slot : 0;
                    const T* const k = kb + (pg * a.kp + sl * a.ks);
                    const T* const v = vb + (pg * a.vp + sl * a.vs);
                    s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                    const int rw = 16 * b + col, sw = few_swz<T, D>(rw);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const uint4 kf = *reinterpret_cast<const uint4*>(k + 4 * E * c);
                        uint4 vf = *reinterpret_cast<const uint4*>(v + 4 * E * c);
                        if constexpr (F32) {
                            const f32x4v_t x = __builtin_bit_cast(f32x4v_t, kf), y = __builtin_bit_cast(f32x4v_t, qf[c]);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], s[b], 0, 0, 0);
                        } else {
                            s[b] = Mma<T>::run(kf, qf[c], s[b]);
                        }
                        vf = walk_values<T>(vf, walk);
                        if (!ok) vf = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(X + rw * LD + ((4 * c + g) ^ sw) * E) = vf;
                    }
                    const uint32_t have = static_cast<uint32_t>(__ballot(ok)) >> (4 * g);
                    const uint32_t back = static_cast<uint32_t>(hi - ub - 16 * b - 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = back - i <= reach && ((have >> i) & 1) && s[b][i] != -INFINITY;
                        const float p = walk == kFinite ? __builtin_amdgcn_exp2f(fmaf(s[b][i], sp.sc2, -ref)) : 1.f;
                        s[b][i] = seen ? p : 0.f;
                    }
                }
                if constexpr (F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rw = 4 * g + i;
#pragma unroll
                        for (int db = 0; db < DB; ++db) {
                            const float x = X[rw * LD + ((4 * db + (col >> 2)) ^ few_swz<T, D>(rw)) * 4 + (col & 3)];
                            o[db] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[0][i], o[db], 0, 0, 0);
                        }
                    }
                } else {
                    const uint4 p = pack8<T>(s);
                    const int r0 = 4 * g + (col >> 2), r1 = 16 + r0;
                    const int s0 = piece_swz<D>(r0), s1 = piece_swz<D>(r1);
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const int pc = 2 * db + ((col & 3) >> 1);
                        const T* const x0 = X + r0 * LD + ((pc ^ s0) << 3) + (col & 1) * 4;
                        const T* const x1 = X + r1 * LD + ((pc ^ s1) << 3) + (col & 1) * 4;
                        const uint2 a2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)x0));
                        const uint2 b2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)x1));
                        o[db] = Mma<T>::run(make_uint4(a2.x, a2.y, b2.x, b2.y), p, o[db]);
                    }
                }
            }
            lds_publish_barrier();
#pragma unroll
            for (int db = 0; db < DB; ++db)
                *reinterpret_cast<f32x4_t*>(parts + (wave * 16 + col) * D + 16 * db + 4 * g) = o[db];
            lds_publish_barrier();
#pragma unroll
            for (int n = 0; n < kItems; ++n) {
                const int e = tid + n * kPagedThreads, rw = e / kQuads, d = 4 * (e - rw * kQuads);
                float mr, lr;
                if (e >= 16 * kQuads || row0 + rw > last || !again(row0 + rw, mr, lr)) continue;
                f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) x += *reinterpret_cast<const f32x4_t*>(parts + (w * 16 + rw) * D + d);
                if (walk == kFinite) {
                    sum[n] = x;
                    continue;
                }
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) bits |= x[i] > 0.f ? 1u << i : 0u;
                if (walk == kPlus) {
                    plus[n] = bits;
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool up = (plus[n] >> i) & 1, down = (bits >> i) & 1;
                    if (up || down) sum[n][i] = up && down ? __builtin_nanf("") : up ? INFINITY : -INFINITY;
                }
                put_four<T>(a, r, row0 + rw, d, sum[n], lr);
            }
            lds_publish_barrier();
        }
    }
}

template <typename T, int D, int NB>
__global__ __launch_bounds__(kPagedThreads, few_waves<T>(D, NB)) void k_paged_few(PagedArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int E = 16 / sizeof(T), C = D / (4 * E);  // elements of a piece, pieces of a lane in a row
    constexpr int LD = row_elems<D>(), DB = D / 16, KS = few_keys<T>(), KB = KS / 16;
    constexpr int kRowsOf = kFewRows * NB;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ float ml[4][kRowsOf][2];
    __shared__ uint32_t bad[4][NB];  // rows of which a wave has a NaN among its sums
    clear_padding<T>(a);
    Share r;
    if (!find_share(a, r)) return;
    if (r.rows <= 0) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, g = lane >> 4;
    const ScaleParts sp = scale_parts<T>(a.scale);
    // queries, their windows, and what all rows of the tile see
    uint4 qf[NB][C];
    int hi[NB];
    const uint32_t reach = a.K ? a.K - 1 : 0x7fffffffu;  // keys behind a query's own
    auto query = [&](int n) {
        int qi, qh;
        row_token(a, r.cls, r.h, r.row0 + imin(16 * n + col, r.rows - 1), qi, qh);
        return static_cast<const T*>(a.q) + r.b * a.lq.b + qi * a.lq.s2 + qh * a.lq.h;
    };
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const T* const q = query(n);
#pragma unroll
        for (int c = 0; c < C; ++c) qf[n][c] = scaled(*reinterpret_cast<const uint4*>(q + E * (4 * c + g)), sp);
        hi[n] = r.w0 + fdiv(r.row0 + imin(16 * n + col, r.rows - 1), a.frep);
    }
    const int all_hi = imin(r.w0 + fdiv(r.row0, a.frep), r.u_hi);
    const int all_lo = first_key(a, r.w0 + fdiv(r.row0 + r.rows - 1, a.frep));
    const int steps = (r.u_hi - r.u_lo + KS) / KS;  // 0 when empty: u_hi = u_lo - 1 at least
    const int* const table = a.table + r.b * a.table_stride;
    const T* const kb = static_cast<const T*>(a.k) + r.h * a.kh + E * g;
    const T* const vb = static_cast<const T*>(a.v) + r.h * a.vh + E * g;
    T* const X = reinterpret_cast<T*>(lds) + wave * (KS * LD);

    int page[KB], slot[KB];
    auto lookup = [&](int st) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int u = imin(r.u_lo + st * KS + 16 * b + col, r.u_hi);
            const int j = r.c + u * a.dil;
            const int pg = fdiv(j, a.fpage);
            slot[b] = j - pg * a.page_size;
            page[b] = table[pg];
        }
    };
    uint4 kf[KB][C], vf[KB][C];
    bool ok[KB];
    auto load = [&](int st) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            ok[b] = page[b] >= 0 && page[b] < a.pages && r.u_lo + st * KS + 16 * b + col <= r.u_hi;
            // keys that are not there: the pool's first slot, masked below
            const int pg = ok[b] ? page[b] : 0, sl = ok[b] ? slot[b] : 0;
            const T* const k = kb + (pg * a.kp + sl * a.ks);
            const T* const v = vb + (pg * a.vp + sl * a.vs);
#pragma unroll
            for (int c = 0; c < C; ++c) kf[b][c] = *reinterpret_cast<const uint4*>(k + 4 * E * c);
#pragma unroll
            for (int c = 0; c < C; ++c) vf[b][c] = *reinterpret_cast<const uint4*>(v + 4 * E * c);
        }
    };

    float m[NB], l[NB];
    f32x4_t o[NB][DB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[n][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    if (wave < steps) {
        lookup(wave);
        load(wave);
        if (wave + 4 < steps) lookup(wave + 4);
    }
    for (int st = wave; st < steps; st += 4) {
        const int ub = r.u_lo + st * KS;
        f32x4_t s[NB][KB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                s[n][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if constexpr (F32) {
                        const f32x4v_t x = __builtin_bit_cast(f32x4v_t, kf[b][c]);
                        const f32x4v_t y = __builtin_bit_cast(f32x4v_t, qf[n][c]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[n][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], s[n][b], 0, 0, 0);
                    } else {
                        s[n][b] = Mma<T>::run(kf[b][c], qf[n][c], s[n][b]);
                    }
                }
            }
        bool there[KB];
        unsigned long long have[KB];
        bool whole = true;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            there[b] = ok[b];
            have[b] = __ballot(there[b]);
            whole = whole && have[b] == ~0ull;
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int rw = 16 * b + col, sw = few_swz<T, D>(rw);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                uint4 x = vf[b][c];
                if (!whole && !there[b]) x = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(X + rw * LD + ((4 * c + g) ^ sw) * E) = x;
            }
        }
        if (st + 4 < steps) {
            load(st + 4);
            if (st + 8 < steps) lookup(st + 8);
        }
        if (!whole || ub + KS - 1 > all_hi || ub < all_lo) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                // keys ahead of the query count as far behind it
                const uint32_t back = static_cast<uint32_t>(hi[n] - ub - 4 * g);
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (back - (16 * b + i) > reach || !((static_cast<uint32_t>(have[b]) >> (4 * g + i)) & 1)) s[n][b][i] = -INFINITY;
            }
        }
        uint4 p[F32 ? 1 : NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float top;
            if constexpr (KB == 2)
                top = max8(s[n]);
            else
                top = fmaxp(fmaxp(s[n][0][0], s[n][0][1]), fmaxp(s[n][0][2], s[n][0][3]));
            top = max_rows(top) * sp.sc2;
            const bool raise = top > m[n] + (kSlack + kCarry<T>);
            if (__ballot(raise)) {
                const float m2 = raise ? top - kCarry<T> : m[n];
                const float keep = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m2);
                m[n] = m2;
                l[n] *= keep;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[n][db] *= keep;
            }
            const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][b][i] = __builtin_amdgcn_exp2f(fmaf(s[n][b][i], sp.sc2, -ref));
                    l[n] += s[n][b][i];
                }
            if constexpr (!F32) p[n] = pack8<T>(s[n]);
        }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rw = 4 * g + i;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const float x = X[rw * LD + ((4 * db + (col >> 2)) ^ few_swz<T, D>(rw)) * 4 + (col & 3)];
#pragma unroll
                    for (int n = 0; n < NB; ++n)
                        o[n][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[n][0][i], o[n][db], 0, 0, 0);
                }
            }
        } else {
            const int r0 = 4 * g + (col >> 2), r1 = 16 + r0;
            const int s0 = piece_swz<D>(r0), s1 = piece_swz<D>(r1);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const int pc = 2 * db + ((col & 3) >> 1);
                const T* const x0 = X + r0 * LD + ((pc ^ s0) << 3) + (col & 1) * 4;
                const T* const x1 = X + r1 * LD + ((pc ^ s1) << 3) + (col & 1) * 4;
                const uint2 lo2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)x0));
                const uint2 hi2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)x1));
                const uint4 x = make_uint4(lo2.x, lo2.y, hi2.x, hi2.y);
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n][db] = Mma<T>::run(x, p[n], o[n][db]);
            }
        }
    }
    // the four waves' parts, through the LDS that held their values
    float* const parts = reinterpret_cast<float*>(lds);  // [4][rows][D]
    lds_publish_barrier();
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        float* const ow = parts + (wave * kRowsOf + 16 * n + col) * D;
        float total = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            *reinterpret_cast<f32x4_t*>(ow + 16 * db + 4 * g) = o[n][db];
            total += (o[n][db][0] + o[n][db][1]) + (o[n][db][2] + o[n][db][3]);
        }
        l[n] = sum_rows(l[n]);
        unsigned long long rows = __ballot(total != total);
        rows |= rows >> 32;
        if (g == 0) {
            ml[wave][16 * n + col][0] = m[n];
            ml[wave][16 * n + col][1] = l[n];
            bad[wave][n] = static_cast<uint32_t>(rows | rows >> 16) & 0xffffu;
        }
    }
    lds_publish_barrier();
    const bool any = __ballot(lane < 4 * NB && (&bad[0][0])[lane] != 0) != 0;
    // A row's maximum and sum over the waves, each wave's weight.
    auto joined = [&](int rw, float& mt, float& lt, float (&wt)[4]) {
        mt = fmaxp(fmaxp(ml[0][rw][0], ml[1][rw][0]), fmaxp(ml[2][rw][0], ml[3][rw][0]));
        const float ref = mt == -INFINITY ? 0.f : mt;
        lt = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            wt[w] = __builtin_amdgcn_exp2f(ml[w][rw][0] - ref);
            lt = fmaf(wt[w], ml[w][rw][1], lt);
        }
    };
    // Rows to be summed again: not where the scores themselves are not finite.
    // A row without a key (sum 0) is, to zeros.
    auto later = [&](int rw, float mt, float lt) {
        const int n = rw >> 4;
        const uint32_t rows = bad[0][n] | bad[1][n] | bad[2][n] | bad[3][n];
        return ((rows >> (rw & 15)) & 1) && (lt == 0.f || (!item_nonfinite(mt) && !item_nonfinite(lt)));
    };
#pragma unroll 1
    for (int e = threadIdx.x; e < r.rows * (D / 4); e += kPagedThreads) {
        const int rw = e / (D / 4), d = 4 * (e - rw * (D / 4));
        float mt, lt, wt[4];
        joined(rw, mt, lt, wt);
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) x += wt[w] * *reinterpret_cast<const f32x4_t*>(parts + (w * kRowsOf + rw) * D + d);
        if (!any || !later(rw, mt, lt)) put_four<T>(a, r, rw, d, x, lt);
        if (d == 0) {
            if (r.split) {
                const long long at = static_cast<long long>(r.index) * kRowsOf + rw;
                a.ml[2 * at] = mt;
                a.ml[2 * at + 1] = lt;
            } else {
                int i, hq;
                row_token(a, r.cls, r.h, r.row0 + rw, i, hq);
                a.lse[r.b * a.ll.b + i * a.ll.s2 + hq * a.ll.h] = row_lse(mt, lt);
            }
        }
    }
    if (any) {
        redo_rows<T, D>(r, lds, [&](int rw, float& mt, float& lt) {
            float wt[4];
            joined(rw, mt, lt, wt);
            return later(rw, mt, lt);
        });
    }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef long long i64x2_t __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ f32x16_t mma32(uint4 a, uint4 b, f32x16_t c) {
    if constexpr (std::is_same<T, bf16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
}

// Swizzles of the chunk kernel's LDS rows (16-byte pieces).  Keys: 16 rows of
// one piece on distinct banks; values: the 8 rows x 2 pairs of pieces of a
// transposing read.
template <int LD>
__device__ __forceinline__ int key_swz(int row) {
    if constexpr (LD == 128) return row & 15;
    else if constexpr (LD == 64) return (row >> 1) & 7;
    else return (row >> 2) & 3;
}

template <int LD>
__device__ __forceinline__ int value_swz(int row) {
    if constexpr (LD == 128) return (row & 7) << 1;
    else if constexpr (LD == 64) return ((row >> 1) & 3) << 1;
    else return ((row >> 2) & 1) << 1;
}

// The other half-wave's value of the same query.
__device__ __forceinline__ float other_half(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? x[0] : x[1]);
}

// 128 QB rows a workgroup: a wave has 32 QB queries (columns of 32x32x16
// products), all waves the same 64 keys, staged in LDS twice over.  As in
// k_paged_few, scores are K Q^T and results V^T P^T, so that the packed
// probabilities are the second product's operand as they lie: of the 16
// accumulators of a 32-key block, half-wave h holds keys 8 (i / 4) + 4 h +
// i % 4, and the values' operand is read (transposed) in that order.
//
// 4096 tokens over 32096 keys, 16/4 heads of 128, two requests: 1.89 to 2.2 ms
// (735 to 860 TFLOP/s; a large matrix product reaches 1257 on this card, both
// at the clock that power leaves).  Products keep the matrix cores 39 % busy
// and the softmax the vector ALUs 45 %; the two waves of a SIMD wait for LDS
// reads and the barrier of a tile in the rest: the four waves read 128 KB a
// step, about as many LDS cycles as the products take.  A step of 64 keys at
// heads of 64 takes 1.25 us where a tile has its compute unit alone, 1.57
// where two share it, and a tile some 8 us besides.  DEPTH 2 keeps two tiles'
// loads in flight, for tiles of one block, whose step is shorter than a trip
// to memory.
constexpr int kChunkKeys = 64;

template <typename T, int D, int QB, int DEPTH>
__global__ __launch_bounds__(kPagedThreads, DEPTH == 2 ? 3 : 2) void k_paged_chunk(PagedArgs a) {
    constexpr int C = D / 16, LD = row_elems<D>(), DT = D / 32;
    constexpr int PR = D / 8;                                // pieces of a row
    constexpr int kLoads = kChunkKeys * PR / kPagedThreads;  // of a thread, keys and values each
    constexpr int kTile = kChunkKeys * LD, kOffs = DEPTH + 1;
    __shared__ i64x2_t off[kOffs][kChunkKeys];  // of a key's row in the key and value pages
    __shared__ int live[kOffs][kChunkKeys];
    __shared__ float fin[128 * QB][2];  // a row's maximum and sum, at the end
    __shared__ uint32_t bad[4 * QB];    // rows to be summed again, 32 a word
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    T* const ks = reinterpret_cast<T*>(lds);
    T* const vs = ks + 2 * kTile;
    clear_padding<T>(a);
    Share r;
    if (!find_share(a, r)) return;
    if (r.rows <= 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, h = lane >> 5;
    const ScaleParts sp = scale_parts<T>(a.scale);
    const int* const table = a.table + r.b * a.table_stride;
    const T* const kb = static_cast<const T*>(a.k) + r.h * a.kh;
    const T* const vb = static_cast<const T*>(a.v) + r.h * a.vh;
    const int wrow = 32 * QB * wave;  // the wave's first row in the tile
    uint4 qf[QB][C];
    int hi[QB];
    const uint32_t reach = a.K ? a.K - 1 : 0x7fffffffu;  // keys behind a query's own
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int row = r.row0 + imin(wrow + 32 * b + col, r.rows - 1);
        int qi, qh;
        row_token(a, r.cls, r.h, row, qi, qh);
        const T* const q = static_cast<const T*>(a.q) + r.b * a.lq.b + qi * a.lq.s2 + qh * a.lq.h;
#pragma unroll
        for (int c = 0; c < C; ++c) qf[b][c] = scaled(*reinterpret_cast<const uint4*>(q + 16 * c + 8 * h), sp);
        hi[b] = r.w0 + fdiv(row, a.frep);
    }
    // what some and what all rows of the wave see
    const int wf = r.w0 + fdiv(r.row0 + imin(wrow, r.rows - 1), a.frep);
    const int wl = r.w0 + fdiv(r.row0 + imin(wrow + 32 * QB, r.rows) - 1, a.frep);
    const int some_lo = first_key(a, wf), all_lo = first_key(a, wl);
    const bool idle = wrow >= r.rows;
    const int steps = (r.u_hi - r.u_lo + kChunkKeys) / kChunkKeys;

    // Where tile st's keys are (the pool's first slot where no page holds one:
    // live 0), by the waves in turn.  The page number is asked for well before
    // it is used, the offsets lie in LDS a step before they are.
    int page = 0, slot = 0;
    bool in = false;
    auto ask = [&](int st) {
        const int u = r.u_lo + st * kChunkKeys + lane;
        in = u <= r.u_hi;
        const int j = r.c + imin(u, r.u_hi) * a.dil, pg = fdiv(j, a.fpage);
        slot = j - pg * a.page_size;
        page = table[pg];
    };
    auto locate = [&](int st) {
        const bool ok = in && page >= 0 && page < a.pages;
        const int pg = ok ? page : 0, sl = ok ? slot : 0;
        off[st % kOffs][lane] = i64x2_t{pg * a.kp + sl * a.ks, pg * a.vp + sl * a.vs};
        live[st % kOffs][lane] = ok;
    };
    auto row_of = [&](int i) { return (tid + i * kPagedThreads) / PR; };
    auto piece_of = [&](int i) { return (tid + i * kPagedThreads) % PR; };
    auto find = [&](int st, i64x2_t (&x)[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) x[i] = off[st % kOffs][row_of(i)];
    };
    auto load = [&](const i64x2_t (&x)[kLoads], u32x4_t (&kv)[2][kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            kv[0][i] = *reinterpret_cast<const u32x4_t*>(kb + 8 * piece_of(i) + x[i].x);
            kv[1][i] = *reinterpret_cast<const u32x4_t*>(vb + 8 * piece_of(i) + x[i].y);
        }
    };
    auto store = [&](int st, bool whole, const u32x4_t (&kv)[2][kLoads]) {
        // values that are not there must not be: 0 times them is in the sum
        uint32_t keep[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) keep[i] = 0xffffffffu;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) keep[i] = live[st % kOffs][row_of(i)] ? 0xffffffffu : 0u;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int rw = row_of(i), pc = piece_of(i);
            *reinterpret_cast<u32x4_t*>(ks + (st & 1) * kTile + rw * LD + ((pc ^ key_swz<LD>(rw)) << 3)) = kv[0][i];
            *reinterpret_cast<u32x4_t*>(vs + (st & 1) * kTile + rw * LD + ((pc ^ value_swz<LD>(rw)) << 3)) =
                kv[1][i] & keep[i];
        }
    };
    auto present = [&](int st) { return __ballot(live[st % kOffs][lane] != 0); };
    // A lane's places in a tile's rows: the swizzles repeat every 16 (keys)
    // and 8 (values) rows, so the rest of an address is constant.
    int kat[C], vat[DT];
#pragma unroll
    for (int c = 0; c < C; ++c) kat[c] = col * LD + (((2 * c + h) ^ key_swz<LD>(col)) << 3);
    const int vr = 4 * h + ((lane & 15) >> 2), vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int t = 0; t < DT; ++t) vat[t] = vr * LD + (((4 * t + vc) ^ value_swz<LD>(vr)) << 3) + (lane & 1) * 4;

    float m[QB], l[QB];
    f32x16_t o[QB][DT];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        m[b] = -INFINITY;
        l[b] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][t][i] = 0.f;
    }
    unsigned long long have = 0;
    u32x4_t buf[DEPTH][2][kLoads];
    if (steps > 0) {
        // tile 0 into LDS; with two in flight, tile 1 on its way
        if (wave < kOffs && wave < steps) {
            ask(wave);
            locate(wave);
        }
        lds_publish_barrier();
        have = present(0);
        i64x2_t x[kLoads];
        find(0, x);
        load(x, buf[0]);
        store(0, false, buf[0]);
        if (DEPTH == 2 && steps > 1) {
            find(1, x);
            load(x, buf[0]);
        }
        lds_publish_barrier();
    }

    // One tile: `next` goes into LDS at its end (with DEPTH 1, loaded at its
    // start), `after` is loaded at its start with DEPTH 2.
    auto step = [&](int st, u32x4_t (&next)[2][kLoads], u32x4_t (&after)[2][kLoads]) {
        const bool more = st + 1 < steps, loads = st + DEPTH < steps;
        const bool asks = st + kOffs < steps && wave == (st & 3);
        unsigned long long have_next = 0;
        i64x2_t x[kLoads];
        if (loads) find(st + DEPTH, x);
        if (more) have_next = present(st + 1);
        const int ub = r.u_lo + st * kChunkKeys;
        const T* const K = ks + (st & 1) * kTile;
        const T* const V = vs + (st & 1) * kTile;
        const bool busy = !idle && ub <= wl && ub + kChunkKeys - 1 >= some_lo;
        f32x16_t s[QB][2];
        if (busy) {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kb2 = 0; kb2 < 2; ++kb2) {
#pragma unroll
                for (int b = 0; b < QB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[b][kb2][i] = 0.f;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint4 kf = *reinterpret_cast<const uint4*>(K + kat[c] + 32 * kb2 * LD);
#pragma unroll
                    for (int b = 0; b < QB; ++b) s[b][kb2] = mma32<T>(kf, qf[b][c], s[b][kb2]);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
        // loads go out behind the scores' products, the page number first:
        // waiting for it then waits for no keys
        if (asks) ask(st + kOffs);
        if (loads) load(x, DEPTH == 2 ? after : next);
        if (busy) {
            if (have != ~0ull || ub + kChunkKeys - 1 > wf || ub < all_lo) {
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    // keys ahead of the query count as far behind it
                    const uint32_t back = static_cast<uint32_t>(hi[b] - ub - 4 * h);
#pragma unroll
                    for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (back - (32 * kb2 + 8 * (i / 4) + (i & 3)) > reach) s[b][kb2][i] = -INFINITY;
                }
                if (have != ~0ull) {
#pragma unroll
                    for (int kb2 = 0; kb2 < 2; ++kb2) {
                        const uint32_t bits = static_cast<uint32_t>(have >> (32 * kb2)) >> (4 * h);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
#pragma unroll
                            for (int b = 0; b < QB; ++b)
                                if (!((bits >> (8 * (i / 4) + (i & 3))) & 1)) s[b][kb2][i] = -INFINITY;
                    }
                }
            }
            float ref[QB];
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                float top = fmaxp(s[b][0][0], s[b][1][0]);
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxp(top, fmaxp(s[b][0][i], s[b][1][i]));
                top = fmaxp(top, other_half(top)) * sp.sc2;
                const bool raise = top > m[b] + (kSlack + kCarry<T>);
                if (__ballot(raise)) {
                    const float m2 = raise ? top - kCarry<T> : m[b];
                    const float keep = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[b] - m2);
                    m[b] = m2;
                    l[b] *= keep;
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[b][t] *= keep;
                }
                ref[b] = m[b] == -INFINITY ? 0.f : m[b];
            }
            // 16 keys at a time: the next ones' exponentials beside these
            // ones' products
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint4 p[QB];
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(fmaf(s[b][kk >> 1][8 * (kk & 1) + i], sp.sc2, -ref[b]));
                        l[b] += e[i];
                    }
                    p[b] = make_uint4(Mma<T>::pack(e[0], e[1]), Mma<T>::pack(e[2], e[3]), Mma<T>::pack(e[4], e[5]),
                                      Mma<T>::pack(e[6], e[7]));
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const T* const x0 = V + vat[t] + 16 * kk * LD;
                    const uint2 lo2 =
                        __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)x0));
                    const uint2 hi2 =
                        __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(x0 + 8 * LD)));
                    const uint4 vf = make_uint4(lo2.x, lo2.y, hi2.x, hi2.y);
#pragma unroll
                    for (int b = 0; b < QB; ++b) o[b][t] = mma32<T>(vf, p[b], o[b][t]);
                }
            }
        }
        if (more) store(st + 1, have_next == ~0ull, next);
        // the offsets of tile st + kOffs replace those of tile st
        if (asks) locate(st + kOffs);
        have = have_next;
        lds_publish_barrier();
    };
    if constexpr (DEPTH == 1) {
        for (int st = 0; st < steps; ++st) step(st, buf[0], buf[0]);
    } else {
        for (int st = 0; st < steps; st += 2) {
            step(st, buf[0], buf[DEPTH - 1]);
            if (st + 1 < steps) step(st + 1, buf[DEPTH - 1], buf[0]);
        }
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int rw = wrow + 32 * b + col;
        const float lt = l[b] + other_half(l[b]);
        float total = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) total += o[b][t][i];
        // Rows to be summed again: not where the scores themselves are not
        // finite.  A row without a key (sum 0) is, to zeros.
        unsigned long long later = __ballot(total != total);
        later |= later >> 32 | later << 32;
        later &= __ballot(rw < r.rows && (lt == 0.f || (!item_nonfinite(m[b]) && !item_nonfinite(lt))));
        if (h == 0) {
            fin[rw][0] = m[b];
            fin[rw][1] = lt;
            bad[QB * wave + b] = static_cast<uint32_t>(later);
        }
        if (rw >= r.rows) continue;
        int qi, qh;
        row_token(a, r.cls, r.h, r.row0 + rw, qi, qh);
        if (h == 0) {
            if (r.split) {
                const long long at = static_cast<long long>(r.index) * a.M + rw;
                a.ml[2 * at] = m[b];
                a.ml[2 * at + 1] = lt;
            } else {
                a.lse[r.b * a.ll.b + qi * a.ll.s2 + qh * a.ll.h] = row_lse(m[b], lt);
            }
        }
        if ((later >> lane) & 1) continue;
        if (r.split) {
            float* const part = a.part + (static_cast<long long>(r.index) * a.M + rw) * D + 4 * h;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float4*>(part + 8 * n) =
                    make_float4(o[b][n / 4][4 * (n & 3)], o[b][n / 4][4 * (n & 3) + 1], o[b][n / 4][4 * (n & 3) + 2],
                                o[b][n / 4][4 * (n & 3) + 3]);
            continue;
        }
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        T* const out = static_cast<T*>(a.out) + r.b * a.lo.b + qi * a.lo.s2 + qh * a.lo.h + 4 * h;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<uint2*>(out + 8 * n) =
                make_uint2(Mma<T>::pack(o[b][n / 4][4 * (n & 3)] * inv, o[b][n / 4][4 * (n & 3) + 1] * inv),
                           Mma<T>::pack(o[b][n / 4][4 * (n & 3) + 2] * inv, o[b][n / 4][4 * (n & 3) + 3] * inv));
    }
    lds_publish_barrier();
    uint32_t any = 0;
#pragma unroll
    for (int n = 0; n < 4 * QB; ++n) any |= bad[n];
    if (__builtin_amdgcn_readfirstlane(any)) {
        redo_rows<T, D>(r, lds, [&](int rw, float& mt, float& lt) {
            mt = fin[rw][0];
            lt = fin[rw][1];
            return ((bad[rw >> 5] >> (rw & 31)) & 1) != 0;
        });
    }
}

// ---------------------------------------------------------------------------
// joining parts
// ---------------------------------------------------------------------------

constexpr int kJoinThreads = 1024;  // at most

// A running (m, l, acc) and one more part's, m base 2; a part without keys
// (m = -inf, l = 0, zeros) changes nothing.
struct Joined {
    float m = -INFINITY, l = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(float m1, float l1, f32x4_t x) {
        const float m2 = fmaxp(m, m1), ref = m2 == -INFINITY ? 0.f : m2;
        const float w0 = __builtin_amdgcn_exp2f(m - ref), w1 = __builtin_amdgcn_exp2f(m1 - ref);
        m = m2;
        l = l * w0 + l1 * w1;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = acc[e] * w0 + x[e] * w1;
    }
};

__device__ __forceinline__ f32x4_t four_of(const float* p, int d, int dim) {
    if (dim % 4 == 0) return *reinterpret_cast<const f32x4_t*>(p + d);
    f32x4_t x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d + e < dim ? p[d + e] : 0.f;
    return x;
}

// Head dims in fours on consecutive lanes.  With WIDE, the groups of lanes
// take different parts of one row (low tiles, many parts) and meet in LDS;
// otherwise each takes a row of its own (tall tiles, few parts).  Either way
// a thread joins its parts in order, so that results do not depend on which
// workgroup ended first.  The parts come from other XCDs' writes, a trip to
// memory each: the record is read beside the count, maxima beside sums and
// results.
template <typename T, bool WIDE>
__global__ __launch_bounds__(WIDE ? kJoinThreads : kPagedThreads) void k_paged_join(PagedArgs a) {
    __shared__ float o[WIDE ? kJoinThreads : 1][7];
    const int tid = threadIdx.x, quads = (a.Dv + 3) >> 2;
    const int groups = static_cast<int>(blockDim.x) / quads;
    const int g = tid / quads, d = 4 * (tid - g * quads);
    const PagedTile t = a.tiles[blockIdx.x];
    if (static_cast<int>(blockIdx.x) >= *a.count || t.parts <= 1) return;
    const int row = WIDE ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.y) * groups + g;
    if (WIDE && row >= t.rows) return;
    Joined j;
    if (g < groups && row < t.rows) {
#pragma unroll 8
        for (int s = WIDE ? g : 0; s < t.parts; s += WIDE ? groups : 1) {
            const long long at = (t.first + static_cast<long long>(s) * t.step) * a.M + row;
            j.add(a.ml[2 * at], a.ml[2 * at + 1], four_of(a.part + at * a.Dv, d, a.Dv));
        }
    }
    if constexpr (WIDE) {
        o[tid][0] = j.m;
        o[tid][1] = j.l;
        for (int e = 0; e < 4; ++e) o[tid][2 + e] = j.acc[e];
        lds_publish_barrier();
        // eight groups join theirs with every eighth one's, then the first
        // joins the eight
        if (g < 8) {
            for (int s = g + 8; s < groups; s += 8) {
                const float* const p = o[s * quads + tid - g * quads];
                j.add(p[0], p[1], f32x4_t{p[2], p[3], p[4], p[5]});
            }
        }
        lds_publish_barrier();
        if (g < 8) {
            o[tid][0] = j.m;
            o[tid][1] = j.l;
            for (int e = 0; e < 4; ++e) o[tid][2 + e] = j.acc[e];
        }
        lds_publish_barrier();
        if (g != 0) return;
        for (int s = 1; s < 8 && s < groups; ++s) {
            const float* const p = o[s * quads + tid];
            j.add(p[0], p[1], f32x4_t{p[2], p[3], p[4], p[5]});
        }
    } else if (g >= groups || row >= t.rows) {
        return;
    }
    int i, hq;
    row_token(a, t.cls, t.h, t.row0 + row, i, hq);
    const float inv = j.l == 0.f ? 0.f : 1.f / j.l;
    T* const out = static_cast<T*>(a.out) + t.b * a.lo.b + i * a.lo.s2 + hq * a.lo.h + d;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < a.Dv) out[e] = from_f<T>(j.acc[e] * inv);
    if (d == 0) a.lse[t.b * a.ll.b + i * a.ll.s2 + hq * a.ll.h] = row_lse(j.m, j.l);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Workgroups aimed at when the tiles are few: two a compute unit.
constexpr int kTarget = 512;

// Rows of cut tiles up to which a workgroup joins each (k_paged_join WIDE);
// more take a group of lanes each.  Tiles x rows, WIDE / not, us: 32 x 4 5 /
// 11, 64 x 12 5 / 8, 256 x 4 5 / 5, 64 x 64 12 / 8, 64 x 128 20 / 8.
constexpr unsigned kWideRows = 1024;

// Rows of a class up to which k_paged_few takes them on one read of the keys;
// more take the tall tiles.  32 requests over up to 16384 keys, few / chunk
// kernel with their joins, us: heads of 128, 32 rows 256 / 266, 64 rows 429 /
// 286; heads of 64, 32 rows 40 / 53, 64 rows 51 / 55, 96 rows 77 / 58.
constexpr int few_rows(int dim) { return dim <= 64 ? 64 : 32; }

enum PagedKind { kRows, kFew, kChunk };

struct PagedPlan {
    PagedKind kind;
    int blocks;  // query blocks of a wave
    int M, KT, least, xcd_run;
    long long rows;   // of a class, at most
    long long tiles;  // tile slots of the batch
    int slots;        // of a (sequence, kv head)
    bool split;       // some tile's keys may be cut
    long long grid;
    size_t bytes;     // workspace
};

constexpr int exponent_of(int n) { return n <= 1 ? 0 : 1 + exponent_of(n / 2); }

long long padded(long long bytes) { return (bytes + 255) & ~255ll; }

// MFMA kernels: equal head dims that they are built for, operands read and
// written in 16-byte vectors.
bool on_mfma(const PagedCall& c) {
    const int d = c.dim_qk;
    return c.vec && d == c.cache.dim_v && (d == 32 || d == 64 || d == 96 || d == 128);
}

PagedPlan plan(const PagedCall& c) {
    PagedPlan p{};
    const long long rep = c.heads_q / c.heads_kv;
    const long long dil = c.dilation, classes = c.tokens < dil ? c.tokens : dil;
    const long long members = (c.tokens + dil - 1) / dil;
    p.kind = !on_mfma(c) ? kRows : members * rep <= few_rows(c.dim_qk) || c.dtype == NATTEN_F32 ? kFew : kChunk;
    const long long rows = p.rows = members * rep;
    if (p.kind == kChunk) {
        // 64 queries a wave where their accumulators leave two waves a SIMD
        // and the tiles still fill the device: half the reads of LDS for each
        // product (2048 tokens in a window of 1025, heads of 64, one / two
        // blocks: 8 requests, 512 tall tiles, 72 / 64 us; 4 requests 41 / 44)
        const long long tall = classes * ((rows + 255) / 256) * c.batch * c.heads_kv;
        p.blocks = c.dim_qk <= 64 && tall >= kTarget ? 2 : 1;
        p.M = 128 * p.blocks;
        p.KT = kChunkKeys;
        // 2048 keys: parts of 128 rows and their join cost as much as 1000
        // keys take (17 blocks whole 42 us, in two parts 32 + 9)
        p.least = 32;
    } else if (p.kind == kFew) {
        // one read of the keys for all rows, if the registers hold them (40
        // rows of 64 dims: 19 us, as three tiles of 16 23)
        p.blocks = rows <= 16 ? 1 : rows <= 32 || c.dim_qk > 64 ? 2 : 4;
        p.M = kFewRows * p.blocks;
        p.KT = 4 * (c.dtype == NATTEN_F32 ? few_keys<float>() : few_keys<bf16>());
        p.least = 256 / p.KT;
    } else {
        p.M = 4;
        p.KT = 64;
        p.least = 4;
    }
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
    if (p.kind == kChunk) {
        // runs of tiles on one XCD, 4 or more on each; whole rounds of them
        p.xcd_run = static_cast<int>(p.grid / 32 < 1 ? 1 : p.grid / 32 > 16 ? 16 : p.grid / 32);
        p.grid = (p.grid + 8 * p.xcd_run - 1) / (8 * p.xcd_run) * (8 * p.xcd_run);
    }
    return p;
}

// LDS of k_paged_few: the waves' values, then their results.
template <typename T, int D>
constexpr size_t few_lds(int blocks) {
    const size_t values = 4 * few_keys<T>() * row_elems<D>() * sizeof(T), results = 4 * kFewRows * blocks * D * sizeof(float);
    return values > results ? values : results;
}

template <typename T, int D>
hipError_t launch_mfma(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
    const dim3 grid = wide_grid(p.grid), block(kPagedThreads);
    if constexpr (!std::is_same<T, float>::value) {
        if (p.kind == kChunk) {
            constexpr int lds = 2 * 2 * kChunkKeys * row_elems<D>() * sizeof(T);
            if constexpr (D <= 64) {
                if (p.blocks == 2)
                    NA_LAUNCH("na_paged_chunk", (k_paged_chunk<T, D, 2, 1>), grid, block, lds, s, a);
                else
                    NA_LAUNCH("na_paged_chunk", (k_paged_chunk<T, D, 1, 2>), grid, block, lds, s, a);
            } else {
                NA_LAUNCH("na_paged_chunk", (k_paged_chunk<T, D, 1, 1>), grid, block, lds, s, a);
            }
            return hipGetLastError();
        }
    }
    if constexpr (D <= 64) {
        if (p.blocks == 4) {
            NA_LAUNCH("na_paged_few", (k_paged_few<T, D, 4>), grid, block, (few_lds<T, D>(4)), s, a);
            return hipGetLastError();
        }
    }
    if (p.blocks == 2)
        NA_LAUNCH("na_paged_few", (k_paged_few<T, D, 2>), grid, block, (few_lds<T, D>(2)), s, a);
    else
        NA_LAUNCH("na_paged_few", (k_paged_few<T, D, 1>), grid, block, (few_lds<T, D>(1)), s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_kind(const PagedArgs& a, const PagedPlan& p, bool vec, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (p.kind == kRows) {
        constexpr int kVec = 16 / sizeof(T);
        if (vec)
            NA_LAUNCH("na_paged_rows", (k_paged_rows<T, kVec>), wide_grid(p.grid), dim3(kPagedThreads), 0, s, a);
        else
            NA_LAUNCH("na_paged_rows", (k_paged_rows<T, 1>), wide_grid(p.grid), dim3(kPagedThreads), 0, s, a);
        e = hipGetLastError();
    } else {
        if (a.Dqk == 32) e = launch_mfma<T, 32>(a, p, s);
        else if (a.Dqk == 64) e = launch_mfma<T, 64>(a, p, s);
        else if (a.Dqk == 96) e = launch_mfma<T, 96>(a, p, s);
        else e = launch_mfma<T, 128>(a, p, s);
    }
    if (e != hipSuccess || !p.split) return e;
    const unsigned tiles = static_cast<unsigned>(p.tiles < kTarget ? p.tiles : kTarget);
    const unsigned rows = static_cast<unsigned>(std::min<long long>(p.M, p.rows));
    if (tiles * rows > kWideRows) {
        const unsigned groups = kPagedThreads / ((a.Dv + 3) / 4);
        NA_LAUNCH("na_paged_join", (k_paged_join<T, false>), dim3(tiles, (rows + groups - 1) / groups),
                  dim3(kPagedThreads), 0, s, a);
    } else {
        // the fewer the tiles, the more parts has each: groups of lanes
        // enough that each joins a handful (513 parts of one tile: 15 us with
        // 256 threads, 6 with 1024; 256 tiles of 4 rows, 9 parts: 5 and 11)
        const int threads = tiles <= 16 ? kJoinThreads : kPagedThreads;
        NA_LAUNCH("na_paged_join", (k_paged_join<T, true>), dim3(tiles, rows), dim3(threads), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace

// The most that a call of this problem takes, whatever its operands' alignment.
size_t paged_workspace(const PagedCall& c) {
    PagedCall x = c;
    size_t most = 0;
    for (bool vec : {false, true}) {
        x.vec = vec;
        most = std::max(most, plan(x).bytes);
    }
    return most;
}

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
    const long long cap = static_cast<long long>(c.cache.width) * c.cache.page_size;
    a.cap = static_cast<int>(std::min<long long>(cap, 0x7fffffff));
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
    a.flen = make_fastdiv(a.L);
    a.fdv = make_fastdiv(a.Dv);
    a.K = c.kernel;
    a.dil = c.dilation;
    a.fdil = make_fastdiv(a.dil);
    a.scale = c.scale;
    a.M = p.M;
    a.log_m = exponent_of(p.M);
    a.log_kt = exponent_of(p.KT);
    a.tile_slots = p.slots;
    a.direct = p.split ? 0 : 1;
    a.log_target = exponent_of(kTarget);
    a.least = p.least;
    a.xcd_run = p.xcd_run;
    const long long waves = p.grid * (kPagedThreads / 64);
    a.per_wave = static_cast<int>((static_cast<long long>(a.B) * a.L + waves - 1) / waves);
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
    if (c.dtype == NATTEN_F32) return launch_kind<float>(a, p, c.vec, s);
    if (c.dtype == NATTEN_F16) return launch_kind<f16>(a, p, c.vec, s);
    return launch_kind<bf16>(a, p, c.vec, s);
}

}  // namespace na
