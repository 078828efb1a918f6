// Rotary positions, alone (natten_hip_rotary) and on the way into a paged
// cache (natten_hip_paged_append).
//
// A pair (u, v) of a head at coordinate p turns by t = 2 pi p f:
//   (u', v') = m (u cos t - v sin t, u sin t + v cos t),
// f in turns per position, m one factor for the whole call.  The gradient is
// the same map with -t (the transpose of a scaled rotation).  Axis a of a
// grid owns dims [2 a P, 2 (a + 1) P) of the head; inside that share, pair j
// is (j, j + P), or (2j, 2j + 1) when interleaved.  Dims past the turned ones
// pass through.
//
// Angles.  f is a 64-bit fixed-point fraction of a turn (f * 2^64 modulo 1:
// whole turns do nothing), so p f modulo a turn is the low 64 bits of an
// integer product: nothing is lost but f's own rounding, 2^-65 |p| turns with
// f the nearest such fraction.  The top 32 bits split into the nearest quarter turn and a rest
// within an eighth, where the Taylor sums of sine (to x^9) and cosine (to
// x^10) leave less than 3e-9 against an fp32 half step of 3e-8.
//
// The op reads and writes each element once, so memory bounds it.  A block
// takes `tb` consecutive tokens: it computes their cosines and sines into
// LDS once for all heads, then walks the tokens' vectors in memory order
// (lanes on consecutive 16-byte vectors), its first loads out before the
// angles.  4 x 16384 tokens of 8/2 heads of 64, bf16: 31 us (5.4 TB/s); 64 x
// 56 x 56 of 4/4 heads of 32, interleaved fp16 views: 33 us (6.2 TB/s); three
// axes of 16 dims, 32768 tokens of 8/8 heads of 64: 31 us (4.3 TB/s); 4096
// tokens of 4 prompts, 32/8 heads of 128, into pages: 53 us (4.7 TB/s).  A
// copy of as many bytes moves 4.9 to 5.2 TB/s over buffers that no cache
// holds, up to 8.5 over one pair that a cache does.
#include <type_traits>

#include "na_launch.h"

namespace na {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;           // units of a thread in flight
constexpr int kMaxTokens = 64;      // tokens per block
constexpr int kAngleFloats = 8192;  // LDS of cosines and sines per block

struct RotaryArgs {
    const void *q, *k, *v;
    void *qo, *ko, *vo;
    Lay lq, lk, lv, lqo, lko, lvo;  // paged: lko / lvo hold page (b), slot (s2) and head strides
    const uint64_t* turns;          // [pairs]
    const void* pos;
    int pos_bits;                   // 0: the grid's own coordinates
    long long pos_b, pos_t, pos_a;
    int tokens, tb;
    int per_seq, len1, len2;
    FastDiv fseq, flen2, flen1;
    FastDiv fpairs, funits, fhead, fvhead;  // turned pairs a token; units a token, a q/k head, a v head
    int hq, hk, hv;
    int dim, turned, axes, pairs;   // pairs per axis
    int half;                       // turned / 2
    float mag, dir;                 // dir -1 turns back
    // paged destination
    const int *table, *lens, *news;
    long long table_stride;
    int width, pages, page_size;
    FastDiv fpage;
};

struct SinCos {
    float s, c;
};

// Sine and cosine of `frac` 2^-32 turns.
__device__ __forceinline__ SinCos sin_cos_turns(uint32_t frac) {
    const uint32_t quarter = (frac + 0x20000000u) >> 30;
    const int rest = static_cast<int>(frac - (quarter << 30));
    const float x = static_cast<float>(rest) * 1.4629180792671596e-9f;  // 2 pi 2^-32
    const float z = x * x;
    float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    s = fmaf(z, s, 8.3333333e-3f);
    s = fmaf(z, s, -1.6666667e-1f);
    s = fmaf(x * z, s, x);
    float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    c = fmaf(z, c, -1.3888889e-3f);
    c = fmaf(z, c, 4.1666667e-2f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    SinCos r;
    r.s = quarter & 1 ? c : s;
    r.c = quarter & 1 ? s : c;
    if (quarter & 2) r.s = -r.s;
    if ((quarter + 1) & 2) r.c = -r.c;
    return r;
}

// Top 32 bits of the low 64 of f * p.
__device__ __forceinline__ uint32_t turn_fraction(uint64_t f, int64_t p) {
    return static_cast<uint32_t>((f * static_cast<uint64_t>(p)) >> 32);
}

// VEC elements as they are moved, in registers of their own.
template <int BYTES>
struct Raw;
template <>
struct Raw<16> {
    typedef uint32_t type __attribute__((ext_vector_type(4)));
};
template <>
struct Raw<8> {
    typedef uint32_t type __attribute__((ext_vector_type(2)));
};
template <>
struct Raw<4> {
    using type = uint32_t;
};
template <>
struct Raw<2> {
    using type = uint16_t;
};
template <typename T, int VEC>
using raw_t = typename Raw<sizeof(T) * VEC>::type;

template <typename T, int VEC>
struct Vec {
    T x[VEC];
};

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

template <typename T, int VEC>
__device__ __forceinline__ void spread(raw_t<T, VEC> r, float* f) {
    const Vec<T, VEC> v = __builtin_bit_cast(Vec<T , VEC>, r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f(v.x[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ raw_t<T, VEC> round_vec(const float* f) {
    if constexpr (std::is_same<T, float>::value || VEC == 1) {
        Vec<T, VEC> r;
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.x[i] = from_f<T>(f[i]);
        return __builtin_bit_cast(raw_t<T , VEC>, r);
    } else {
        using P = typename std::conditional<std::is_same<T, bf16>::value, bf16x2v, f16x2v>::type;
        struct Pairs {
            P p[VEC / 2];
        } r;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) r.p[i] = __builtin_convertvector((f32x2v{f[2 * i], f[2 * i + 1]}), P);
        return __builtin_bit_cast(raw_t<T , VEC>, r);
    }
}

template <bool STREAM, typename R>
__device__ __forceinline__ void put(R* to, R v) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(v, to);
    else
        *to = v;
}

// One unit of work: two vectors of a head that hold VEC pairs, `gap` elements
// apart (neighbours that pair up: one vector of VEC / 2 pairs, gap 0), or one
// vector that is copied (angle -1: dims that do not turn, and values).
template <typename T>
struct Unit {
    const T* src;
    T* dst;
    int gap;
    int angle;  // first pair's index among the block's angles
    int zero;   // padding: zeros are written
};

// STREAM: results go past the caches.
template <typename T, int VEC, bool INTER, bool PAGED, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a) {
    extern __shared__ float angles[];  // [tb * half] cosines, then sines
    __shared__ long long off[kMaxTokens][6];
    __shared__ int coord[kMaxTokens][3];  // paged: coord[.][0] is the position
    const int tid = threadIdx.x;
    const int t0 = wide_block() * a.tb;
    if (t0 >= a.tokens) return;
    const int nt = imin(a.tb, a.tokens - t0);

    for (int t = tid; t < nt; t += kThreads) {
        const int b = fdiv(t0 + t, a.fseq), n = t0 + t - b * a.per_seq;
        if constexpr (PAGED) {
            const int cnt = a.news ? imin(imax(a.news[b], 0), a.per_seq) : a.per_seq;
            const long long p = static_cast<long long>(a.lens[b]) - cnt + n;
            const bool live = n < cnt && p >= 0;
            off[t][0] = live ? b * a.lq.b + n * a.lq.s2 : -1;
            off[t][1] = b * a.lqo.b + n * a.lqo.s2;
            off[t][2] = b * a.lk.b + n * a.lk.s2;
            off[t][4] = b * a.lv.b + n * a.lv.s2;
            long long ko = -1, vo = -1;
            if (live) {
                const int pg = fdiv(static_cast<int>(p), a.fpage);
                if (pg < a.width) {
                    const int at = a.table[b * a.table_stride + pg];
                    if (at >= 0 && at < a.pages) {
                        const int slot = static_cast<int>(p) - pg * a.page_size;
                        ko = at * a.lko.b + slot * a.lko.s2;
                        vo = at * a.lvo.b + slot * a.lvo.s2;
                    }
                }
            }
            off[t][3] = ko;
            off[t][5] = vo;
            coord[t][0] = live ? static_cast<int>(p) : 0;
        } else {
            const int r = fdiv(n, a.flen2), i2 = n - r * a.len2;
            const int i0 = fdiv(r, a.flen1), i1 = r - i0 * a.len1;
            off[t][0] = a.lq.at(b, i0, i1, i2, 0);
            off[t][1] = a.lqo.at(b, i0, i1, i2, 0);
            off[t][2] = a.lk.at(b, i0, i1, i2, 0);
            off[t][3] = a.lko.at(b, i0, i1, i2, 0);
            coord[t][0] = i0;
            coord[t][1] = i1;
            coord[t][2] = i2;
        }
    }
    lds_publish_barrier();

    // The block's first loads go out before its angles are computed.
    using R = raw_t<T, VEC>;
    constexpr bool kOne = INTER && VEC > 1;
    const int turning = kOne ? a.turned / VEC : a.half / VEC;  // units of a head that turn
    const int uqk = (a.hq + a.hk) * static_cast<int>(a.fhead.d);
    const int total = nt * static_cast<int>(a.funits.d);
    Unit<T> u[kUnits];
    R x[kUnits], y[kUnits];
    auto fetch = [&](int e0) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int e = e0 + i * kThreads;
            u[i].dst = nullptr;
            if (e >= total) continue;
            const int t = fdiv(e, a.funits);
            int r = e - t * static_cast<int>(a.funits.d);
            u[i].zero = 0;
            u[i].gap = 0;
            u[i].angle = -1;
            if (r < uqk) {
                int h = fdiv(r, a.fhead);
                const int w = r - h * static_cast<int>(a.fhead.d);
                const bool isq = h < a.hq;
                if (!isq) h -= a.hq;
                const long long so = isq ? off[t][0] : off[t][2], to = isq ? off[t][1] : off[t][3];
                if (PAGED && !isq && to < 0) continue;
                int d;
                if (w < turning) {
                    if constexpr (kOne) {
                        u[i].angle = t * a.half + w * (VEC / 2);
                        d = w * VEC;
                    } else if constexpr (INTER) {
                        u[i].angle = t * a.half + w;
                        u[i].gap = 1;
                        d = 2 * w;
                    } else {
                        u[i].angle = t * a.half + w * VEC;
                        int ax = 0, j = w * VEC;
                        while (ax + 1 < a.axes && j >= a.pairs) {
                            j -= a.pairs;
                            ++ax;
                        }
                        d = 2 * ax * a.pairs + j;
                        u[i].gap = a.pairs;
                    }
                } else {
                    d = a.turned + (w - turning) * VEC;
                }
                u[i].zero = PAGED && isq && so < 0;
                u[i].src = static_cast<const T*>(isq ? a.q : a.k) + (so + h * (isq ? a.lq.h : a.lk.h) + d);
                u[i].dst = static_cast<T*>(isq ? a.qo : a.ko) + (to + h * (isq ? a.lqo.h : a.lko.h) + d);
            } else if (PAGED) {
                r -= uqk;
                const int h = fdiv(r, a.fvhead), w = r - h * static_cast<int>(a.fvhead.d);
                const long long to = off[t][5];
                if (to < 0) continue;
                u[i].src = static_cast<const T*>(a.v) + (off[t][4] + h * a.lv.h + w * VEC);
                u[i].dst = static_cast<T*>(a.vo) + (to + h * a.lvo.h + w * VEC);
            }
            if (!u[i].zero) {
                x[i] = *reinterpret_cast<const R*>(u[i].src);
                if (u[i].gap) y[i] = *reinterpret_cast<const R*>(u[i].src + u[i].gap);
            }
        }
    };
    fetch(tid);

    const int nangle = nt * a.half;
    float* const cosv = angles;
    float* const sinv = angles + a.tb * a.half;
    for (int e = tid; e < nangle; e += kThreads) {
        const int t = fdiv(e, a.fpairs);
        int j = e - t * a.half, ax = 0;
        while (ax + 1 < a.axes && j >= a.pairs) {
            j -= a.pairs;
            ++ax;
        }
        int64_t p;
        if constexpr (PAGED) {
            p = coord[t][0];
        } else if (a.pos_bits) {
            const int b = fdiv(t0 + t, a.fseq), n = t0 + t - b * a.per_seq;
            const long long at = b * a.pos_b + n * a.pos_t + ax * a.pos_a;
            p = a.pos_bits == 64 ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int32_t*>(a.pos)[at];
        } else {
            p = coord[t][3 - a.axes + ax];
        }
        const SinCos r = sin_cos_turns(turn_fraction(a.turns[j], p));
        cosv[e] = r.c * a.mag;
        sinv[e] = r.s * (a.mag * a.dir);
    }
    lds_publish_barrier();
    for (int e0 = tid; e0 < total; e0 += kThreads * kUnits) {
        if (e0 != tid) fetch(e0);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            if (!u[i].dst) continue;
            R* const to = reinterpret_cast<R*>(u[i].dst);
            R* const to2 = reinterpret_cast<R*>(u[i].dst + u[i].gap);
            if (u[i].zero) {
                *to = R{};
                if (u[i].gap) *to2 = R{};
                continue;
            }
            if (u[i].angle < 0) {
                put<STREAM>(to, x[i]);
                continue;
            }
            if constexpr (kOne) {
                float p[VEC], o[VEC];
                spread<T, VEC>(x[i], p);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const float c = cosv[u[i].angle + j], s = sinv[u[i].angle + j];
                    o[2 * j] = fmaf(p[2 * j], c, -(p[2 * j + 1] * s));
                    o[2 * j + 1] = fmaf(p[2 * j], s, p[2 * j + 1] * c);
                }
                put<STREAM>(to, round_vec<T, VEC>(o));
            } else {
                float p[VEC], q[VEC], o1[VEC], o2[VEC];
                spread<T, VEC>(x[i], p);
                spread<T, VEC>(y[i], q);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float c = cosv[u[i].angle + j], s = sinv[u[i].angle + j];
                    o1[j] = fmaf(p[j], c, -(q[j] * s));
                    o2[j] = fmaf(p[j], s, q[j] * c);
                }
                put<STREAM>(to, round_vec<T, VEC>(o1));
                put<STREAM>(to2, round_vec<T, VEC>(o2));
            }
        }
    }
}

template <typename T, int VEC, bool PAGED>
hipError_t launch(const RotaryArgs& a, bool inter, bool stream, hipStream_t s) {
    const dim3 grid = wide_grid((static_cast<long long>(a.tokens) + a.tb - 1) / a.tb), block(kThreads);
    const size_t shm = sizeof(float) * 2 * static_cast<size_t>(a.tb) * a.half;
    const char* const name = PAGED ? "na_paged_append" : "na_rotary";
    if constexpr (VEC > 1) {
        if (stream) {
            if (inter)
                NA_LAUNCH(name, (k_rotary<T, VEC, true, PAGED, true>), grid, block, shm, s, a);
            else
                NA_LAUNCH(name, (k_rotary<T, VEC, false, PAGED, true>), grid, block, shm, s, a);
            return hipGetLastError();
        }
    }
    if (inter)
        NA_LAUNCH(name, (k_rotary<T, VEC, true, PAGED, false>), grid, block, shm, s, a);
    else
        NA_LAUNCH(name, (k_rotary<T, VEC, false, PAGED, false>), grid, block, shm, s, a);
    return hipGetLastError();
}

template <bool PAGED>
hipError_t launch_any(RotaryArgs& a, int dtype, int vec, bool inter, int dim_v, hipStream_t s) {
    a.half = a.turned / 2;
    a.pairs = a.half / a.axes;
    // units of a head: see k_rotary
    const int turning = inter && vec > 1 ? a.turned / vec : a.half / vec;
    const int uh = turning + (a.dim - a.turned) / vec, uv = PAGED ? dim_v / vec : 0;
    const int units = (a.hq + a.hk) * uh + a.hv * uv;
    const int elem = dtype == NATTEN_F32 ? 4 : 2;
    a.fpairs = make_fastdiv(imax(a.half, 1));
    a.fhead = make_fastdiv(imax(uh, 1));
    a.fvhead = make_fastdiv(imax(uv, 1));
    a.funits = make_fastdiv(units);
    // Tokens per block: up to a batch of units a thread, as long as that leaves
    // four blocks a compute unit; the angles of a block fit their LDS.
    int tb = 1;
    while (tb < kMaxTokens && 2 * tb * units <= kThreads * kUnits && 2 * tb * 1024 <= a.tokens) tb *= 2;
    while (tb > 1 && 2 * tb * a.half > kAngleFloats) tb /= 2;
    a.tb = tb;
    // Results that no cache can hold for their reader are stored past them,
    // if a store instruction writes runs of 64 bytes: 168 MB at heads of 64
    // (runs of 64) 36 -> 31 us, 205 MB interleaved 44 -> 34 us; at runs of 16
    // bytes (three axes of 16 dims) it would be 31 -> 67 us.
    const long long bytes = static_cast<long long>(elem) * a.tokens *
                            (static_cast<long long>(a.hq + a.hk) * a.dim + static_cast<long long>(a.hv) * dim_v);
    const int rest = a.dim - a.turned;
    const bool stream = bytes >= (32ll << 20) && (inter || a.pairs * elem >= 64) && (!rest || rest * elem >= 64);
    if (dtype == NATTEN_F32) {
        if (vec == 4) return launch<float, 4, PAGED>(a, inter, stream, s);
        return launch<float, 1, PAGED>(a, inter, stream, s);
    }
    if (dtype == NATTEN_F16) {
        if (vec == 8) return launch<f16, 8, PAGED>(a, inter, stream, s);
        if (vec == 4) return launch<f16, 4, PAGED>(a, inter, stream, s);
        return launch<f16, 1, PAGED>(a, inter, stream, s);
    }
    if (vec == 8) return launch<bf16, 8, PAGED>(a, inter, stream, s);
    if (vec == 4) return launch<bf16, 4, PAGED>(a, inter, stream, s);
    return launch<bf16, 1, PAGED>(a, inter, stream, s);
}

}  // namespace

hipError_t rotary(const RotaryCall& c, hipStream_t s) {
    RotaryArgs a{};
    a.q = c.q;
    a.k = c.k;
    a.qo = c.qo;
    a.ko = c.ko;
    a.lq = c.lq;
    a.lk = c.lk;
    a.lqo = c.lqo;
    a.lko = c.lko;
    a.turns = c.turns;
    a.pos = c.pos;
    a.pos_bits = c.pos_bits;
    a.pos_b = c.pos_stride[0];
    a.pos_t = c.pos_stride[1];
    a.pos_a = c.pos_stride[2];
    a.per_seq = c.len[0] * c.len[1] * c.len[2];
    a.tokens = c.batch * a.per_seq;
    a.len1 = c.len[1];
    a.len2 = c.len[2];
    a.fseq = make_fastdiv(a.per_seq);
    a.flen1 = make_fastdiv(a.len1);
    a.flen2 = make_fastdiv(a.len2);
    a.hq = c.heads_q;
    a.hk = c.heads_k;
    a.dim = c.dim;
    a.turned = c.turned;
    a.axes = c.axes;
    a.mag = c.magnitude;
    a.dir = c.inverse ? -1.f : 1.f;
    return launch_any<false>(a, c.dtype, c.vec, c.interleaved, 0, s);
}

hipError_t paged_append(const PagedCache& c, const RotaryCall& r, const void* v, Lay lv, hipStream_t s) {
    RotaryArgs a{};
    a.q = r.q;
    a.k = r.k;
    a.v = v;
    a.qo = r.qo;
    a.ko = const_cast<void*>(c.k);
    a.vo = const_cast<void*>(c.v);
    a.lq = r.lq;
    a.lk = r.lk;
    a.lv = lv;
    a.lqo = r.lqo;
    a.lko.b = c.ks[0];
    a.lko.s2 = c.ks[1];
    a.lko.h = c.ks[2];
    a.lvo.b = c.vs[0];
    a.lvo.s2 = c.vs[1];
    a.lvo.h = c.vs[2];
    a.turns = r.turns;
    a.per_seq = r.len[2];
    a.tokens = r.batch * a.per_seq;
    a.len1 = 1;
    a.len2 = r.len[2];
    a.fseq = make_fastdiv(a.per_seq);
    a.flen1 = make_fastdiv(1);
    a.flen2 = make_fastdiv(a.len2);
    a.hq = r.heads_q;
    a.hk = r.heads_k;
    a.hv = r.heads_k;
    a.dim = r.dim;
    a.turned = r.turned;
    a.axes = 1;
    a.mag = r.magnitude;
    a.dir = 1.f;
    a.table = c.table;
    a.lens = c.lens;
    a.news = c.news;
    a.table_stride = c.table_stride;
    a.width = c.width;
    a.pages = c.pages;
    a.page_size = c.page_size;
    a.fpage = make_fastdiv(c.page_size);
    return launch_any<true>(a, r.dtype, r.vec, r.interleaved, c.dim_v, s);
}

}  // namespace na
