// gsx_adamw8.hip — AdamW over many tensors with moments in 8 bits, and the row selection of such moments (include/gsx_optim.h).
#include "gsx_adamw.hpp"

namespace gsx {
namespace optim {

constexpr uint32_t kChunk = 1024;   // values of one pass of a workgroup: four of each lane, 32 lanes to a run
// Chunks of a workgroup: two in a row share its start, where there are workgroups enough to fill the card either way; more spread what is in flight too far
// (5 M splats: 786 us with two, 838 with one, 840 with eight; 1 M: 164, 183, 173).
inline uint32_t per_of(uint32_t chunks) { return chunks >= 4096 ? 2 : 1; }
constexpr uint32_t kInfinity = 0x7F800000u;
constexpr float kCodeTop = 448.0f, kScaleFloor = 0x1p-120f, kCodeMin = 0x1p-9f;
static_assert(GSX_MOMENT_RUN == 128, "the exchanges below are among 32 lanes of four values");

// Two products between shifts, their factors taken by what they do: over 2^22 inputs, random or counted, a flipped bit of the input flips every bit of the result with
// probability 0.5 +- 0.0026; neighbouring draws of either half are correlated by less than 0.001, and so are the halves.
GSX_DEV uint32_t mix(uint32_t x) {
    x ^= x >> 16; x *= 0x9E46A9E5u;
    x ^= x >> 15; x *= 0xF4B0A2DBu;
    return x ^ (x >> 16);
}

// Square roots to the last bit: x times the hardware's reciprocal root (1 ulp), corrected by what that leaves of x.  For 2^-96 and up, and zero (every float32 from 2^-96 to
// the largest compared with the root in 64 bits, rounded: none differs); where a wave has others (smaller: the remainder would be subnormal; infinities, NaN) the library's
// root, which takes twice the instructions.
GSX_DEV f32x4 roots(f32x4 x) {
    uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        low = std::min(low, __float_as_uint(x[j]) - 1u);   // (zero becomes the largest)
        high = std::max(high, __float_as_uint(x[j]));
    }
    f32x4 r;
    if (__any(low < 0x0F800000u - 1u || high >= kInfinity)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = sqrtf(x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = __builtin_amdgcn_rsqf(fmaxf(x[j], 0x1p-126f)), s = x[j] * y;
            r[j] = fmaf(fmaf(-s, s, x[j]), 0.5f * y, s);
        }
    }
    return r;
}

// Largest of the 32 lanes that hold a run (4 values each), in all of them; every lane of the wave takes part.  Floats from zero up, compared as whole numbers.
template <int C> GSX_DEV uint32_t dpp_max(uint32_t x) {
    return std::max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, C, 0xF, 0xF, true));
}
GSX_DEV uint32_t run_max(uint32_t x) {
    x = dpp_max<0xB1>(x);    // neighbours
    x = dpp_max<0x4E>(x);    // pairs of a quad
    x = dpp_max<0x141>(x);   // halves of eight
    x = dpp_max<0x140>(x);   // halves of a row of 16
    return std::max(x, (uint32_t)__builtin_amdgcn_ds_swizzle((int)x, 0x401F));   // rows of a run
}
GSX_DEV uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
GSX_DEV uint32_t top_of(f32x4 x) { return std::max(std::max(std::max(magnitude(x.x), magnitude(x.y)), magnitude(x.z)), magnitude(x.w)); }
GSX_DEV uint32_t finite_top_of(f32x4 x) {
    uint32_t f = 0;
    for (int j = 0; j < 4; ++j) f = std::max(f, magnitude(x[j]) < kInfinity ? magnitude(x[j]) : 0u);
    return f;
}
GSX_DEV float scale_of(uint32_t top) { return fmaxf(__uint_as_float(top) * (1.0f / kCodeTop), kScaleFloor); }
// The scales of a run's two moments: of their largest finite values.
GSX_DEV void scales_of(f32x4 m, f32x4 r, float* m_scale, float* r_scale) {
    uint32_t mt = run_max(top_of(m)), rt = run_max(top_of(r));
    if (__any(std::max(mt, rt) >= kInfinity)) {   // infinities or NaN among them
        mt = run_max(finite_top_of(m));
        rt = run_max(finite_top_of(r));
    }
    *m_scale = scale_of(mt);
    *r_scale = scale_of(rt);
}

// x / scale to the last bit, by the reciprocal that the four share: the hardware's (1 ulp), corrected by what it leaves of 1, is the nearest number to 1 / scale (for all
// 2^23 significands; a scale is neither below 2^-120 nor above 2^120).  Then the quotient's estimate, what that leaves of x, and the correction that this gives: the error of
// the correction is 1.5 * 2^-24 of a place at most, so only quotients nearer than that to the middle between two numbers could go wrong, X 2^24 = (2 Q + 1) S + d with
// |d| < 3 in significands; all with |d| <= 16 (93 million) come out right.  With the hardware's reciprocal as it is 47 045 of them did not.  What is left of x is
// exact for scales from 2^-93 up, and for 2^-120, where the quotient is; between the two the quotient may be off by one place.
GSX_DEV f32x4 over(f32x4 x, float scale) {
    const float near = __builtin_amdgcn_rcpf(scale), inv = fmaf(fmaf(-scale, near, 1.0f), near, near);
    f32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float q = x[j] * inv;
        y[j] = fmaf(-fmaf(q, scale, -x[j]), inv, q);   // (NaN for an infinity too; with these signs -0 stays -0)
    }
    return y;
}

// Four values of a run to their codes.  The hardware's conversions are the definition's: to nearest even, and the stochastic one adds its random word's high
// 20 bits below the last mantissa bit kept (also in the subnormal codes) and cuts; NaN and infinities become NaN.
template <bool POSITIVE, bool STOCHASTIC> GSX_DEV uint32_t encode4(f32x4 x, float scale, const uint32_t* u) {
    f32x4 y = over(x, scale);
    if (POSITIVE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = x[j] > 0.0f && y[j] < kCodeMin ? kCodeMin : y[j];
    }
    uint32_t w = 0;
    if (STOCHASTIC) {
        w = __builtin_amdgcn_cvt_sr_fp8_f32(y.x, u[0], w, 0);
        w = __builtin_amdgcn_cvt_sr_fp8_f32(y.y, u[1], w, 1);
        w = __builtin_amdgcn_cvt_sr_fp8_f32(y.z, u[2], w, 2);
        w = __builtin_amdgcn_cvt_sr_fp8_f32(y.w, u[3], w, 3);
    } else {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y.x, y.y, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y.z, y.w, w, true);
    }
    return w;
}
GSX_DEV f32x4 decode4(uint32_t w, float scale) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return f32x4{a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
}
// Four codes from `off` of `count` > 0: those behind the end are zero.  (Four loads at once, none of them behind the end, instead of one after the other.)
GSX_DEV uint32_t load_codes(const uint8_t* p, uint32_t off, uint32_t count) {
    uint32_t w = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t c = p[std::min(off + j, count - 1u)];
        w |= off + j < count ? c << (8 * j) : 0u;
    }
    return w;
}
GSX_DEV void store_codes(uint32_t w, uint8_t* p, uint32_t off, uint32_t count) {
    for (uint32_t j = 0; j < 4 && off + j < count; ++j) p[off + j] = (uint8_t)(w >> (8 * j));
}

template <uint32_t L> struct List { static constexpr uint32_t kRoom = L; Chunks<Rec, L> c; Betas b; };

template <class P, class G, bool STOCHASTIC, bool HELD, uint32_t L>
__global__ __launch_bounds__(256) void adamw8_kernel(List<L> list) {
    const Betas& a = list.b;
    const Control ctl = control_of(a);
    if (ctl.skip) return;
    walk(list.c, [&](const Rec& r, uint32_t chunk, uint32_t stop) {
        const Rates k = rates_of(r, ctl);
        const uint32_t off = threadIdx.x * 4u, run = off / GSX_MOMENT_RUN;
        const uint32_t key = STOCHASTIC ? mix(mix(a.seed + 0x9E3779B9u * (r.step ? r.step : ctl.step)) + 0xC2A6F0B5u * r.ordinal) : 0u;
        Place at(r, k.split, chunk, kChunk);
        auto pass = [&](auto whole) {   // (compiled twice: the ends of tensors and the views stay out of the way of the whole chunks)
            uint8_t* m = (uint8_t*)r.m + at.base; uint8_t* v = (uint8_t*)r.v + at.base;
            float* ms = r.m_scale + at.base / GSX_MOMENT_RUN; float* vs = r.v_scale + at.base / GSX_MOMENT_RUN;
            f32x4 pv, gv, mv, rv;
            if constexpr (whole.value) {
                const uint32_t mw = __builtin_nontemporal_load(reinterpret_cast<const u32_any*>(m + off)), vw = __builtin_nontemporal_load(reinterpret_cast<const u32_any*>(v + off));
                gv = load4((const G*)r.grad + at.base + off);
                pv = load4((const P*)r.param + at.base + off);
                mv = decode4(mw, ms[run]);
                rv = decode4(vw, vs[run]);
            } else {   // the end of a tensor, or a view: value by value, all loads at once, none behind the end
                const uint32_t mw = load_codes(m, off, at.count), vw = load_codes(v, off, at.count), here = std::min(off, at.count - 1u) / GSX_MOMENT_RUN;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const Place::Spot s = at.spot(std::min(off + j, at.count - 1u));
                    const float g1 = (float)((const G*)r.grad)[at(s, r.ld_grad)];
                    gv[j] = off + j < at.count ? g1 : 0.0f;
                    pv[j] = (float)((const P*)r.param)[at(s, r.ld_param)];
                }
                mv = decode4(mw, ms[here]);
                rv = decode4(vw, vs[here]);
            }
            // (from here on every lane, also those behind the end: the lanes of a run exchange their largest values)
            uint32_t held = 0;
            const Steps o = steps_of(k, at.mine, at.cols, HELD ? &held : nullptr);
            f32x4 m1, r1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                gv[j] *= ctl.factor;
                m1[j] = first_moment(a, mv[j], gv[j]);
                r1[j] = second_moment(a, rv[j] * rv[j], gv[j]);
            }
            r1 = roots(r1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p1 = stepped(a, k, o.lrwd[j], o.step[j], pv[j], m1[j], r1[j]);
                pv[j] = HELD && (held >> j & 1u) ? pv[j] : p1;
            }
            if constexpr (!HELD) {
                mv = m1;
                rv = r1;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mv[j] = held >> j & 1u ? mv[j] : m1[j];
                    rv[j] = held >> j & 1u ? rv[j] : r1[j];
                }
            }
            float m_scale, v_scale;
            scales_of(mv, rv, &m_scale, &v_scale);
            uint32_t um[4], uv[4];
            if (STOCHASTIC) {
                const uint32_t i = (uint32_t)at.base + key + 0x61C8864Fu * (uint32_t)(at.base >> 32) + off;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t w = mix(i + j);
                    um[j] = w & 0xFFFF0000u;
                    uv[j] = __builtin_amdgcn_perm(w, 0u, 0x05040C0Cu);   // w << 16 (as a shift it would become a third product)
                }
            }
            const uint32_t mw = encode4<false, STOCHASTIC>(mv, m_scale, um), vw = encode4<true, STOCHASTIC>(rv, v_scale, uv);
            if constexpr (whole.value) {
                __builtin_nontemporal_store(mw, reinterpret_cast<u32_any*>(m + off));
                __builtin_nontemporal_store(vw, reinterpret_cast<u32_any*>(v + off));
                store4(pv, (P*)r.param + at.base + off);
            } else {
                store_codes(mw, m, off, at.count);
                store_codes(vw, v, off, at.count);
                for (uint32_t j = 0; j < 4 && off + j < at.count; ++j)
                    if (!HELD || !(held >> j & 1u)) ((P*)r.param)[at(at.spot(off + j), r.ld_param)] = (P)pv[j];
            }
            if (off < at.count && (off & (GSX_MOMENT_RUN - 1)) == 0) { ms[run] = m_scale; vs[run] = v_scale; }
        };
        for (; chunk < stop; ++chunk, at.next(kChunk)) {
            if (at.whole) pass(std::true_type{});
            else pass(std::false_type{});
        }
    });
}

// ---- rows of 8-bit moments --------------------------------------------------------------------------------------------------------------------------------
struct SelectRec { const uint8_t *m, *v; const float *ms, *vs; uint8_t *mo, *vo; float *mso, *vso; uint64_t cols; };
template <uint32_t L> struct SelectList {
    static constexpr uint32_t kRoom = L;
    Chunks<SelectRec, L> c;
    const int64_t* index;
    uint64_t rows_in, rows_out;
};

constexpr uint32_t kSelect = 2048;   // values of a chunk
constexpr uint32_t kPasses = kSelect / 1024u;

// n / d for n < 2^22, d < 2^22 (the quotient's estimate is off by one at most).
GSX_DEV uint32_t small_div(uint32_t n, uint32_t d, float rcp) {
    uint32_t q = (uint32_t)((float)n * rcp);
    q -= q * d > n ? 1u : 0u;
    return n - q * d >= d ? q + 1u : q;
}

// Codes four new values of each moment and stores them; off: the first of them in the chunk.  Every lane of the wave takes part, those behind the end with zeros.
GSX_DEV void store_selected(const SelectRec& r, uint64_t base, uint32_t off, uint32_t count, f32x4 m, f32x4 v) {
    float m_scale, v_scale;
    scales_of(m, v, &m_scale, &v_scale);
    if (off >= count) return;
    const uint32_t mw = encode4<false, false>(m, m_scale, nullptr), vw = encode4<true, false>(v, v_scale, nullptr);
    if (off + 4 <= count) {
        *reinterpret_cast<u32_any*>(r.mo + base + off) = mw;
        *reinterpret_cast<u32_any*>(r.vo + base + off) = vw;
    } else {
        store_codes(mw, r.mo + base, off, count);
        store_codes(vw, r.vo + base, off, count);
    }
    if ((off & (GSX_MOMENT_RUN - 1)) == 0) { r.mso[(base + off) / GSX_MOMENT_RUN] = m_scale; r.vso[(base + off) / GSX_MOMENT_RUN] = v_scale; }
}

// Rows whose length is a multiple of four: a lane's four values come from one row and one run, straight into its registers.
GSX_DEV void select_fours(const SelectRec& r, const int64_t* __restrict__ index, uint64_t rows_in, uint64_t base, uint64_t row0, uint32_t col0, uint32_t count) {
    const uint32_t cols = (uint32_t)r.cols;
    const bool small = cols < (1u << 21);
    const float rcp = 1.0f / (float)cols;
    uint32_t mw[kPasses], vw[kPasses], c[kPasses];
    float ms[kPasses], vs[kPasses];
    int64_t src[kPasses];
#pragma unroll
    for (uint32_t u = 0; u < kPasses; ++u) {
        const uint32_t q = col0 + std::min(u * 1024u + threadIdx.x * 4u, count - 4u), dr = small ? small_div(q, cols, rcp) : q / cols;
        c[u] = q - dr * cols;
        src[u] = index[row0 + dr];
    }
#pragma unroll
    for (uint32_t u = 0; u < kPasses; ++u) {
        mw[u] = vw[u] = 0;
        ms[u] = vs[u] = 0.0f;
        if (src[u] < 0 || (uint64_t)src[u] >= rows_in || u * 1024u + threadIdx.x * 4u >= count) continue;
        const uint64_t at = (uint64_t)src[u] * cols + c[u];
        mw[u] = *reinterpret_cast<const u32_any*>(r.m + at);
        vw[u] = *reinterpret_cast<const u32_any*>(r.v + at);
        ms[u] = r.ms[at / GSX_MOMENT_RUN];
        vs[u] = r.vs[at / GSX_MOMENT_RUN];
    }
#pragma unroll
    for (uint32_t u = 0; u < kPasses; ++u) store_selected(r, base, u * 1024u + threadIdx.x * 4u, count, decode4(mw[u], ms[u]), decode4(vw[u], vs[u]));
}

// Other rows: a chunk is gathered into LDS in pieces of up to four values of one row (an index, two words of codes and two scales or four a piece, wherever old and new
// runs begin), and coded from there.
constexpr uint32_t kBatch = 3;   // pieces of a lane whose loads are in flight together
GSX_DEV void select_pieces(const SelectRec& r, const int64_t* __restrict__ index, uint64_t rows_in, uint64_t base, uint64_t row0, uint32_t col0, uint32_t count,
                           float (*lds)[kSelect]) {
    const uint32_t cols = (uint32_t)r.cols, pieces = (cols + 3) / 4, last = col0 + count - 1u;
    const uint64_t n_in = rows_in * r.cols;
    const uint32_t items = last / cols * pieces + last % cols / 4u + 1u;   // pieces from the start of the first row to the last value
    const bool small = items < (1u << 22) && pieces < (1u << 22);
    const float rcp = 1.0f / (float)pieces;
    __syncthreads();
    for (uint32_t i = col0 / 4u + threadIdx.x; i < items; i += 256u * kBatch) {
        uint32_t c[kBatch], len[kBatch], left[kBatch], mw[kBatch], vw[kBatch];
        int32_t to[kBatch];   // where in the chunk a piece goes; the first may start before it and the last end behind it
        int64_t src[kBatch];
        float m0[kBatch], v0[kBatch], m1[kBatch], v1[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t item = std::min(i + 256u * b, items - 1u), dr = small ? small_div(item, pieces, rcp) : item / pieces;
            c[b] = (item - dr * pieces) * 4u;
            len[b] = std::min(cols - c[b], 4u);
            to[b] = (int32_t)(dr * cols + c[b] - col0);
            src[b] = index[row0 + dr];
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            mw[b] = vw[b] = 0;
            m0[b] = v0[b] = m1[b] = v1[b] = 0.0f;
            left[b] = 4;
            if (src[b] < 0 || (uint64_t)src[b] >= rows_in) continue;
            const uint64_t at = (uint64_t)src[b] * cols + c[b], run = at / GSX_MOMENT_RUN;
            if (at + 4 <= n_in) {
                mw[b] = *reinterpret_cast<const u32_any*>(r.m + at);
                vw[b] = *reinterpret_cast<const u32_any*>(r.v + at);
            } else {
                mw[b] = load_codes(r.m + at, 0, len[b]);
                vw[b] = load_codes(r.v + at, 0, len[b]);
            }
            m0[b] = r.ms[run];
            v0[b] = r.vs[run];
            left[b] = GSX_MOMENT_RUN - (uint32_t)(at % GSX_MOMENT_RUN);   // values up to the next run
            if (left[b] < len[b]) { m1[b] = r.ms[run + 1]; v1[b] = r.vs[run + 1]; }
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            if (i + 256u * b >= items) continue;
            const f32x4 mv = decode4(mw[b], 1.0f), rv = decode4(vw[b], 1.0f);
#pragma unroll
            for (int32_t j = 0; j < 4; ++j) {
                if (j < (int32_t)len[b] && to[b] + j >= 0 && to[b] + j < (int32_t)count) {
                    lds[0][to[b] + j] = mv[j] * ((uint32_t)j < left[b] ? m0[b] : m1[b]);
                    lds[1][to[b] + j] = rv[j] * ((uint32_t)j < left[b] ? v0[b] : v1[b]);
                }
            }
        }
    }
    __syncthreads();
    for (uint32_t u = 0; u < kPasses; ++u) {
        const uint32_t off = u * 1024u + threadIdx.x * 4u;
        f32x4 m = *reinterpret_cast<const f32x4*>(&lds[0][off]), v = *reinterpret_cast<const f32x4*>(&lds[1][off]);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            m[j] = off + j < count ? m[j] : 0.0f;
            v[j] = off + j < count ? v[j] : 0.0f;
        }
        store_selected(r, base, off, count, m, v);
    }
}

// What bounds it, 1 M splats by a random order (122 MB of codes), 171 us: rows of 48 bytes (85 of them) the 128-byte lines that they lie in, 4.6 M misses at 6.9 TB/s; rows of
// one to four bytes (92) the requests, one for every row and moment and one for its scale, 15 M (fewer misses there took the same time).  In an order near the old one, as a growth
// step's is: 80 us.  100 k splats: 20 us, 16 in the near order: a round and a half of workgroups that wait for record, index and codes in turn.
template <uint32_t L> __global__ __launch_bounds__(256, 8) void select_rows_kernel(SelectList<L> a) {
    __shared__ __align__(16) float lds[2][kSelect];
    walk(a.c, [&](const SelectRec& r, uint32_t chunk, uint32_t stop) {
        const uint64_t n = a.rows_out * r.cols;
        for (; chunk < stop; ++chunk) {
            const uint64_t base = (uint64_t)chunk * kSelect, row0 = base >> 32 ? base / r.cols : (uint32_t)base / (uint32_t)r.cols;
            const uint32_t count = (uint32_t)std::min<uint64_t>(n - base, kSelect), col0 = (uint32_t)(base - row0 * r.cols);
            if (r.cols % 4 == 0) select_fours(r, a.index, a.rows_in, base, row0, col0, count);
            else select_pieces(r, a.index, a.rows_in, base, row0, col0, count, lds);
        }
    });
}

}  // namespace optim
}  // namespace gsx

using namespace gsx;
using namespace gsx::optim;

extern "C" int gsx_adamw8_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, int stochastic, uint32_t seed,
                                     const double* control, void* stream) {
    const int bad = check_adamw(count, tensors, beta1, beta2, eps, true, control);
    if (bad != GSX_OK || count == 0) return bad;
    const Betas betas = betas_of(beta1, beta2, eps, seed, control);
    Corrections last = {};
    const uint32_t mask = types_of(count, tensors);
    const bool held = any_held(count, tensors);
    for (uint32_t types = 0; types < 9; ++types) {
        if (!(mask >> types & 1u)) continue;
        const uint32_t pd = types / 3, gd = types % 3;
        const int rc = launch_lists<List>(
            count, kChunk, per_of,
            [&](uint32_t i, Rec* r, uint64_t* n) {
                if (tensors[i].param_dtype != pd || tensors[i].grad_dtype != gd) return false;
                *r = rec_of(tensors[i], i, betas, &last);
                *n = r->n;
                return true;
            },
            [&](auto& a, uint32_t blocks) {
                a.b = betas;
                constexpr uint32_t L = std::remove_reference_t<decltype(a)>::kRoom;
                int rc = GSX_OK;
                by_dtype(pd, [&](auto p) {
                    by_dtype(gd, [&](auto g) {
                        typedef decltype(p) P;
                        typedef decltype(g) G;
                        const auto kernel = stochastic ? (held ? adamw8_kernel<P, G, true, true, L> : adamw8_kernel<P, G, true, false, L>)
                                                       : (held ? adamw8_kernel<P, G, false, true, L> : adamw8_kernel<P, G, false, false, L>);
                        rc = launch_list(kernel, a, blocks, stream, "adamw8_step_multi");
                    });
                });
                return rc;
            });
        if (rc != GSX_OK) return rc;
    }
    return GSX_OK;
}

extern "C" int gsx_adamw8_select_rows(uint32_t count, const gsx_moments8* tensors, uint64_t rows_in, uint64_t rows_out, const int64_t* index, void* stream) {
    if (count == 0 || rows_out == 0) return GSX_OK;
    if (tensors == nullptr || index == nullptr) return invalid("adamw8_select_rows: null list or index");
    for (uint32_t i = 0; i < count; ++i) {
        const gsx_moments8& x = tensors[i];
        uint64_t n;
        if (!count_of(rows_in, x.cols, &n) || !count_of(rows_out, x.cols, &n) || x.cols > (1ull << 31)) return invalid("adamw8_select_rows: tensor too large");
        if (x.cols == 0) continue;
        if (!x.avg_out || !x.rms_out || !x.avg_scale_out || !x.rms_scale_out) return invalid("adamw8_select_rows: null tensor");
        if (rows_in != 0 && (!x.avg_in || !x.rms_in || !x.avg_scale_in || !x.rms_scale_in)) return invalid("adamw8_select_rows: null tensor");
    }
    return launch_lists<SelectList>(
        count, kSelect, [](uint32_t) { return 1u; },
        [&](uint32_t i, SelectRec* r, uint64_t* n) {
            const gsx_moments8& x = tensors[i];
            *r = SelectRec{(const uint8_t*)x.avg_in, (const uint8_t*)x.rms_in, x.avg_scale_in, x.rms_scale_in, (uint8_t*)x.avg_out, (uint8_t*)x.rms_out,
                           x.avg_scale_out, x.rms_scale_out, x.cols};
            *n = rows_out * x.cols;
            return true;
        },
        [&](auto& a, uint32_t blocks) {
            a.index = index; a.rows_in = rows_in; a.rows_out = rows_out;
            constexpr uint32_t L = std::remove_reference_t<decltype(a)>::kRoom;
            return launch_list(select_rows_kernel<L>, a, blocks, stream, "adamw8_select_rows");
        });
}
