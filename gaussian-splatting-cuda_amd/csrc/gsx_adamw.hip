// gsx_adamw.hip — the optimizer operators over many tensors at once (include/gsx_optim.h): AdamW with moments in 32 or in 8 bits, the norm of all
// gradients, the row selection of 8-bit moments.
//
// All four are streams over memory (0.25 - 1 operation a byte): what bounds them is HBM, for small models the launch.  A launch takes up to kList tensors as
// kernel arguments (no table in device memory: nothing to allocate, copy or keep, and a captured graph holds all it needs).  The tensors are cut into
// chunks, numbered through the list; a workgroup finds its chunk's tensor with one load and one ballot of the wave: lane l holds the first chunk of tensor l.
#include <math.h>

#include <algorithm>

#include "gsx_device.hpp"
#include "../../include/gsx_optim.h"

namespace gsx {

void set_error(const char* msg);
int check_launch(const char* what);

namespace {

constexpr uint32_t kList = 32;    // tensors of one launch: the argument block stays below 4 KB
constexpr uint32_t kChunk = 2048; // values of one pass of a workgroup
constexpr uint32_t kGrid = 16384; // workgroups of a launch at most
constexpr float kCodeTop = 448.0f, kScaleFloor = 0x1p-120f, kCodeMin = 0x1p-9f;

// Vectors of four values at any address that the type itself may have: gfx950 loads and stores them with one instruction wherever they lie.
template <class T> struct Vec4;
template <> struct Vec4<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec4<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Vec4<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2))); };
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

template <class T> GSX_DEV f32x4 load4(const T* p) {
    return __builtin_convertvector(__builtin_nontemporal_load(reinterpret_cast<const typename Vec4<T>::type*>(p)), f32x4);
}
template <class T> GSX_DEV void store4(f32x4 x, T* p) {
    typedef typename Vec4<T>::type V;
    __builtin_nontemporal_store((V)__builtin_convertvector(x, V), reinterpret_cast<V*>(p));
}

// The tensor that chunk `c` of a launch belongs to (begin[l]: first chunk of tensor l, all ones behind the last tensor).
GSX_DEV uint32_t tensor_of(const uint32_t* begin, uint32_t c) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t in = __ballot(c >= begin[lane < kList ? lane : kList - 1] && lane < kList);
    return (uint32_t)__builtin_popcountll(in) - 1u;
}

struct Rec {
    void* param; const void* grad; void* m; void* v; float* m_scale; float* v_scale;
    uint64_t n, cols, ld_param, ld_grad;
    uint32_t step, split, flags, ordinal;
    float lr, lr_b, wd, wd_b;
};
enum : uint32_t { kHold = 1, kHoldB = 2, kScalar = 4 };

struct List {
    Rec rec[kList];
    uint32_t begin[kList];
    const double* control;
    double log_b1, log_b2;
    uint32_t chunks, seed;
    float b1, b1c, b2, b2c, eps;
};
static_assert(sizeof(List) <= 4096, "kernel arguments");

// What one tensor's update needs of the step: 1 - beta^t = -expm1(t log beta), whose relative error is that of the product (2^-24), where 1 - pow() would
// lose beta's own rounding (0.999 in 32 bits: 3e-5 of 1 - beta).
struct Rates { float step, step_b, lrwd, lrwd_b, bc2; };
GSX_DEV Rates rates_of(const List& a, const Rec& r, uint32_t t) {
    const float bc1 = -expm1f((float)(a.log_b1 * (double)t)), bc2 = -expm1f((float)(a.log_b2 * (double)t));
    return {r.lr / bc1, r.lr_b / bc1, r.lr * r.wd, r.lr_b * r.wd_b, 1.0f / sqrtf(bc2)};
}

template <class P, class G>
__global__ __launch_bounds__(256) void adamw_kernel(List a) {
    float gs = 1.0f;
    uint32_t control_step = 0;
    if (a.control != nullptr) {
        if (a.control[2] != 0.0) return;
        gs = (float)a.control[1];
        control_step = std::max((uint32_t)a.control[3], 1u);   // (a block that no norm has advanced: the first step)
    }
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const uint32_t t = tensor_of(a.begin, chunk);
        const Rec& r = a.rec[t];
        const Rates k = rates_of(a, r, r.step ? r.step : control_step);
        const uint64_t base = (uint64_t)(chunk - a.begin[t]) * kChunk;
        const uint32_t count = (uint32_t)std::min<uint64_t>(r.n - base, kChunk);
        P* __restrict__ p = (P*)r.param; const G* __restrict__ g = (const G*)r.grad;
        float* __restrict__ m = (float*)r.m + base; float* __restrict__ v = (float*)r.v + base;
        const uint64_t row0 = r.flags & kScalar ? base / r.cols : 0;
        const uint32_t col0 = r.split || (r.flags & kScalar) ? (uint32_t)(base % r.cols) : 0, cols = (uint32_t)r.cols;
        for (uint32_t off = threadIdx.x; off < count; off += 256u) {
            const uint32_t q = col0 + off, dr = r.split || (r.flags & kScalar) ? q / cols : 0, c = q - dr * cols;
            const bool b = r.split && c >= r.split;
            if (r.flags & (b ? kHoldB : kHold)) continue;
            const uint64_t at_p = r.flags & kScalar ? (row0 + dr) * r.ld_param + c : base + off, at_g = r.flags & kScalar ? (row0 + dr) * r.ld_grad + c : base + off;
            const float gv = (float)g[at_g] * gs, pv = (float)p[at_p];
            const float mv = a.b1 * m[off] + a.b1c * gv, vv = a.b2 * v[off] + a.b2c * gv * gv;
            p[at_p] = (P)(pv - (b ? k.lrwd_b : k.lrwd) * pv - (b ? k.step_b : k.step) * mv / (sqrtf(vv) * k.bc2 + a.eps));
            m[off] = mv;
            v[off] = vv;
        }
    }
}

// The moments as the formulas write them, each product and sum rounded by itself: what is stored in 8 bits is then a function of the inputs that can be
// computed anywhere to the last bit (a fused product moves a value by 2^-25, and where it lies next to a border of the format, its code by a whole step).
GSX_DEV float first_moment(const List& a, float m, float g) {
#pragma clang fp contract(off)
    return a.b1 * m + a.b1c * g;
}
GSX_DEV float second_moment(const List& a, float v, float g) {
#pragma clang fp contract(off)
    return a.b2 * v + a.b2c * g * g;
}

// ---- 8-bit moments ---------------------------------------------------------------------------------------------------------------------------------
GSX_DEV uint32_t mix(uint32_t x) {
    x ^= x >> 16; x *= 0x9E46A9E5u;
    x ^= x >> 15; x *= 0xF4B0A2DBu;
    return x ^ (x >> 16);
}

template <int C> GSX_DEV float dpp_max(float x) {
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), C, 0xF, 0xF, true)));
}
// Largest of the 32 lanes that hold a run (4 values each), in all of them; every lane of the wave takes part.
GSX_DEV float run_max(float x) {
    x = dpp_max<0xB1>(x);    // neighbours
    x = dpp_max<0x4E>(x);    // pairs of a quad
    x = dpp_max<0x141>(x);   // halves of eight
    x = dpp_max<0x140>(x);   // halves of a row of 16
    return fmaxf(x, __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(x), 0x401F)));   // rows of a run
}

GSX_DEV float top_of(f32x4 x) {
    const float top = run_max(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));   // (fmaxf passes over NaN)
    if (__any(isinf(top))) {   // a run with infinities: the largest of the finite values
        float f = 0.0f;
        for (int j = 0; j < 4; ++j) f = fmaxf(f, isinf(x[j]) ? 0.0f : fabsf(x[j]));
        return run_max(f);
    }
    return top;
}
GSX_DEV float scale_of(float top) { return fmaxf(top * (1.0f / kCodeTop), kScaleFloor); }

// Four values of a run to their codes.  The hardware's conversions are the definition's: to nearest even, and the stochastic one adds its random word's high
// 20 bits below the last mantissa bit kept (also in the subnormal codes) and cuts; NaN and infinities become NaN.
template <bool POSITIVE> GSX_DEV uint32_t encode4(f32x4 x, float scale, bool stochastic, const uint32_t* u) {
    const f32x4 s = {scale, scale, scale, scale};
    f32x4 y = x / s;
    for (int j = 0; j < 4; ++j) {
        if (POSITIVE) y[j] = y[j] > 0.0f && y[j] < kCodeMin ? kCodeMin : x[j] > 0.0f && y[j] == 0.0f ? kCodeMin : y[j];
    }
    uint32_t w = 0;
    if (stochastic) {
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
    return f32x4{__builtin_amdgcn_cvt_f32_fp8(w, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale,
                 __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale};
}
// Four codes from `off` of `count`: bytes behind the end are zero, and are not touched.
GSX_DEV uint32_t load_codes(const uint8_t* p, uint32_t off, uint32_t count) {
    if (off + 4 <= count) return *reinterpret_cast<const u32_any*>(p + off);
    uint32_t w = 0;
    for (uint32_t j = 0; j < 4 && off + j < count; ++j) w |= (uint32_t)p[off + j] << (8 * j);
    return w;
}
GSX_DEV void store_codes(uint32_t w, uint8_t* p, uint32_t off, uint32_t count) {
    if (off + 4 <= count) { *reinterpret_cast<u32_any*>(p + off) = w; return; }
    for (uint32_t j = 0; j < 4 && off + j < count; ++j) p[off + j] = (uint8_t)(w >> (8 * j));
}

template <class P, class G>
__global__ __launch_bounds__(256) void adamw8_kernel(List a, int stochastic) {
    float gs = 1.0f;
    uint32_t control_step = 0;
    if (a.control != nullptr) {
        if (a.control[2] != 0.0) return;
        gs = (float)a.control[1];
        control_step = std::max((uint32_t)a.control[3], 1u);   // (a block that no norm has advanced: the first step)
    }
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const uint32_t t = tensor_of(a.begin, chunk);
        const Rec& r = a.rec[t];
        const uint32_t step = r.step ? r.step : control_step;
        const Rates k = rates_of(a, r, step);
        const uint64_t base = (uint64_t)(chunk - a.begin[t]) * kChunk;
        const uint32_t count = (uint32_t)std::min<uint64_t>(r.n - base, kChunk);
        P* __restrict__ p = (P*)r.param; const G* __restrict__ g = (const G*)r.grad;
        uint8_t* __restrict__ m = (uint8_t*)r.m + base; uint8_t* __restrict__ v = (uint8_t*)r.v + base;
        float* __restrict__ ms = r.m_scale + base / GSX_MOMENT_RUN; float* __restrict__ vs = r.v_scale + base / GSX_MOMENT_RUN;
        const bool by_column = r.split || (r.flags & kScalar);
        const uint64_t row0 = r.flags & kScalar ? base / r.cols : 0;
        const uint32_t col0 = by_column ? (uint32_t)(base % r.cols) : 0, cols = (uint32_t)r.cols;
        const uint32_t key = mix(mix(a.seed + 0x9E3779B9u * step) + 0xC2A6F0B5u * r.ordinal) + 0x61C8864Fu * (uint32_t)(base >> 32);
        for (uint32_t pass = 0; pass < kChunk; pass += 1024u) {   // (the same number of passes for every lane: the runs' lanes exchange their largest values)
            const uint32_t off = pass + threadIdx.x * 4u, run = off / GSX_MOMENT_RUN;
            const bool any = off < count;
            f32x4 mv = {0, 0, 0, 0}, rv = {0, 0, 0, 0};
            if (any) {
                mv = decode4(load_codes(m, off, count), ms[run]);
                rv = decode4(load_codes(v, off, count), vs[run]);
                for (uint32_t j = 0; j < 4 && off + j < count; ++j) {
                    const uint32_t q = col0 + off + j, dr = by_column ? q / cols : 0, c = q - dr * cols;
                    const bool b = r.split && c >= r.split;
                    if (r.flags & (b ? kHoldB : kHold)) continue;
                    const uint64_t at_p = r.flags & kScalar ? (row0 + dr) * r.ld_param + c : base + off + j;
                    const uint64_t at_g = r.flags & kScalar ? (row0 + dr) * r.ld_grad + c : base + off + j;
                    const float gv = (float)g[at_g] * gs, pv = (float)p[at_p];
                    mv[j] = first_moment(a, mv[j], gv);
                    rv[j] = sqrtf(second_moment(a, rv[j] * rv[j], gv));
                    p[at_p] = (P)(pv - (b ? k.lrwd_b : k.lrwd) * pv - (b ? k.step_b : k.step) * mv[j] / (rv[j] * k.bc2 + a.eps));
                }
            }
            const float m_scale = scale_of(top_of(mv)), v_scale = scale_of(top_of(rv));
            if (!any) continue;
            uint32_t um[4], uv[4];
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t w = mix((uint32_t)(base + off + j) + key);
                um[j] = w & 0xFFFF0000u;
                uv[j] = w << 16;
            }
            store_codes(encode4<false>(mv, m_scale, stochastic, um), m, off, count);
            store_codes(encode4<true>(rv, v_scale, stochastic, uv), v, off, count);
            if ((off & (GSX_MOMENT_RUN - 1)) == 0) { ms[run] = m_scale; vs[run] = v_scale; }
        }
    }
}

struct SelectRec { const uint8_t *m, *v; const float *ms, *vs; uint8_t *mo, *vo; float *mso, *vso; uint64_t cols; };
struct SelectList {
    SelectRec rec[kList];
    uint32_t begin[kList];
    const int64_t* index;
    uint64_t rows_in, rows_out;
    uint32_t chunks;
};
static_assert(sizeof(SelectList) <= 4096, "kernel arguments");

__global__ __launch_bounds__(256) void select_rows_kernel(SelectList a) {
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const uint32_t t = tensor_of(a.begin, chunk);
        const SelectRec& r = a.rec[t];
        const uint64_t base = (uint64_t)(chunk - a.begin[t]) * kChunk, n = a.rows_out * r.cols;
        const uint32_t count = (uint32_t)std::min<uint64_t>(n - base, kChunk);
        const uint64_t row0 = base / r.cols;
        const uint32_t col0 = (uint32_t)(base - row0 * r.cols), cols = (uint32_t)r.cols;
        for (uint32_t pass = 0; pass < kChunk; pass += 1024u) {
            const uint32_t off = pass + threadIdx.x * 4u;
            f32x4 mv = {0, 0, 0, 0}, rv = {0, 0, 0, 0};
            for (uint32_t j = 0; j < 4 && off + j < count; ++j) {
                const uint32_t q = col0 + off + j, dr = q / cols;
                const int64_t src = a.index[row0 + dr];
                if (src < 0 || (uint64_t)src >= a.rows_in) continue;
                const uint64_t at = (uint64_t)src * cols + (q - dr * cols);
                mv[j] = __builtin_amdgcn_cvt_f32_fp8(r.m[at], 0) * r.ms[at / GSX_MOMENT_RUN];
                rv[j] = __builtin_amdgcn_cvt_f32_fp8(r.v[at], 0) * r.vs[at / GSX_MOMENT_RUN];
            }
            const float m_scale = scale_of(top_of(mv)), v_scale = scale_of(top_of(rv));
            if (off >= count) continue;
            store_codes(encode4<false>(mv, m_scale, false, nullptr), r.mo + base, off, count);
            store_codes(encode4<true>(rv, v_scale, false, nullptr), r.vo + base, off, count);
            if ((off & (GSX_MOMENT_RUN - 1)) == 0) { r.mso[(base + off) / GSX_MOMENT_RUN] = m_scale; r.vso[(base + off) / GSX_MOMENT_RUN] = v_scale; }
        }
    }
}

// ---- the norm ----------------------------------------------------------------------------------------------------------------------------------------
struct NormRec { const void* grad; uint64_t n, cols, ld; };
struct NormList {
    NormRec rec[kList];
    uint32_t begin[kList];
    double* partial;   // of the whole call: one for each workgroup
    double* control;
    double max_norm;
    uint32_t chunks, first, blocks;   // this launch's chunks and first partial; workgroups of the whole call
};
static_assert(sizeof(NormList) <= 4096, "kernel arguments");

GSX_DEV double block_sum(double x, double* lds) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Sums of squares in 64 bits: no square of a 32-bit number overflows, so the sum is finite exactly if all gradients are.  Every workgroup leaves its sum, the
// last one to finish adds them up in their order (the same bits every time) and writes the control block.
template <class G>
__global__ __launch_bounds__(256) void grad_norm_kernel(NormList a) {
    __shared__ double lds[4];
    __shared__ uint32_t last;
    double sum = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const uint32_t t = tensor_of(a.begin, chunk);
        const NormRec& r = a.rec[t];
        const uint64_t base = (uint64_t)(chunk - a.begin[t]) * kChunk;
        const uint32_t count = (uint32_t)std::min<uint64_t>(r.n - base, kChunk);
        const G* __restrict__ g = (const G*)r.grad;
        const bool strided = r.ld != r.cols;
        const uint64_t row0 = strided ? base / r.cols : 0;
        const uint32_t col0 = strided ? (uint32_t)(base % r.cols) : 0, cols = (uint32_t)r.cols;
        for (uint32_t off = threadIdx.x; off < count; off += 256u) {
            const uint32_t q = col0 + off, dr = strided ? q / cols : 0;
            const double x = (double)(float)g[strided ? (row0 + dr) * r.ld + (q - dr * cols) : base + off];
            sum += x * x;
        }
    }
    sum = block_sum(sum, lds);
    uint32_t* ticket = reinterpret_cast<uint32_t*>(a.control + 4);
    if (threadIdx.x == 0) {
        __hip_atomic_store(a.partial + a.first + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.blocks - 1u;
    }
    __syncthreads();
    if (!last) return;
    double total = 0.0;
    for (uint32_t i = threadIdx.x; i < a.blocks; i += 256u) total += __hip_atomic_load(a.partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    total = block_sum(total, lds);
    if (threadIdx.x == 0) {
        const bool fine = isfinite(total);
        const double norm = sqrt(total);
        a.control[0] = norm;
        a.control[1] = fine ? fmin(1.0, a.max_norm / (norm + 1e-6)) : 0.0;
        a.control[2] = fine ? 0.0 : 1.0;
        a.control[3] += fine ? 1.0 : 0.0;
        __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// ---- launching -----------------------------------------------------------------------------------------------------------------------------------------
int invalid(const char* msg) { set_error(msg); return GSX_ERR_INVALID_ARGUMENT; }

uint64_t chunks_of(uint64_t n) { return (n + kChunk - 1) / kChunk; }

// rows x cols as the kernels take it: the number of values, or false where it does not fit.
bool count_of(uint64_t rows, uint64_t cols, uint64_t* n) {
    if (rows != 0 && cols > (1ull << 44) / rows) return false;
    *n = rows * cols;
    return true;
}

template <class F> void by_dtype(uint32_t d, F f) {
    if (d == GSX_DTYPE_F32) f(float{});
    else if (d == GSX_DTYPE_BF16) f(__bf16{});
    else f(_Float16{});
}

void launch_adamw(const List& a, uint32_t pd, uint32_t gd, bool eight, int stochastic, hipStream_t st) {
    const dim3 grid(std::min(a.chunks, kGrid)), block(256);
    by_dtype(pd, [&](auto p) {
        by_dtype(gd, [&](auto g) {
            typedef decltype(p) P;
            typedef decltype(g) G;
            if (eight) hipLaunchKernelGGL((adamw8_kernel<P, G>), grid, block, 0, st, a, stochastic);
            else hipLaunchKernelGGL((adamw_kernel<P, G>), grid, block, 0, st, a);
        });
    });
}

int adamw_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, bool eight, int stochastic, uint32_t seed,
                const double* control, void* stream, const char* what) {
    if (count == 0) return GSX_OK;
    if (tensors == nullptr) return invalid("adamw_step_multi: null list");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return invalid("adamw_step_multi: betas lie in [0, 1)");
    if (!(eps >= 0.0)) return invalid("adamw_step_multi: eps is not negative");
    for (uint32_t i = 0; i < count; ++i) {
        const gsx_adamw_tensor& x = tensors[i];
        uint64_t n;
        if (!count_of(x.rows, x.cols, &n)) return invalid("adamw_step_multi: tensor too large");
        if (x.param_dtype > GSX_DTYPE_F16 || x.grad_dtype > GSX_DTYPE_F16) return invalid("adamw_step_multi: unknown dtype");
        if (n == 0) continue;
        if (!x.param || !x.grad || !x.exp_avg || !x.exp_avg_sq || (eight && (!x.avg_scale || !x.rms_scale))) return invalid("adamw_step_multi: null tensor");
        if (x.rows > 1 && (x.ld_param < x.cols || x.ld_grad < x.cols)) return invalid("adamw_step_multi: rows overlap (ld smaller than cols)");
        if (x.split > x.cols) return invalid("adamw_step_multi: split beyond the columns");
        if ((x.rows > 1 && (x.ld_param != x.cols || x.ld_grad != x.cols)) || x.split)
            if (x.cols > (1ull << 31)) return invalid("adamw_step_multi: rows of more than 2^31 values");
        if (x.step == 0 && control == nullptr) return invalid("adamw_step_multi: a step counts from 1 (0 takes the control block's)");
        if (x.step > 0xFFFFFFFFull) return invalid("adamw_step_multi: step beyond 32 bits");
    }
    for (uint32_t pd = 0; pd <= GSX_DTYPE_F16; ++pd) {
        for (uint32_t gd = 0; gd <= GSX_DTYPE_F16; ++gd) {
            List a;
            uint32_t k = 0;
            uint64_t chunks = 0;
            a.control = control;
            a.log_b1 = log(beta1); a.log_b2 = log(beta2);
            a.b1 = (float)beta1; a.b1c = (float)(1.0 - beta1); a.b2 = (float)beta2; a.b2c = (float)(1.0 - beta2); a.eps = (float)eps;
            a.seed = seed;
            for (uint32_t i = 0; i <= count; ++i) {
                const gsx_adamw_tensor* x = i < count ? tensors + i : nullptr;
                if (x && (x->param_dtype != pd || x->grad_dtype != gd || x->rows == 0 || x->cols == 0)) continue;
                const uint64_t more = x ? chunks_of(x->rows * x->cols) : 0;
                if (k != 0 && (x == nullptr || k == kList || chunks + more > 0x7FFFFFFFull)) {
                    for (uint32_t j = k; j < kList; ++j) a.begin[j] = 0xFFFFFFFFu;
                    a.chunks = (uint32_t)chunks;
                    launch_adamw(a, pd, gd, eight, stochastic, (hipStream_t)stream);
                    const int rc = check_launch(what);
                    if (rc != GSX_OK) return rc;
                    k = 0; chunks = 0;
                }
                if (x == nullptr) break;
                if (more > 0x7FFFFFFFull) return invalid("adamw_step_multi: tensor too large");
                const bool dense = x->rows <= 1 || (x->ld_param == x->cols && x->ld_grad == x->cols);
                a.rec[k] = Rec{x->param, x->grad, x->exp_avg, x->exp_avg_sq, x->avg_scale, x->rms_scale, x->rows * x->cols, x->cols, x->ld_param, x->ld_grad,
                               (uint32_t)x->step, x->split, (x->hold ? kHold : 0u) | (x->hold_b ? kHoldB : 0u) | (dense ? 0u : kScalar), i,
                               x->lr, x->lr_b, x->weight_decay, x->weight_decay_b};
                a.begin[k++] = (uint32_t)chunks;
                chunks += more;
            }
        }
    }
    return GSX_OK;
}

constexpr uint32_t kNormGrid = 2048;

// Calls f(list, dtype) for every launch of a norm over these tensors; the lists' partial, control and blocks are the caller's.
template <class F> int norm_lists(uint32_t count, const gsx_grad_tensor* tensors, F f) {
    for (uint32_t d = 0; d <= GSX_DTYPE_F16; ++d) {
        NormList a;
        uint32_t k = 0;
        uint64_t chunks = 0;
        for (uint32_t i = 0; i <= count; ++i) {
            const gsx_grad_tensor* x = i < count ? tensors + i : nullptr;
            if (x && (x->dtype != d || x->rows == 0 || x->cols == 0)) continue;
            const uint64_t more = x ? chunks_of(x->rows * x->cols) : 0;
            if (k != 0 && (x == nullptr || k == kList || chunks + more > 0x7FFFFFFFull)) {
                for (uint32_t j = k; j < kList; ++j) a.begin[j] = 0xFFFFFFFFu;
                a.chunks = (uint32_t)chunks;
                const int rc = f(a, d);
                if (rc != GSX_OK) return rc;
                k = 0; chunks = 0;
            }
            if (x == nullptr) break;
            a.rec[k] = NormRec{x->grad, x->rows * x->cols, x->cols, x->rows > 1 ? x->ld : x->cols};
            a.begin[k++] = (uint32_t)chunks;
            chunks += more;
        }
    }
    return GSX_OK;
}

int check_grads(uint32_t count, const gsx_grad_tensor* tensors) {
    if (count != 0 && tensors == nullptr) return invalid("grad_norm_multi: null list");
    for (uint32_t i = 0; i < count; ++i) {
        const gsx_grad_tensor& x = tensors[i];
        uint64_t n;
        if (!count_of(x.rows, x.cols, &n) || chunks_of(n) > 0x7FFFFFFFull) return invalid("grad_norm_multi: tensor too large");
        if (x.dtype > GSX_DTYPE_F16) return invalid("grad_norm_multi: unknown dtype");
        if (n == 0) continue;
        if (!x.grad) return invalid("grad_norm_multi: null tensor");
        if (x.rows > 1 && x.ld < x.cols) return invalid("grad_norm_multi: rows overlap (ld smaller than cols)");
        if (x.rows > 1 && x.ld != x.cols && x.cols > (1ull << 31)) return invalid("grad_norm_multi: rows of more than 2^31 values");
    }
    return GSX_OK;
}

uint32_t norm_blocks(uint32_t count, const gsx_grad_tensor* tensors) {
    uint32_t blocks = 0;
    norm_lists(count, tensors, [&](NormList& a, uint32_t) { blocks += std::min(a.chunks, kNormGrid); return GSX_OK; });
    return std::max(blocks, 1u);
}

}  // namespace
}  // namespace gsx

using namespace gsx;

extern "C" int gsx_optim_abi_version(void) { return GSX_OPTIM_ABI_VERSION; }

extern "C" int gsx_adamw_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, const double* control,
                                    void* stream) {
    return adamw_multi(count, tensors, beta1, beta2, eps, false, 0, 0, control, stream, "adamw_step_multi");
}

extern "C" int gsx_adamw8_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, int stochastic, uint32_t seed,
                                     const double* control, void* stream) {
    return adamw_multi(count, tensors, beta1, beta2, eps, true, stochastic != 0, seed, control, stream, "adamw8_step_multi");
}

extern "C" size_t gsx_grad_norm_multi_workspace_bytes(uint32_t count, const gsx_grad_tensor* tensors) {
    if (check_grads(count, tensors) != GSX_OK) return 0;
    return (size_t)norm_blocks(count, tensors) * sizeof(double);
}

extern "C" int gsx_grad_norm_multi(uint32_t count, const gsx_grad_tensor* tensors, double max_norm, double* control, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int rc = check_grads(count, tensors);
    if (rc != GSX_OK) return rc;
    if (!(max_norm > 0.0)) return invalid("grad_norm_multi: max_norm is positive (infinite for no clipping)");
    if (control == nullptr || workspace == nullptr) return invalid("grad_norm_multi: null control block or workspace");
    const uint32_t blocks = norm_blocks(count, tensors);
    if (workspace_bytes < blocks * sizeof(double)) { set_error("grad_norm_multi: workspace too small"); return GSX_ERR_WORKSPACE_TOO_SMALL; }
    uint32_t first = 0;
    auto launch = [&](NormList& a, uint32_t d) {
        a.partial = (double*)workspace; a.control = control; a.max_norm = max_norm; a.first = first; a.blocks = blocks;
        const uint32_t grid = std::max(1u, std::min(a.chunks, kNormGrid));
        by_dtype(d, [&](auto g) { hipLaunchKernelGGL((grad_norm_kernel<decltype(g)>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a); });
        first += grid;
        return check_launch("grad_norm_multi");
    };
    const int done = norm_lists(count, tensors, launch);
    if (done != GSX_OK) return done;
    if (first == 0) {   // nothing to add up: the norm is zero
        NormList a;
        for (uint32_t j = 0; j < kList; ++j) a.begin[j] = 0xFFFFFFFFu;
        a.chunks = 0;
        return launch(a, GSX_DTYPE_F32);
    }
    return GSX_OK;
}

extern "C" int gsx_adamw8_select_rows(uint32_t count, const gsx_moments8* tensors, uint64_t rows_in, uint64_t rows_out, const int64_t* index, void* stream) {
    if (count == 0 || rows_out == 0) return GSX_OK;
    if (tensors == nullptr || index == nullptr) return invalid("adamw8_select_rows: null list or index");
    for (uint32_t i = 0; i < count; ++i) {
        const gsx_moments8& x = tensors[i];
        uint64_t n;
        if (!count_of(rows_in, x.cols, &n) || !count_of(rows_out, x.cols, &n) || chunks_of(n) > 0x7FFFFFFFull || x.cols > (1ull << 31))
            return invalid("adamw8_select_rows: tensor too large");
        if (x.cols == 0) continue;
        if (!x.avg_out || !x.rms_out || !x.avg_scale_out || !x.rms_scale_out) return invalid("adamw8_select_rows: null tensor");
        if (rows_in != 0 && (!x.avg_in || !x.rms_in || !x.avg_scale_in || !x.rms_scale_in)) return invalid("adamw8_select_rows: null tensor");
    }
    SelectList a;
    uint32_t k = 0;
    uint64_t chunks = 0;
    a.index = index; a.rows_in = rows_in; a.rows_out = rows_out;
    for (uint32_t i = 0; i <= count; ++i) {
        const gsx_moments8* x = i < count ? tensors + i : nullptr;
        if (x && x->cols == 0) continue;
        const uint64_t more = x ? chunks_of(rows_out * x->cols) : 0;
        if (k != 0 && (x == nullptr || k == kList || chunks + more > 0x7FFFFFFFull)) {
            for (uint32_t j = k; j < kList; ++j) a.begin[j] = 0xFFFFFFFFu;
            a.chunks = (uint32_t)chunks;
            hipLaunchKernelGGL(select_rows_kernel, dim3(std::min(a.chunks, kGrid)), dim3(256), 0, (hipStream_t)stream, a);
            const int rc = check_launch("adamw8_select_rows");
            if (rc != GSX_OK) return rc;
            k = 0; chunks = 0;
        }
        if (x == nullptr) break;
        a.rec[k] = SelectRec{(const uint8_t*)x->avg_in, (const uint8_t*)x->rms_in, x->avg_scale_in, x->rms_scale_in, (uint8_t*)x->avg_out, (uint8_t*)x->rms_out,
                             x->avg_scale_out, x->rms_scale_out, x->cols};
        a.begin[k++] = (uint32_t)chunks;
        chunks += more;
    }
    return GSX_OK;
}
