// gsx_adamw.hip — AdamW over many tensors with moments in 32 bits, and the norm of all gradients (include/gsx_optim.h).
#include "gsx_adamw.hpp"

namespace gsx {
namespace optim {

constexpr uint32_t kChunk = 1024;   // values of one pass of a workgroup: four of each lane
// One chunk to a workgroup: what is in flight then lies close together in every one of the arrays.  5 M splats (8.3 GB): 5.8 TB/s; runs of 18 chunks, which spread
// the 2 048 workgroups in flight over 150 MB of every array, 5.2.
constexpr uint32_t kPer = 1;

template <uint32_t L> struct List { static constexpr uint32_t kRoom = L; Chunks<Rec, L> c; Betas b; };

template <class P, class G, bool HELD, uint32_t L>
__global__ __launch_bounds__(256) void adamw_kernel(List<L> list) {
    const Betas& a = list.b;
    const Control ctl = control_of(a);
    if (ctl.skip) return;
    walk(list.c, [&](const Rec& r, uint32_t chunk, uint32_t stop) {
        const Rates k = rates_of(r, ctl);
        Place at(r, k.split, chunk, kChunk);
        for (; chunk < stop; ++chunk, at.next(kChunk)) {
            float* m = (float*)r.m + at.base; float* v = (float*)r.v + at.base;
            if (at.whole) {
                const uint32_t off = threadIdx.x * 4u;
                f32x4 gv = load4((const G*)r.grad + at.base + off), mv = load4(m + off), vv = load4(v + off), pv = load4((const P*)r.param + at.base + off);
                uint32_t held = 0;
                const Steps o = steps_of(k, at.mine, at.cols, HELD ? &held : nullptr);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float g1 = gv[j] * ctl.factor, m1 = a.b1 * mv[j] + a.b1c * g1, v1 = a.b2 * vv[j] + a.b2c * g1 * g1;
                    const float p1 = stepped(a, k, o.lrwd[j], o.step[j], pv[j], m1, sqrtf(v1));
                    const bool keep = HELD && (held >> j & 1u);
                    mv[j] = keep ? mv[j] : m1;
                    vv[j] = keep ? vv[j] : v1;
                    pv[j] = keep ? pv[j] : p1;
                }
                store4(mv, m + off);
                store4(vv, v + off);
                store4(pv, (P*)r.param + at.base + off);
                continue;
            }
            // the end of a tensor, or a view: neighbouring values to neighbouring lanes, all loads of a lane at once, none behind the end
            float gv[4], mv[4], vv[4], pv[4];
            Place::Spot s[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                s[j] = at.spot(std::min(j * 256u + threadIdx.x, at.count - 1u));
                gv[j] = (float)((const G*)r.grad)[at(s[j], r.ld_grad)];
                pv[j] = (float)((const P*)r.param)[at(s[j], r.ld_param)];
                mv[j] = m[s[j].i];
                vv[j] = v[s[j].i];
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const bool b = k.split && s[j].c >= k.split;
                if (j * 256u + threadIdx.x >= at.count || (HELD && (k.flags & (b ? kHoldB : kHold)))) continue;
                const float g1 = gv[j] * ctl.factor, m1 = a.b1 * mv[j] + a.b1c * g1, v1 = a.b2 * vv[j] + a.b2c * g1 * g1;
                ((P*)r.param)[at(s[j], r.ld_param)] = (P)stepped(a, k, b ? k.lrwd_b : k.lrwd, b ? k.step_b : k.step, pv[j], m1, sqrtf(v1));
                m[s[j].i] = m1;
                v[s[j].i] = v1;
            }
        }
    });
}

// ---- the norm ----------------------------------------------------------------------------------------------------------------------------------------
constexpr uint32_t kNormVecs = 4, kNormChunk = 1024 * kNormVecs, kNormGrid = 2048;
// Up to this many workgroups the last one to finish adds the sums up; every one costs 45 ns there (an atomic on one word, and what the release before it waits for: 2 048 of
// them took 100 of 284 us), a launch of its own 3 us.  66 workgroups: 6.0 us in one launch, 7.8 in two; 175: 7.9 and 7.8.
constexpr uint32_t kTickets = 128;
// Gradients that fit the last-level cache (256 MB) are read to stay there for the update behind the norm: 1 M splats, norm and update 300 us (330 without; 8-bit moments
// 195 and 201), the norm alone 47 (43).  Larger ones stream past it: 295 M values 178 us, 203 without.
constexpr uint64_t kCacheBytes = 256ull << 20;

struct NormRec { const void* grad; uint64_t n, cols, ld; };
struct NormEnd { double* partial; double* control; double max_norm; uint32_t blocks; };   // partial: one for each workgroup of the whole call
template <uint32_t L> struct NormList {
    static constexpr uint32_t kRoom = L;
    Chunks<NormRec, L> c;
    NormEnd e;
    uint32_t first;   // this launch's first partial
};

template <int C> GSX_DEV double dpp_add(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, C, 0xF, 0xF, true);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), C, 0xF, 0xF, true);
    return x + __longlong_as_double((long long)((uint64_t)high << 32 | low));
}
GSX_DEV double of_lane(double x, int lane) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), high = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __longlong_as_double((long long)((uint64_t)high << 32 | low));
}
// Sum over the workgroup, in all of it: within the rows of 16 lanes, over a wave's four rows, over the four waves.
GSX_DEV double block_sum(double x, double* lds) {
    x = dpp_add<0xB1>(x);    // neighbours
    x = dpp_add<0x4E>(x);    // pairs of a quad
    x = dpp_add<0x141>(x);   // halves of eight
    x = dpp_add<0x140>(x);   // halves of a row
    x = (of_lane(x, 0) + of_lane(x, 16)) + (of_lane(x, 32) + of_lane(x, 48));
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// One workgroup adds the partial sums up in their order (the same bits every time) and writes the control block.
GSX_DEV void norm_end(const NormEnd& e, double* lds) {
    double total = 0.0;
    for (uint32_t i = threadIdx.x; i < e.blocks; i += 256u) total += __hip_atomic_load(e.partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    total = block_sum(total, lds);
    if (threadIdx.x == 0) {
        const bool fine = isfinite(total);
        const double norm = sqrt(total);
        e.control[0] = norm;
        e.control[1] = fine ? fmin(1.0, e.max_norm / (norm + 1e-6)) : 0.0;
        e.control[2] = fine ? 0.0 : 1.0;
        e.control[3] += fine ? 1.0 : 0.0;
    }
}

// Sums of squares in 64 bits: no square of a 32-bit number overflows, so the sum is finite exactly if all gradients are.
template <class G, uint32_t L, bool KEEP>
__global__ __launch_bounds__(256) void grad_norm_kernel(NormList<L> a) {
    __shared__ double lds[4];
    __shared__ uint32_t last;
    double sum = 0.0;
    walk(a.c, [&](const NormRec& r, uint32_t chunk, uint32_t stop) {
        const uint64_t n = r.n;
        const bool view = r.ld != r.cols;
        for (; chunk < stop; ++chunk) {
            const uint64_t base = (uint64_t)chunk * kNormChunk;
            const uint32_t count = (uint32_t)std::min<uint64_t>(n - base, kNormChunk);
            const G* g = (const G*)r.grad + base;
            if (!view) {
                f32x4 x[kNormVecs];
#pragma unroll
                for (uint32_t u = 0; u < kNormVecs; ++u) {
                    const uint32_t off = (u * 256u + threadIdx.x) * 4u;
                    x[u] = off + 4 > count ? f32x4{0, 0, 0, 0} : KEEP ? load4_keep(g + off) : load4(g + off);
                }
#pragma unroll
                for (uint32_t u = 0; u < kNormVecs; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum = fma((double)x[u][j], (double)x[u][j], sum);
                if (const uint32_t rest = count & 3u; rest != 0 && threadIdx.x < rest) {   // the last one to three values of the tensor
                    const double x1 = (double)(float)g[(count & ~3u) + threadIdx.x];
                    sum = fma(x1, x1, sum);
                }
            } else {
                const uint64_t row = base / r.cols;
                const uint32_t col = (uint32_t)(base - row * r.cols), cols = (uint32_t)r.cols;
                for (uint32_t off = threadIdx.x; off < count; off += 256u) {
                    const uint32_t q = col + off, dr = q / cols;
                    const double x1 = (double)(float)((const G*)r.grad)[(row + dr) * r.ld + (q - dr * cols)];
                    sum = fma(x1, x1, sum);
                }
            }
        }
    });
    sum = block_sum(sum, lds);
    uint32_t* ticket = reinterpret_cast<uint32_t*>(a.e.control + 4);
    if (threadIdx.x == 0) {
        __hip_atomic_store(a.e.partial + a.first + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = a.e.blocks <= kTickets && __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.e.blocks - 1u;
    }
    __syncthreads();
    if (!last) return;
    norm_end(a.e, lds);
    if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(256) void grad_norm_end_kernel(NormEnd e) {
    __shared__ double lds[4];
    norm_end(e, lds);
}

// Calls f(list, workgroups, dtype) for every launch of a norm over these tensors; what the lists hold besides the tensors is f's.
template <class F> int norm_lists(uint32_t count, const gsx_grad_tensor* tensors, F f) {
    uint32_t mask = 0;
    for (uint32_t i = 0; i < count; ++i) mask |= 1u << tensors[i].dtype;
    for (uint32_t d = 0; d <= GSX_DTYPE_F16; ++d) {
        if (!(mask >> d & 1u)) continue;
        const int rc = launch_lists<NormList>(
            count, kNormChunk, [](uint32_t chunks) { return (chunks + kNormGrid - 1) / kNormGrid; },
            [&](uint32_t i, NormRec* r, uint64_t* n) {
                const gsx_grad_tensor& x = tensors[i];
                *n = x.rows * x.cols;
                *r = NormRec{x.grad, *n, x.cols, x.rows > 1 ? x.ld : x.cols};
                return x.dtype == d;
            },
            [&](auto& a, uint32_t blocks) { return f(a, blocks, d); });
        if (rc != GSX_OK) return rc;
    }
    return GSX_OK;
}

int check_grads(uint32_t count, const gsx_grad_tensor* tensors) {
    if (count != 0 && tensors == nullptr) return invalid("grad_norm_multi: null list");
    for (uint32_t i = 0; i < count; ++i) {
        const gsx_grad_tensor& x = tensors[i];
        uint64_t n;
        if (!count_of(x.rows, x.cols, &n)) return invalid("grad_norm_multi: tensor too large");
        if (x.dtype > GSX_DTYPE_F16) return invalid("grad_norm_multi: unknown dtype");
        if (n == 0) continue;
        if (!x.grad) return invalid("grad_norm_multi: null tensor");
        if (x.rows > 1 && x.ld < x.cols) return invalid("grad_norm_multi: rows overlap (ld smaller than cols)");
        if (x.rows > 1 && x.ld != x.cols && x.cols > (1ull << 31)) return invalid("grad_norm_multi: rows of more than 2^31 values");
    }
    return GSX_OK;
}

uint32_t norm_blocks(uint32_t count, const gsx_grad_tensor* tensors) {
    uint32_t sum = 0;
    norm_lists(count, tensors, [&](auto&, uint32_t blocks, uint32_t) { sum += blocks; return GSX_OK; });
    return std::max(sum, 1u);
}

// Room for the sums of all workgroups: three types, each in launches of up to kMany tensors.
size_t norm_bytes(uint32_t count) { return ((size_t)count / kMany + 3) * kNormGrid * sizeof(double); }

// ---- what both AdamW entry points check and prepare -----------------------------------------------------------------------------------------------------
int check_adamw(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, bool eight, const double* control) {
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
    return GSX_OK;
}

Betas betas_of(double beta1, double beta2, double eps, uint32_t seed, const double* control) {
    return Betas{control, log(beta1), log(beta2), (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), std::max((float)eps, 0x1p-126f), seed};
}

Rec rec_of(const gsx_adamw_tensor& x, uint32_t ordinal, const Betas& b, Corrections* last) {
    if (last->step != x.step || last->step == 0)   // (the tensors of a list mostly share their step)
        *last = Corrections{x.step, (float)(1.0 / -expm1(b.log_b1 * (double)x.step)), (float)(1.0 / sqrt(-expm1(b.log_b2 * (double)x.step)))};
    const bool dense = x.rows <= 1 || (x.ld_param == x.cols && x.ld_grad == x.cols);
    return Rec{x.param, x.grad, x.exp_avg, x.exp_avg_sq, x.avg_scale, x.rms_scale, x.rows * x.cols, x.cols, x.ld_param, x.ld_grad, (uint32_t)x.step, x.split,
               (x.hold ? kHold : 0u) | (x.hold_b ? kHoldB : 0u) | (dense ? 0u : kRows), ordinal, last->bc1, last->bc2, x.lr, x.lr_b, x.weight_decay,
               x.weight_decay_b};
}

}  // namespace optim
}  // namespace gsx

using namespace gsx;
using namespace gsx::optim;

extern "C" int gsx_optim_abi_version(void) { return GSX_OPTIM_ABI_VERSION; }

extern "C" int gsx_adamw_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, const double* control,
                                    void* stream) {
    const int bad = check_adamw(count, tensors, beta1, beta2, eps, false, control);
    if (bad != GSX_OK || count == 0) return bad;
    const Betas betas = betas_of(beta1, beta2, eps, 0, control);
    Corrections last = {};
    const uint32_t mask = types_of(count, tensors);
    const bool held = any_held(count, tensors);
    for (uint32_t types = 0; types < 9; ++types) {
        if (!(mask >> types & 1u)) continue;
        const uint32_t pd = types / 3, gd = types % 3;
        const int rc = launch_lists<List>(
            count, kChunk, [](uint32_t) { return kPer; },
            [&](uint32_t i, Rec* r, uint64_t* n) {
                if (tensors[i].param_dtype != pd || tensors[i].grad_dtype != gd) return false;
                *r = rec_of(tensors[i], i, betas, &last);
                *n = r->n;
                return true;
            },
            [&](auto& a, uint32_t blocks) {
                a.b = betas;
                int rc = GSX_OK;
                by_dtype(pd, [&](auto p) {
                    by_dtype(gd, [&](auto g) {
                        constexpr uint32_t L = std::remove_reference_t<decltype(a)>::kRoom;
                        typedef decltype(p) P;
                        typedef decltype(g) G;
                        rc = launch_list(held ? adamw_kernel<P, G, true, L> : adamw_kernel<P, G, false, L>, a, blocks, stream, "adamw_step_multi");
                    });
                });
                return rc;
            });
        if (rc != GSX_OK) return rc;
    }
    return GSX_OK;
}

extern "C" size_t gsx_grad_norm_multi_workspace_bytes(uint32_t count, const gsx_grad_tensor* tensors) {
    return check_grads(count, tensors) == GSX_OK ? norm_bytes(count) : 0;
}

extern "C" int gsx_grad_norm_multi(uint32_t count, const gsx_grad_tensor* tensors, double max_norm, double* control, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int bad = check_grads(count, tensors);
    if (bad != GSX_OK) return bad;
    if (!(max_norm > 0.0)) return invalid("grad_norm_multi: max_norm is positive (infinite for no clipping)");
    if (control == nullptr || workspace == nullptr) return invalid("grad_norm_multi: null control block or workspace");
    const uint32_t blocks = norm_blocks(count, tensors);
    if (workspace_bytes < std::max(norm_bytes(count), blocks * sizeof(double))) { set_error("grad_norm_multi: workspace too small"); return GSX_ERR_WORKSPACE_TOO_SMALL; }
    uint64_t bytes = 0;
    for (uint32_t i = 0; i < count; ++i) bytes += tensors[i].rows * tensors[i].cols * (tensors[i].dtype == GSX_DTYPE_F32 ? 4 : 2);
    const NormEnd end = {(double*)workspace, control, max_norm, blocks};
    uint32_t first = 0;
    auto launch = [&](auto& a, uint32_t grid, uint32_t d) {
        a.e = end; a.first = first;
        int rc = GSX_OK;
        by_dtype(d, [&](auto g) {
            typedef decltype(g) G;
            constexpr uint32_t L = std::remove_reference_t<decltype(a)>::kRoom;
            rc = launch_list(bytes <= kCacheBytes ? grad_norm_kernel<G, L, true> : grad_norm_kernel<G, L, false>, a, grid, stream, "grad_norm_multi");
        });
        first += grid;
        return rc;
    };
    int rc = norm_lists(count, tensors, launch);
    if (rc == GSX_OK && first == 0) {   // nothing to add up: the norm is zero
        NormList<kFew> none;
        for (uint32_t j = 0; j <= kFew; ++j) none.c.begin[j] = 0xFFFFFFFFu;
        none.c.chunks = 0;
        none.c.per = 1;
        rc = launch(none, 1, GSX_DTYPE_F32);
    }
    if (rc != GSX_OK || blocks <= kTickets) return rc;
    hipLaunchKernelGGL(grad_norm_end_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, end);
    return check_launch("grad_norm_multi");
}
