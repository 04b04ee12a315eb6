// gsx_adamw.hpp — what the optimizer operators over many tensors (include/gsx_optim.h) share: the list of tensors a launch takes, and the walk over its chunks.
//
// All of them are streams over memory (0.25 - 1 operation a byte): what bounds them is HBM, for small models the launch.  A launch takes its tensors as
// kernel arguments (no table in device memory: nothing to allocate, copy or keep, and a captured graph holds all it needs).  The tensors are cut into
// chunks, numbered through the list; every workgroup takes a run of consecutive chunks and looks a chunk's tensor up with one ballot of the wave for every 64 tensors:
// lane l holds the first chunk of tensor l (of l + 64, ...).
#pragma once
#include <math.h>

#include <algorithm>

#include "gsx_device.hpp"
#include "../../include/gsx_optim.h"

namespace gsx {

void set_error(const char* msg);
int check_launch(const char* what);

namespace optim {

// A launch's argument block has room for few tensors (a model's parameter groups), for some or for many (a network's): the smallest that holds the list is
// taken.  A launch with room for 16 takes 4 us of the host, for 64 one more, for 256 three more; a list of 150 in launches of 32 would take five.
constexpr uint32_t kFew = 16, kSome = 64, kMany = 256;

// Vectors of four values at any address that the type itself may have: gfx950 loads and stores them with one instruction wherever they lie.
template <class T> struct Vec4;
template <> struct Vec4<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec4<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Vec4<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2))); };
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

template <class T> GSX_DEV f32x4 load4(const T* p) {   // (of what is not read again soon)
    return __builtin_convertvector(__builtin_nontemporal_load(reinterpret_cast<const typename Vec4<T>::type*>(p)), f32x4);
}
template <class T> GSX_DEV f32x4 load4_keep(const T* p) {   // (of what is)
    return __builtin_convertvector(*reinterpret_cast<const typename Vec4<T>::type*>(p), f32x4);
}
template <class T> GSX_DEV void store4(f32x4 x, T* p) {
    typedef typename Vec4<T>::type V;
    __builtin_nontemporal_store((V)__builtin_convertvector(x, V), reinterpret_cast<V*>(p));
}

// The tensors of a launch and their chunks: begin[i] is the first chunk of tensor i, all ones behind the last tensor.
template <class R, uint32_t L> struct Chunks {
    R rec[L];
    uint32_t begin[L + 1];
    uint32_t chunks, per;   // of the launch; of a workgroup
};

// Walks this workgroup's chunks: tensor(rec, first, stop) for every tensor among them, first and stop counted within the tensor.
template <class R, uint32_t L, class T> GSX_DEV void walk(const Chunks<R, L>& a, T tensor) {
    uint32_t begin[(L + 63) / 64];
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t i = 0; i < (L + 63) / 64; ++i) begin[i] = lane + 64u * i < L ? a.begin[lane + 64u * i] : 0xFFFFFFFFu;
    uint32_t c = blockIdx.x * a.per;
    const uint32_t end = std::min(c + a.per, a.chunks);
    while (c < end) {
        uint32_t t = 0;
#pragma unroll
        for (uint32_t i = 0; i < (L + 63) / 64; ++i) t += (uint32_t)__builtin_popcountll(__ballot(c >= begin[i]));
        t = __builtin_amdgcn_readfirstlane(t - 1u);
        const uint32_t first = a.begin[t], stop = std::min(end, a.begin[t + 1]);
        tensor(a.rec[t], c - first, stop - first);
        c = stop;
    }
}

inline int invalid(const char* msg) { set_error(msg); return GSX_ERR_INVALID_ARGUMENT; }
inline uint64_t chunks_of(uint64_t n, uint32_t chunk) { return (n + chunk - 1) / chunk; }
constexpr uint64_t kMostChunks = 0x7FFFFFFFull;   // of a launch
constexpr uint32_t kMostBlocks = 1u << 23;        // of a launch: HIP counts its threads in 32 bits

// The number of values of rows x cols, or false where it is beyond what the kernels count.
inline bool count_of(uint64_t rows, uint64_t cols, uint64_t* n) {
    return !__builtin_mul_overflow(rows, cols, n) && *n <= 1ull << 40;
}

// Gathers tensors and launches them: item(i, &rec, &values) is false for a tensor that does not belong here; launch(args, workgroups) for every full list, args an
// Args<L> (with its tensors in args.c) whose other members are the launch's to fill.  per(chunks): how many of them a workgroup takes.
template <uint32_t L, template <uint32_t> class Args, class Per, class Item, class Launch>
int launch_lists_of(uint32_t count, uint32_t chunk, Per per, Item item, Launch launch) {
    Args<L> a;
    uint32_t i = 0;
    while (i < count) {
        uint32_t k = 0;
        uint64_t chunks = 0;
        for (; i < count && k < L; ++i) {
            uint64_t n = 0;
            if (!item(i, &a.c.rec[k], &n) || n == 0) continue;
            if (k != 0 && chunks + chunks_of(n, chunk) > kMostChunks) break;
            a.c.begin[k++] = (uint32_t)chunks;
            chunks += chunks_of(n, chunk);
        }
        if (k == 0) break;
        std::fill(a.c.begin + k, a.c.begin + L + 1, 0xFFFFFFFFu);
        a.c.chunks = (uint32_t)chunks;
        a.c.per = std::max(per(a.c.chunks), (a.c.chunks + kMostBlocks - 1) / kMostBlocks);
        const int rc = launch(a, (a.c.chunks + a.c.per - 1) / a.c.per);
        if (rc != GSX_OK) return rc;
    }
    return GSX_OK;
}
template <template <uint32_t> class Args, class Per, class Item, class Launch>
int launch_lists(uint32_t count, uint32_t chunk, Per per, Item item, Launch launch) {
    if (count <= kFew) return launch_lists_of<kFew, Args>(count, chunk, per, item, launch);
    if (count <= kSome) return launch_lists_of<kSome, Args>(count, chunk, per, item, launch);
    return launch_lists_of<kMany, Args>(count, chunk, per, item, launch);
}

// Launches a kernel whose one argument is a list, from where the list lies (the launch expression would copy its 2 to 32 KB once more).
template <class A> int launch_list(void (*kernel)(A), A& list, uint32_t blocks, void* stream, const char* what) {
    void* args[] = {&list};
    (void)hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3(256), args, 0, (hipStream_t)stream);
    return check_launch(what);
}

template <class F> void by_dtype(uint32_t d, F f) {
    if (d == GSX_DTYPE_F32) f(float{});
    else if (d == GSX_DTYPE_BF16) f(__bf16{});
    else f(_Float16{});
}

// ---- AdamW ---------------------------------------------------------------------------------------------------------------------------------------------
struct Rec {
    void* param; const void* grad; void* m; void* v; float* m_scale; float* v_scale;
    uint64_t n, cols, ld_param, ld_grad;
    uint32_t step, split, flags, ordinal;
    float bc1, bc2;   // 1 / (1 - beta1^t) and 1 / sqrt(1 - beta2^t) of the step; unused where it is 0: the control block's decides
    float lr, lr_b, wd, wd_b;
};
enum : uint32_t { kHold = 1, kHoldB = 2, kRows = 4 };   // kRows: parameter or gradient is a view whose rows lie apart

struct Betas {
    const double* control;
    double log_b1, log_b2;
    float b1, b1c, b2, b2c, eps;   // (eps at least 2^-126)
    uint32_t seed;
};

// 1 - exp(x), x <= 0, to 6 * 2^-24 of itself (x is rounded too): the series where it is small, where 1 - exp(x) would lose its leading digits (beta2 = 0.999, first step: 1e-4
// of it).  A third of the library's expm1f in instructions; every workgroup computes it.
GSX_DEV float one_minus_exp(float x) {
    float s = 1.0f / 40320.0f;   // (1 + x/2 + x^2/6 + ...: what is cut is below x^8 / 9!, 2^-26 at -1/2)
    s = fmaf(s, x, 1.0f / 5040.0f); s = fmaf(s, x, 1.0f / 720.0f); s = fmaf(s, x, 1.0f / 120.0f);
    s = fmaf(s, x, 1.0f / 24.0f); s = fmaf(s, x, 1.0f / 6.0f); s = fmaf(s, x, 0.5f); s = fmaf(s, x, 1.0f);
    return x > -0.5f ? -x * s : 1.0f - __builtin_amdgcn_exp2f(x * 1.44269504f);
}

// What the control block says, and the bias corrections of its step.  1 - beta^t = 1 - exp(t log beta), the product in 64 bits.
struct Control { bool skip; float factor, bc1, bc2; uint32_t step; };
GSX_DEV Control control_of(const Betas& a) {
    Control c = {false, 1.0f, 0.0f, 0.0f, 0u};
    if (a.control == nullptr) return c;
    c.skip = a.control[2] != 0.0;
    c.factor = (float)a.control[1];
    c.step = std::max((uint32_t)a.control[3], 1u);   // (a block that no norm has advanced: the first step)
    c.bc1 = __builtin_amdgcn_rcpf(one_minus_exp((float)(a.log_b1 * (double)c.step)));
    c.bc2 = __builtin_amdgcn_rsqf(one_minus_exp((float)(a.log_b2 * (double)c.step)));
    return c;
}

struct Rates { float step, step_b, lrwd, lrwd_b, bc2; uint32_t split, flags; };
GSX_DEV Rates rates_of(const Rec& r, const Control& c) {
    const float bc1 = r.step ? r.bc1 : c.bc1;
    return {r.lr * bc1, r.lr_b * bc1, r.lr * r.wd, r.lr_b * r.wd_b, r.step ? r.bc2 : c.bc2, r.split, r.flags};
}

// The moments as the formulas write them, each product and sum rounded by itself: what is stored in 8 bits is then a function of the inputs that can be
// computed anywhere to the last bit (a fused product moves a value by 2^-25, and where it lies next to a border of the format, its code by a whole step).
GSX_DEV float first_moment(const Betas& a, float m, float g) {
#pragma clang fp contract(off)
    return a.b1 * m + a.b1c * g;
}
GSX_DEV float second_moment(const Betas& a, float v, float g) {
#pragma clang fp contract(off)
    return a.b2 * v + a.b2c * g * g;
}

// The rates of a lane's four values, c the column of the first of them, and which of the values their group holds as they are.
struct Steps { float lrwd[4], step[4]; };
GSX_DEV Steps steps_of(const Rates& k, uint32_t c, uint32_t cols, uint32_t* held = nullptr) {
    Steps o;
    if (held) *held = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) { o.lrwd[j] = k.lrwd; o.step[j] = k.step; }
    if (k.split) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool b = c >= k.split;
            o.lrwd[j] = b ? k.lrwd_b : k.lrwd;
            o.step[j] = b ? k.step_b : k.step;
            if (held) *held |= k.flags & (b ? kHoldB : kHold) ? 1u << j : 0u;
            ++c;
            c = std::min(c, c - cols);   // (c - cols wraps round to a large number while c is a column)
        }
    } else if (held && (k.flags & kHold)) {
        *held = 15u;
    }
    return o;
}

// One parameter's step, after its moments (root: sqrt(v)).  The denominator is at least eps, which is at least 2^-126 (betas_of): its reciprocal is the
// hardware's (1 ulp).
GSX_DEV float stepped(const Betas& a, const Rates& k, float lrwd, float step, float p, float m, float root) {
    return p - lrwd * p - step * m * __builtin_amdgcn_rcpf(root * k.bc2 + a.eps);
}

// Where the values of a chunk lie.  Rows and columns are followed from chunk to chunk, and only where something goes by them.
struct Place {
    const uint64_t n;
    const uint32_t cols;
    const bool view, by_column;
    uint64_t base, row = 0;   // first value of the chunk, and its row (of a view)
    uint32_t col = 0, count;  // its column; values in the chunk
    uint32_t mine = 0;        // column of the lane's first value (of four)
    bool whole;               // a full chunk, its values one behind the other in all of the tensor's arrays
    GSX_DEV Place(const Rec& r, uint32_t split, uint32_t index, uint32_t chunk)
        : n(r.n), cols((uint32_t)r.cols), view(r.flags & kRows), by_column(split || view), base((uint64_t)index * chunk) {
        if (view || (split && cols > 0xFFFFu)) {
            row = base / r.cols;
            col = (uint32_t)(base - row * r.cols);
        } else if (split) {   // (the same without a quotient of 64 bits, which would be a fifth of the instructions of a pass)
            col = (index % cols) * (chunk % cols) % cols;
        }
        if (by_column) mine = (col + threadIdx.x * 4u) % cols;
        size(chunk);
    }
    GSX_DEV void size(uint32_t chunk) {
        count = (uint32_t)std::min<uint64_t>(n - base, chunk);
        whole = !view && count == chunk;
    }
    GSX_DEV void next(uint32_t chunk) {
        base += chunk;
        if (by_column) {
            const uint32_t q = col + chunk, dr = q / cols;
            row += dr;
            mine += q - dr * cols >= col ? q - dr * cols - col : q - dr * cols + cols - col;   // (the step from column to column, less than cols)
            mine = std::min(mine, mine - cols);
            col = q - dr * cols;
        }
        size(chunk);   // (behind the last chunk: not used)
    }
    // Value i of the chunk: its column, and where it is in an array whose rows are ld apart if the tensor is a view.
    struct Spot { uint32_t i, dr, c; };
    GSX_DEV Spot spot(uint32_t i) const {
        if (!by_column) return {i, 0, 0};
        const uint32_t q = col + i, dr = q / cols;
        return {i, dr, q - dr * cols};
    }
    GSX_DEV uint64_t operator()(Spot s, uint64_t ld) const { return view ? (row + s.dr) * ld + s.c : base + s.i; }
};

// Whether any of the tensors has a group that is held: kernels of their own (held groups inside the others took 20 registers and two of the six waves).
inline bool any_held(uint32_t count, const gsx_adamw_tensor* tensors) {
    for (uint32_t i = 0; i < count; ++i)
        if (tensors[i].hold || (tensors[i].split && tensors[i].hold_b)) return true;
    return false;
}

// The pairs of parameter and gradient types among the tensors: bit 3 * param_dtype + grad_dtype.
inline uint32_t types_of(uint32_t count, const gsx_adamw_tensor* tensors) {
    uint32_t mask = 0;
    for (uint32_t i = 0; i < count; ++i) mask |= 1u << (3 * tensors[i].param_dtype + tensors[i].grad_dtype);
    return mask;
}

struct Corrections { uint64_t step; float bc1, bc2; };
int check_adamw(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, bool eight, const double* control);
Betas betas_of(double beta1, double beta2, double eps, uint32_t seed, const double* control);
Rec rec_of(const gsx_adamw_tensor& x, uint32_t ordinal, const Betas& b, Corrections* last);

}  // namespace optim
}  // namespace gsx
