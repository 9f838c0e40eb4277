// A step of AdamW over many tensors at once, with moments in 32 or in 8 bits.
//   g = diff * factor;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   w = w - lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay w)
// Bound by memory: 28 bytes an element with fp32 weights and moments, 16 with fp16 weights, their fp32 copies and moments in 8 bits, which takes
// some sixty operations.  A wave has 256 elements at a time, four neighbours a lane: they are what shares a scale in 8 bits, so that its largest
// root is found without a barrier.  The tensors' places travel in the kernel's arguments, 32 tensors a launch: no table in memory has to
// be written, and the launches can be captured.
// Measured: 23 million fp32 weights and moments 110 us (5.9 TB/s), 92 million fp16 weights with copies and moments in 8 bits 247 us (6.0); a large
// copy reaches 5.0 on the same card.  1 million fp32 weights in 12 tensors 7.3 us.
// In 8 bits the roots are held, not the moments: a block's moments span decades (v the squares of m's), and the fourth root brings
// the 65025^2 that v spans between its smallest code and its largest to 255.
#include <memory>
#include <new>

#include "ptl_row_sums.hpp"
#include "ptl_rows.hpp"
#include "ptl_tuning.h"

namespace ptl {

constexpr int ADAM_BLOCK = 256;   // elements of a scale
constexpr int ADAM_TENSORS = 32;

struct AdamTensor {
    const void *g, *w;        // w: NULL where `master` is read
    void *w_out;
    const float *master;      // NULL: w is read
    float *master_out;        // NULL: none
    const void *m, *v;        // fp32, or codes; NULL: 0
    void *m_out, *v_out;
    const float *m_scale, *v_scale;  // (m_scale_out NULL: moments in fp32)
    float *m_scale_out, *v_scale_out;
    float lr, decay;
    unsigned n;               // elements
};
struct AdamTable {
    unsigned first[ADAM_TENSORS];  // workgroup of each tensor (behind the last: none)
    AdamTensor t[ADAM_TENSORS];
    int count;
    float b1, c1, b2, c2, eps;     // c1 = 1 - b1, c2 = 1 - b2
    float i1, i2, root2;           // 1 / (1 - b1^t), 1 / (1 - b2^t) and its root
    float log1, log2;              // of b1 and b2, where t is read from ...
    const int *step;               // (NULL: i1 and i2 are given)
    const float *factor;           // (NULL: 1)
};
static_assert(sizeof(AdamTable) <= 4096, "kernel arguments");

typedef unsigned adam_u4 __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned adam_u2 __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned adam_u1 __attribute__((aligned(1)));
template <int BYTES>
struct AdamRaw;
template <>
struct AdamRaw<4> { typedef adam_u4 type; };
template <>
struct AdamRaw<2> { typedef adam_u2 type; };
template <>
struct AdamRaw<1> { typedef adam_u1 type; };

// Four neighbouring values, of which `left` exist (4 and more: all).  Stores pass by the caches, and so do loads (STREAM) of calls that move more
// than the caches hold.
template <typename S>
struct Adam4 {
    typedef typename AdamRaw<sizeof(S)>::type Raw;
    union {
        Raw raw;
        S e[4];
    };
    template <bool STREAM>
    __device__ inline void load(const void *from, size_t at, long left) {
        const S *p = static_cast<const S *>(from) + at;
        if (left >= 4) {
            raw = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const Raw *>(p)) : *reinterpret_cast<const Raw *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = i < left ? p[i] : (S)0;
        }
    }
    __device__ inline void store(void *to, size_t at, long left) const {
        S *p = static_cast<S *>(to) + at;
        if (left >= 4) {
            __builtin_nontemporal_store(raw, reinterpret_cast<Raw *>(p));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) p[i] = e[i];
        }
    }
};

// The root to one step of fp32, as the inverse below is: the step of a weight, lr times their quotient, is off by some 1e-7 of itself, which is less than its sum with
// the weight rounds away; a division and a root that are rounded right are another twenty instructions for each element.  The instruction takes subnormal values for 0, so small ones are worked on 2^64 times as large.
__device__ inline float adam_root(float x) {
    const bool tiny = x < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(tiny ? x * 0x1p64f : x);
    return tiny ? r * 0x1p-32f : r;
}

// What a launch has in registers of a lane's four elements.
template <typename T>
struct AdamPart {
    Adam4<T> g, w;
    Adam4<float> master;
};

struct AdamRates {
    float b1, c1, b2, c2, eps, i1, i2, factor, lr, decay, root2;  // root2: of i2
    // One element: the moments and the weight behind the step.  Moments in 8 bits (ROOT: the root of v is wanted too, and subnormal ones are 0).
    template <bool ROOT>
    __device__ inline float step(float g, float &m, float &v, float &w) const {
        g *= factor;
        m = fmaf(b1, m, c1 * g);
        v = fmaf(b2, v, c2 * g * g);
        const float root = ROOT ? __builtin_amdgcn_sqrtf(v) : adam_root(v * i2);
        w = fmaf(-lr, fmaf(decay, w, m * i1 * __builtin_amdgcn_rcpf(ROOT ? fmaf(root, root2, eps) : root + eps)), w);
        return root;
    }
};

// Four weights behind the step, in both forms.
template <typename T>
__device__ inline void adam_put(const AdamTensor &t, const float (&w)[4], size_t at, long left) {
    Adam4<T> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.e[i] = row_round<T>(w[i]);
    o.store(t.w_out, at, left);
    if (t.master_out) {
        Adam4<float> f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f.e[i] = w[i];
        f.store(t.master_out, at, left);
    }
}

template <typename T>
__device__ inline void adam_weights(const AdamTensor &t, const AdamPart<T> &p, float (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = t.master ? p.master.e[i] : (float)p.w.e[i];
}

// The largest of four magnitudes over the wave, or what is no number: as integers they have the same order, and NaN is the largest.
__device__ inline float adam_most(const float (&f)[4]) {
    unsigned u = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) u = max(u, __builtin_bit_cast(unsigned, f[i]) & 0x7fffffffu);
    return lanes_most(u);
}
// 127 or 255 over the largest root, 0 where that is 0 or no number.
template <int MOST>
__device__ inline float adam_unit(float most) { return most > 0.f ? (float)MOST / most : 0.f; }
// An integer in the low bits of a float: 2^23 + 2^22 leave no room for anything else, so that the addition rounds to it (ties to even).
constexpr float ADAM_INTEGER = 12582912.f;
__device__ inline unsigned adam_pack(const float (&f)[4]) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(unsigned, f[i]);
    // (the low byte of each: bytes 0 and 4 of a pair)
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
}

// A step that changes nothing: what is not updated in place is copied.
template <typename T>
__device__ inline void adam_copy(const AdamTensor &t, size_t at, long left, size_t block, int lane) {
    if (t.w != t.w_out || t.master) {
        AdamPart<T> p;
        float w[4];
        if (t.master) p.master.template load<false>(t.master, at, left);
        else p.w.template load<false>(t.w, at, left);
        adam_weights<T>(t, p, w);
        AdamTensor o = t;
        if (t.master_out == t.master) o.master_out = nullptr;
        if (!t.master || t.w != t.w_out) adam_put<T>(o, w, at, left);
        else if (o.master_out) p.master.store(o.master_out, at, left);
    } else if (t.master_out) {  // (the weights in fp32 begin here)
        AdamPart<T> p;
        Adam4<float> f;
        p.w.template load<false>(t.w, at, left);
#pragma unroll
        for (int i = 0; i < 4; ++i) f.e[i] = (float)p.w.e[i];
        f.store(t.master_out, at, left);
    }
    // (each moment and each scale may have a place of its own, or that of the old one)
    if (t.m_scale_out) {
        auto codes = [&](const void *from, void *to) {
            Adam4<int8_t> c = {};
            if (from) c.load<false>(from, at, left);
            if (from != to) c.store(to, at, left);
        };
        codes(t.m, t.m_out);
        codes(t.v, t.v_out);
        if (lane == 0 && t.m_scale != t.m_scale_out) t.m_scale_out[block] = t.m ? t.m_scale[block] : 0.f;
        if (lane == 0 && t.v_scale != t.v_scale_out) t.v_scale_out[block] = t.m ? t.v_scale[block] : 0.f;
    } else {
        auto moments = [&](const void *from, void *to) {
            Adam4<float> f = {};
            if (from) f.load<false>(from, at, left);
            if (from != to) f.store(to, at, left);
        };
        moments(t.m, t.m_out);
        moments(t.v, t.v_out);
    }
}

template <typename T, int U, bool STREAM>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamTable a) {
    int k = 0;  // (those behind the last begin nowhere)
#pragma unroll
    for (int half = ADAM_TENSORS / 2; half >= 1; half /= 2)
        if (blockIdx.x >= a.first[k + half]) k += half;
    const AdamTensor &t = a.t[k];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (a workgroup's blocks lie side by side: wave w has blocks w, w + 4, ...)
    const size_t first = (size_t)(blockIdx.x - a.first[k]) * (4 * U) + wave;
    auto place = [&](int u) { return (first + 4 * u) * ADAM_BLOCK + 4 * (size_t)lane; };
    auto left = [&](int u) { return (long)t.n - (long)place(u); };
    auto none = [&](int u) { return (first + 4 * u) * ADAM_BLOCK >= t.n; };  // (of the whole wave)
    AdamPart<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (none(u)) break;
        p[u].g.template load<STREAM>(t.g, place(u), left(u));
        if (t.master) p[u].master.template load<STREAM>(t.master, place(u), left(u));
        else p[u].w.template load<STREAM>(t.w, place(u), left(u));
    }
    AdamRates r = {a.b1, a.c1, a.b2, a.c2, a.eps, a.i1, a.i2, a.factor ? *a.factor : 1.f, t.lr, t.decay, a.root2};
    if (!(fabsf(r.factor) < __builtin_inff())) {
#pragma unroll 1
        for (int u = 0; u < U; ++u)
            if (!none(u)) adam_copy<T>(t, place(u), left(u), first + 4 * u, lane);
        return;
    }
    if (a.step) {
        const float s = (float)*a.step;
        r.i1 = -1.f / expm1f(s * a.log1);
        r.i2 = -1.f / expm1f(s * a.log2);
        r.root2 = sqrtf(r.i2);
    }
    if (t.m_scale_out) {
        Adam4<int8_t> mq[U], vq[U];
        float ms[U], vs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (none(u)) break;
            ms[u] = vs[u] = 0.f;
            mq[u].raw = vq[u].raw = 0;
            if (!t.m) continue;
            mq[u].template load<STREAM>(t.m, place(u), left(u));
            vq[u].template load<STREAM>(t.v, place(u), left(u));
            ms[u] = t.m_scale[first + 4 * u];
            vs[u] = t.v_scale[first + 4 * u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (none(u)) break;
            float w[4], m[4], v[4];  // (later their roots, that of m with its sign)
            adam_weights<T>(t, p[u], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = (float)mq[u].e[i] * ms[u], c = (float)(uint8_t)vq[u].e[i] * vs[u];
                m[i] = q * fabsf(q);
                v[i] = c * c * (c * c);
                const float root = r.template step<true>((float)p[u].g.e[i], m[i], v[i], w[i]);
                m[i] = copysignf(__builtin_amdgcn_sqrtf(fabsf(m[i])), m[i]);
                v[i] = __builtin_amdgcn_sqrtf(root);
            }
            adam_put<T>(t, w, place(u), left(u));
            const float m_most = adam_most(m), v_most = adam_most(v), m_unit = adam_unit<127>(m_most), v_unit = adam_unit<255>(v_most);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[i] = fmaf(m[i], m_unit, ADAM_INTEGER);
                // (1 at least where there is a root at all: the smallest is 1e-10)
                v[i] = fmaxf(v[i] * v_unit, __builtin_amdgcn_fmed3f(v[i] * 1e30f, 0.f, 1.f)) + ADAM_INTEGER;
            }
            Adam4<int8_t> mo, vo;
            mo.raw = adam_pack(m);
            vo.raw = adam_pack(v);
            mo.store(t.m_out, place(u), left(u));
            vo.store(t.v_out, place(u), left(u));
            if (lane == 0) {
                t.m_scale_out[first + 4 * u] = m_most / 127.f;
                t.v_scale_out[first + 4 * u] = v_most / 255.f;
            }
        }
    } else {
        Adam4<float> mv[U], vv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (none(u)) break;
            mv[u].raw = vv[u].raw = adam_u4{0, 0, 0, 0};
            if (!t.m) continue;
            mv[u].template load<STREAM>(t.m, place(u), left(u));
            vv[u].template load<STREAM>(t.v, place(u), left(u));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (none(u)) break;
            float w[4];
            adam_weights<T>(t, p[u], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) r.template step<false>((float)p[u].g.e[i], mv[u].e[i], vv[u].e[i], w[i]);
            adam_put<T>(t, w, place(u), left(u));
            mv[u].store(t.m_out, place(u), left(u));
            vv[u].store(t.v_out, place(u), left(u));
        }
    }
}

// What is wrong with a tensor's arguments (NULL: nothing).
template <typename Args>
static const char *adamw_check(const Args &a) {
    if (!a.weights) return "null argument structure";
    const adamw_state *to = a.new_state ? a.new_state : a.state, *from = a.state;
    if (!to) return "neither state nor new_state is given";
    if (a.weights->dim < 0 || (a.updated && a.updated->dim != a.weights->dim)) return "invalid tensor geometry";
    if (a.weights->dim == 0) return nullptr;
    const bool eight = to->m_root != nullptr;
    auto whole = [&](const adamw_state *s) {
        return eight ? s->m_root && s->v_root && s->m_scale && s->v_scale && !s->m && !s->v
                     : s->m && s->v && !s->m_root && !s->v_root && !s->m_scale && !s->v_scale;
    };
    if (!whole(to) || (from && !whole(from))) return "a state holds either m and v or all of m_root, v_root, m_scale and v_scale, the same in both";
    if (from && !from->master != !to->master) return "master is in one of state and new_state only";
    const bool master = from && from->master;
    if (!a.weights->diff || (!master && !a.weights->data) || !(a.updated ? a.updated->data : a.weights->data)) return "null buffer";
    if (!(fabsf(a.learning_rate) < __builtin_inff()) || !(fabsf(a.weight_decay) < __builtin_inff())) return "a rate is no finite number";
    return nullptr;
}

// Allocations of the device that a call has met: a program's tensors lie in a few, and to ask the runtime for each of a tensor's ten addresses takes
// longer than the step of a small model (72 tensors: 25 us of asking, 9 of work).  Tensors that lie in more than these are asked for one by one, and
// each time for their allocation too: a call for 72 tensors with four addresses each takes the host 14 us where they lie in one allocation, 53 in 24
// in turn, 57 in one each.
struct AdamMemory {
    struct Range {
        uintptr_t base, end;
    } ranges[8];
    int n = 0;
    bool has(const void *p, size_t bytes) const {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        for (int i = 0; i < n; ++i)
            if (at >= ranges[i].base && at + bytes <= ranges[i].end) return true;
        return false;
    }
    void add(const void *p) {
        hipDeviceptr_t base = nullptr;
        size_t size = 0;
        if (hipMemGetAddressRange(&base, &size, const_cast<void *>(p)) != hipSuccess) {
            (void)hipGetLastError();
            return;
        }
        if (n == 8) {  // the one that came first goes
            for (int i = 1; i < 8; ++i) ranges[i - 1] = ranges[i];
            n = 7;
        }
        ranges[n].base = reinterpret_cast<uintptr_t>(base);
        ranges[n++].end = reinterpret_cast<uintptr_t>(base) + size;
    }
};

template <typename T, typename Args>
static int adamw_multi(const Args *list, int count, const adamw_step *s, const char *fn) {
    if (count <= 0) return 0;
    if (!list || !s) return rows_bad(fn, "null argument structure");
    if (!(s->beta1 >= 0.f && s->beta1 < 1.f && s->beta2 >= 0.f && s->beta2 < 1.f)) return rows_bad(fn, "beta1 or beta2 is not in 0 .. 1");
    if (!(s->eps >= 1e-30f && s->eps < __builtin_inff())) return rows_bad(fn, "eps is no finite number from 1e-30 on");
    if (!s->step_data && s->step < 1) return rows_bad(fn, "steps are counted from 1 on");
    double bytes = 0;
    for (int i = 0; i < count; ++i) {
        if (const char *bad = adamw_check(list[i])) return rows_bad(fn, bad);
        const adamw_state *to = list[i].new_state ? list[i].new_state : list[i].state;
        bytes += (double)list[i].weights->dim * (3 * sizeof(T) + (to->m_root ? 4 : 16) + (to->master ? 8 : 0));
    }
    if (!ensure_init()) return 2;
    Stager sg;
    AdamTable k = {};
    k.b1 = s->beta1;
    k.c1 = (float)(1.0 - (double)s->beta1);
    k.b2 = s->beta2;
    k.c2 = (float)(1.0 - (double)s->beta2);
    k.eps = s->eps;
    k.log1 = (float)log((double)s->beta1);
    k.log2 = (float)log((double)s->beta2);
    if (s->step_data) {
        k.step = sg.in<int>(s->step_data, 1);
    } else {
        k.i1 = (float)(-1.0 / expm1(s->step * log((double)s->beta1)));
        const double i2 = -1.0 / expm1(s->step * log((double)s->beta2));
        k.i2 = (float)i2;
        k.root2 = (float)sqrt(i2);
    }
    if (s->grad_factor) k.factor = sg.in<float>(s->grad_factor, 1);
    AdamMemory known;
    auto map = [&](auto *p, size_t n, bool in, bool out) {
        if (known.has(p, n * sizeof(*p))) return p;
        auto *q = in && out ? sg.inout(p, n) : in ? const_cast<decltype(p)>(sg.in(p, n)) : sg.out(p, n);
        if (q && q == p) known.add(p);
        return q;
    };
    // Every tensor has its place before the first launch: a call that gets no memory for one has changed none.  (What one launch takes lies in its
    // table from the start: 7.3 us for 12 tensors, 7.7 by way of a list.)
    std::unique_ptr<AdamTensor[]> more_than_one;
    if (count > ADAM_TENSORS) {
        more_than_one.reset(new (std::nothrow) AdamTensor[count]);
        if (!more_than_one) {
            set_error("%s: no memory for %d tensors' places", fn, count);
            return 2;
        }
    }
    AdamTensor *const all = more_than_one ? more_than_one.get() : k.t;
    for (int i = 0; i < count; ++i) {
        const Args &a = list[i];
        const size_t n = (size_t)a.weights->dim, blocks = (n + ADAM_BLOCK - 1) / ADAM_BLOCK;
        AdamTensor &t = all[i];
        t = {};
        if (n == 0) continue;
        const adamw_state *from = a.state, *to = a.new_state ? a.new_state : a.state;
        const auto *out = a.updated ? a.updated : a.weights;
        auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
        t.g = map(as(a.weights->diff), n, true, false);
        if (from && from->master) t.master = map(from->master, n, true, false);
        else t.w = map(as(a.weights->data), n, true, false);
        if (t.master && a.weights->data == out->data) t.w = t.w_out = map(as(out->data), n, true, true);  // (left as they are without a step)
        else t.w_out = map(as(out->data), n, false, true);
        if (to->master) t.master_out = map(to->master, n, false, true);
        if (to->m_root) {
            if (from) {
                t.m = map(from->m_root, n, true, false);
                t.v = map(from->v_root, n, true, false);
                t.m_scale = map(from->m_scale, blocks, true, false);
                t.v_scale = map(from->v_scale, blocks, true, false);
            }
            t.m_out = map(to->m_root, n, false, true);
            t.v_out = map(to->v_root, n, false, true);
            t.m_scale_out = map(to->m_scale, blocks, false, true);
            t.v_scale_out = map(to->v_scale, blocks, false, true);
        } else {
            if (from) {
                t.m = map(from->m, n, true, false);
                t.v = map(from->v, n, true, false);
            }
            t.m_out = map(to->m, n, false, true);
            t.v_out = map(to->v, n, false, true);
        }
        t.n = (unsigned)n;
        t.lr = a.learning_rate;
        t.decay = a.weight_decay;
    }
    if (sg.failed()) return 2;
    // More than the 256 MB of the memory's cache: past it, one block a wave (23 million fp32 weights 110 us, 116 with two, 126 with four, and
    // 119 with one through the caches); less: two, through them (1 million 7.3 us; one 7.9; past them 8.8).
    const bool large = bytes > 256e6;
    const int group = 4 * ADAM_BLOCK * (large ? 1 : 2);  // elements of a workgroup
    unsigned groups = 0;
    auto flush = [&]() {
        for (int i = k.count; i < ADAM_TENSORS; ++i) k.first[i] = 0xffffffffu;
        if (k.count > 0) {
            if (large) hipLaunchKernelGGL((adamw_kernel<T, 1, true>), dim3(groups), dim3(256), 0, state().stream, k);
            else hipLaunchKernelGGL((adamw_kernel<T, 2, false>), dim3(groups), dim3(256), 0, state().stream, k);
        }
        k.count = 0;
        groups = 0;
        return hip_ok(hipGetLastError(), "optimizer launch");
    };
    for (int i = 0; i < count; ++i) {
        if (all[i].n == 0) continue;
        const size_t more = ((size_t)all[i].n + group - 1) / group;
        if ((k.count == ADAM_TENSORS || (groups + more) * 256 > (size_t)ROW_THREADS) && !flush()) return sg.finish(2);
        k.t[k.count] = all[i];  // (k.count is at most i)
        k.first[k.count] = groups;
        groups += (unsigned)more;
        ++k.count;
    }
    return sg.finish(flush() ? 0 : 2);
}

}  // namespace ptl

extern "C" {
int ptl_adamw_fp32_multi(const struct adamw_args *list, int count, const struct adamw_step *step) {
    return ptl::adamw_multi<float>(list, count, step, "ptl_adamw_fp32_multi");
}
int ptl_adamw_fp16_multi(const struct adamw_args_fp16 *list, int count, const struct adamw_step *step) {
    return ptl::adamw_multi<ptl::half_t>(list, count, step, "ptl_adamw_fp16_multi");
}
}
