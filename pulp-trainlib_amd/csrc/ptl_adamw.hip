// A step of AdamW over many tensors at once, with moments in 32 or in 8 bits.
//   g = diff * factor;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   w = w - lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay w)
// Bound by memory: 28 bytes an element with fp32 weights and moments, 16 with moments in 8 bits, and some forty operations on them.
// A wave has 256 elements at a time, four neighbours a lane: they are what shares a scale in 8 bits, so that its largest
// root is found without a barrier.  The tensors' places travel in the kernel's arguments, 32 tensors a launch: no table in memory has to
// be written, and the launches can be captured.
// In 8 bits the roots are held, not the moments: a block's moments span decades (v the squares of m's), and the fourth root brings
// the 65025^2 that v spans between its smallest code and its largest to 255.
#include "ptl_rows.hpp"
#include "ptl_tuning.h"

namespace ptl {

constexpr int ADAM_BLOCK = 256;   // elements of a scale
constexpr int ADAM_UNROLL = 4;    // blocks of a wave
constexpr int ADAM_GROUP = 4 * ADAM_UNROLL * ADAM_BLOCK;  // elements of a workgroup
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
    unsigned n, first;        // elements; first workgroup
};
struct AdamTable {
    AdamTensor t[ADAM_TENSORS];
    int count;
    float b1, c1, b2, c2, eps;     // c1 = 1 - b1, c2 = 1 - b2
    float i1, i2;                  // 1 / (1 - b1^t), 1 / (1 - b2^t)
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

// Four neighbouring values, of which `left` exist (4 and more: all).
template <typename S>
struct Adam4 {
    union {
        typename AdamRaw<sizeof(S)>::type raw;
        S e[4];
    };
    __device__ inline void load(const S *p, size_t at, long left) {
        if (left >= 4) {
            raw = *reinterpret_cast<const typename AdamRaw<sizeof(S)>::type *>(p + at);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = i < left ? p[at + i] : (S)0;
        }
    }
    __device__ inline void store(S *p, size_t at, long left) const {
        if (left >= 4) {
            *reinterpret_cast<typename AdamRaw<sizeof(S)>::type *>(p + at) = raw;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) p[at + i] = e[i];
        }
    }
};

// The root to one step of fp32.  The instruction takes subnormal values for 0, so small ones are worked on 2^64 times as large.
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
    float b1, c1, b2, c2, eps, i1, i2, factor, lr, decay;
    // One element: the moments and the weight behind the step.
    __device__ inline void step(float g, float &m, float &v, float &w) const {
        g *= factor;
        m = fmaf(b1, m, c1 * g);
        v = fmaf(b2, v, c2 * g * g);
        const float root = adam_root(v * i2) + eps;
        w = fmaf(-lr, fmaf(decay, w, m * i1 * __builtin_amdgcn_rcpf(root)), w);
    }
};

// Four weights behind the step, in both forms.
template <typename T>
__device__ inline void adam_put(const AdamTensor &t, const float (&w)[4], size_t at, long left) {
    Adam4<T> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.e[i] = row_round<T>(w[i]);
    o.store(static_cast<T *>(t.w_out), at, left);
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

// The codes of four roots (127 or 255: the largest), and the wave's scale of them.
template <int MOST>
__device__ inline void adam_codes(const float (&root)[4], const float (&of)[4], int (&code)[4], float &scale) {
    const float most = wave_nan_max(nan_max(nan_max(root[0], root[1]), nan_max(root[2], root[3])));
    const float unit = most > 0.f ? (float)MOST / most : 0.f;
    scale = most / (float)MOST;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = (int)fminf(rintf(root[i] * unit), (float)MOST);
        code[i] = MOST == 255 && of[i] != 0.f && c == 0 ? 1 : c;
    }
}

// A step that changes nothing: what is not updated in place is copied.
template <typename T>
__device__ inline void adam_copy(const AdamTensor &t, size_t at, long left, size_t block, int lane) {
    if (t.w != t.w_out || t.master) {
        AdamPart<T> p;
        float w[4];
        if (t.master) p.master.load(t.master, at, left);
        else p.w.load(static_cast<const T *>(t.w), at, left);
        adam_weights<T>(t, p, w);
        AdamTensor o = t;
        if (t.master_out == t.master) o.master_out = nullptr;
        if (!t.master || t.w != t.w_out) adam_put<T>(o, w, at, left);
        else if (o.master_out) p.master.store(o.master_out, at, left);
    } else if (t.master_out) {  // (the weights in fp32 begin here)
        AdamPart<T> p;
        Adam4<float> f;
        p.w.load(static_cast<const T *>(t.w), at, left);
#pragma unroll
        for (int i = 0; i < 4; ++i) f.e[i] = (float)p.w.e[i];
        f.store(t.master_out, at, left);
    }
    if (t.m_out == t.m) return;
    if (t.m_scale_out) {
        Adam4<int8_t> c = {};
        if (t.m) c.load(static_cast<const int8_t *>(t.m), at, left);
        c.store(static_cast<int8_t *>(t.m_out), at, left);
        if (t.m) c.load(static_cast<const int8_t *>(t.v), at, left);
        c.store(static_cast<int8_t *>(t.v_out), at, left);
        if (lane == 0) {
            t.m_scale_out[block] = t.m ? t.m_scale[block] : 0.f;
            t.v_scale_out[block] = t.m ? t.v_scale[block] : 0.f;
        }
    } else {
        Adam4<float> f = {};
        if (t.m) f.load(static_cast<const float *>(t.m), at, left);
        f.store(static_cast<float *>(t.m_out), at, left);
        if (t.m) f.load(static_cast<const float *>(t.v), at, left);
        f.store(static_cast<float *>(t.v_out), at, left);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamTable a) {
    int k = 0;
#pragma unroll
    for (int half = ADAM_TENSORS / 2; half >= 1; half /= 2)
        if (k + half < a.count && blockIdx.x >= a.t[k + half].first) k += half;
    const AdamTensor &t = a.t[k];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (a workgroup's blocks lie side by side: wave w has blocks w, w + 4, ...)
    const size_t first = (size_t)(blockIdx.x - t.first) * (ADAM_GROUP / ADAM_BLOCK) + wave;
    auto place = [&](int u) { return (first + 4 * u) * ADAM_BLOCK + 4 * (size_t)lane; };
    auto left = [&](int u) { return (long)t.n - (long)place(u); };
    auto none = [&](int u) { return (first + 4 * u) * ADAM_BLOCK >= t.n; };  // (of the whole wave)
    AdamPart<T> p[ADAM_UNROLL];
#pragma unroll
    for (int u = 0; u < ADAM_UNROLL; ++u) {
        if (none(u)) break;
        p[u].g.load(static_cast<const T *>(t.g), place(u), left(u));
        if (t.master) p[u].master.load(t.master, place(u), left(u));
        else p[u].w.load(static_cast<const T *>(t.w), place(u), left(u));
    }
    AdamRates r = {a.b1, a.c1, a.b2, a.c2, a.eps, a.i1, a.i2, a.factor ? *a.factor : 1.f, t.lr, t.decay};
    if (!(fabsf(r.factor) < __builtin_inff())) {
#pragma unroll 1
        for (int u = 0; u < ADAM_UNROLL; ++u)
            if (!none(u)) adam_copy<T>(t, place(u), left(u), first + 4 * u, lane);
        return;
    }
    if (a.step) {
        const float s = (float)*a.step;
        r.i1 = -1.f / expm1f(s * a.log1);
        r.i2 = -1.f / expm1f(s * a.log2);
    }
    if (t.m_scale_out) {
        Adam4<int8_t> mq[ADAM_UNROLL], vq[ADAM_UNROLL];
        float ms[ADAM_UNROLL], vs[ADAM_UNROLL];
#pragma unroll
        for (int u = 0; u < ADAM_UNROLL; ++u) {
            if (none(u)) break;
            ms[u] = vs[u] = 0.f;
            mq[u].raw = vq[u].raw = 0;
            if (!t.m) continue;
            mq[u].load(static_cast<const int8_t *>(t.m), place(u), left(u));
            vq[u].load(static_cast<const int8_t *>(t.v), place(u), left(u));
            ms[u] = t.m_scale[first + 4 * u];
            vs[u] = t.v_scale[first + 4 * u];
        }
#pragma unroll
        for (int u = 0; u < ADAM_UNROLL; ++u) {
            if (none(u)) break;
            float w[4], m[4], v[4], mr[4], vr[4];
            adam_weights<T>(t, p[u], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = (float)mq[u].e[i] * ms[u], c = (float)(uint8_t)vq[u].e[i] * vs[u];
                m[i] = q * fabsf(q);
                v[i] = c * c * (c * c);
                r.step((float)p[u].g.e[i], m[i], v[i], w[i]);
                mr[i] = adam_root(fabsf(m[i]));
                vr[i] = adam_root(adam_root(v[i]));
            }
            int mc[4], vc[4];
            float scale[2];
            adam_codes<127>(mr, m, mc, scale[0]);
            adam_codes<255>(vr, v, vc, scale[1]);
            Adam4<int8_t> mo, vo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mo.e[i] = (int8_t)(m[i] < 0.f ? -mc[i] : mc[i]);
                vo.e[i] = (int8_t)vc[i];
            }
            adam_put<T>(t, w, place(u), left(u));
            mo.store(static_cast<int8_t *>(t.m_out), place(u), left(u));
            vo.store(static_cast<int8_t *>(t.v_out), place(u), left(u));
            if (lane == 0) {
                t.m_scale_out[first + 4 * u] = scale[0];
                t.v_scale_out[first + 4 * u] = scale[1];
            }
        }
    } else {
        Adam4<float> mv[ADAM_UNROLL], vv[ADAM_UNROLL];
#pragma unroll
        for (int u = 0; u < ADAM_UNROLL; ++u) {
            if (none(u)) break;
            mv[u].raw = vv[u].raw = adam_u4{0, 0, 0, 0};
            if (!t.m) continue;
            mv[u].load(static_cast<const float *>(t.m), place(u), left(u));
            vv[u].load(static_cast<const float *>(t.v), place(u), left(u));
        }
#pragma unroll
        for (int u = 0; u < ADAM_UNROLL; ++u) {
            if (none(u)) break;
            float w[4];
            adam_weights<T>(t, p[u], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) r.step((float)p[u].g.e[i], mv[u].e[i], vv[u].e[i], w[i]);
            adam_put<T>(t, w, place(u), left(u));
            mv[u].store(static_cast<float *>(t.m_out), place(u), left(u));
            vv[u].store(static_cast<float *>(t.v_out), place(u), left(u));
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

template <typename T, typename Args>
static int adamw_multi(const Args *list, int count, const adamw_step *s, const char *fn) {
    if (count <= 0) return 0;
    if (!list || !s) return rows_bad(fn, "null argument structure");
    if (!(s->beta1 >= 0.f && s->beta1 < 1.f && s->beta2 >= 0.f && s->beta2 < 1.f)) return rows_bad(fn, "beta1 or beta2 is not in 0 .. 1");
    if (!(s->eps >= 1e-30f && s->eps < __builtin_inff())) return rows_bad(fn, "eps is no finite number from 1e-30 on");
    if (!s->step_data && s->step < 1) return rows_bad(fn, "steps are counted from 1 on");
    for (int i = 0; i < count; ++i)
        if (const char *bad = adamw_check(list[i])) return rows_bad(fn, bad);
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
        k.i2 = (float)(-1.0 / expm1(s->step * log((double)s->beta2)));
    }
    if (s->grad_factor) k.factor = sg.in<float>(s->grad_factor, 1);
    unsigned groups = 0;
    auto flush = [&]() {
        if (k.count > 0) hipLaunchKernelGGL((adamw_kernel<T>), dim3(groups), dim3(256), 0, state().stream, k);
        k.count = 0;
        groups = 0;
        return hip_ok(hipGetLastError(), "optimizer launch");
    };
    for (int i = 0; i < count; ++i) {
        const Args &a = list[i];
        const size_t n = (size_t)a.weights->dim, blocks = (n + ADAM_BLOCK - 1) / ADAM_BLOCK;
        if (n == 0) continue;
        const adamw_state *from = a.state, *to = a.new_state ? a.new_state : a.state;
        const auto *out = a.updated ? a.updated : a.weights;
        if (k.count == ADAM_TENSORS && !flush()) return sg.finish(2);
        AdamTensor &t = k.t[k.count];
        t = {};
        t.g = sg.in(reinterpret_cast<const T *>(a.weights->diff), n);
        if (from && from->master) t.master = sg.in<float>(from->master, n);
        else t.w = sg.in(reinterpret_cast<const T *>(a.weights->data), n);
        if (t.master && a.weights->data == out->data) t.w = t.w_out = sg.inout(reinterpret_cast<T *>(out->data), n);  // (left as they are without a step)
        else t.w_out = sg.out(reinterpret_cast<T *>(out->data), n);
        if (to->master) t.master_out = sg.out<float>(to->master, n);
        if (to->m_root) {
            if (from) {
                t.m = sg.in<int8_t>(from->m_root, n);
                t.v = sg.in<uint8_t>(from->v_root, n);
                t.m_scale = sg.in<float>(from->m_scale, blocks);
                t.v_scale = sg.in<float>(from->v_scale, blocks);
            }
            t.m_out = sg.out<int8_t>(to->m_root, n);
            t.v_out = sg.out<uint8_t>(to->v_root, n);
            t.m_scale_out = sg.out<float>(to->m_scale, blocks);
            t.v_scale_out = sg.out<float>(to->v_scale, blocks);
        } else {
            if (from) {
                t.m = sg.in<float>(from->m, n);
                t.v = sg.in<float>(from->v, n);
            }
            t.m_out = sg.out<float>(to->m, n);
            t.v_out = sg.out<float>(to->v, n);
        }
        if (sg.failed()) return 2;
        t.n = (unsigned)n;
        t.lr = a.learning_rate;
        t.decay = a.weight_decay;
        t.first = groups;
        groups += (unsigned)((n + ADAM_GROUP - 1) / ADAM_GROUP);
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
