// Both products behind the gradients dh of a gated layer's pre-activations, in one launch: dx = dh W (k: the 2 n_out rows of W) and
// dW = dh^T x (k: the tokens), fp16.
// W and x are contiguous along the inputs, which are not k: their tiles lie in LDS as they come, [k][row], and the fragments, eight k
// of one row, are read with the transposing reads.  Of dh, the second operand, dx takes rows of k and dW again [k][row].
//   * A [k][row] tile has 256 bytes of a k side by side.  A fragment's reads touch eight k at the same 64 of them, a quarter of the
//     banks: the 64-byte blocks of row k are therefore exchanged by k % 4 (on the way in, where a lane chooses which piece it loads).
//   * Tiles of 128 x 128 with two workgroups a compute unit, one of which stores or waits while the other multiplies.  The two
//     products' tiles differ in length (2 n_out against the number of tokens): the longer ones come first in the grid and the
//     shorter ones fill up behind them.
//   * Where that leaves compute units idle k is cut into parts, each with sums of its own in fp32, which another launch adds up.
// 2048 tokens, 2048 -> 5632: 210 us (900 TFLOP/s; with the gradients of the pre-activations 231), as a dense layer's call 245;
// 256 tokens of the same layer 58 and 82, 64 tokens 31 and 49.
// Rows that are no whole 16-byte pieces come as copies (rows_copy(), gate_back_kernel): 2047 -> 5631 252 us with them.
// Tried: slabs of 32 k, four of them in flight, instead of two of 64: 3 to 8 % longer.
#include "ptl_rows_mm.inc"

namespace ptl {

template <typename OUT>
struct GradTile {
    typedef OUT Out;
    typedef f32x16 Acc;
    static constexpr bool GATE = false;
    static constexpr int ROWS_W = 128, ROWS_X = 128, WM = 64, WN = 64, FM = 2, FN = 2, OC = 64, PITCH = OC * (int)sizeof(OUT) + 16, GROUPS = 1;
    static constexpr int NT = 256, TILE = 128 * ROWB, STAGE = 2 * TILE, RING = 2 * STAGE, TABLE = (2 * ROWS_W + ROWS_X) * 4;
    static_assert(TABLE + 4 * 32 * PITCH <= RING, "what follows the sums fits the ring");
};

struct GradProd {
    RowsArgs out;       // y, outs (the inputs), tokens (rows of the second operand), tiles; no scales and biases
    const char *f, *s;  // first operand: k rows of outs values; second one: its rows of k values, or k rows of them
    int k, f_b, s_b;    // k, bytes of a row of either
    int f_n, s_n;       // rows that have values of their own in [k][row] tiles: whole eights
    int parts, chunk;   // k in parts of so many slabs, each with its own sums in fp32 (part) where there are more than one
    float *part;
};
struct GradArgs {
    GradProd p[2];  // dx, dW
    int first, lead;  // workgroups of the product that comes first, and which one that is
};

// 16 bytes (eight k of row `row` of a 32-row fragment) from a [k][row] tile; chunk: k / 8.
__device__ inline uint4 grad_frag(const char *tile, int block, int lane, int chunk) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const int i = lane & 15;
    const char *p = tile + (chunk * 8 + (i >> 2)) * 256 + ((block ^ (i >> 2)) << 6) + ((lane & 16) << 1) + (i & 3) * 8;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(lds_char *)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(lds_char *)(p + 4 * 256));
    union {
        s4 h[2];
        uint4 v;
    } t;
    t.h[0] = lo;
    t.h[1] = hi;
    return t.v;
}

// Floats between the sums of two parts: whole fours.
__host__ __device__ inline size_t grad_part(int tokens, int outs) { return ((size_t)tokens * outs + 3) & ~(size_t)3; }

// ROWS: the second operand has k along its rows.
template <bool ROWS>
__device__ inline void grad_tile(const GradProd &g, int id, char *smem) {
    typedef GradTile<half_t> C;
    typedef GradTile<float> P;
    constexpr int NT = C::NT;
    const RowsArgs &a = g.out;
    const int tiles = a.tiles_w * a.tiles_t, z = id / tiles, k0 = z * g.chunk * 64, k_n = min(g.k - k0, g.chunk * 64);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave & 1, ww = wave >> 1;
    int tw, tt;
    rows_place(a, id - z * tiles, tw, tt);
    const int o0 = tw * 128, t0 = tt * 128, slabs = (k_n + 63) / 64, tail = k_n - (slabs - 1) * 64;
    const unsigned ring = (unsigned)(uintptr_t)(lds_char *)smem;
    const char *f_ptr = g.f + (long long)o0 * 2 + (long long)k0 * g.f_b;
    const char *s_ptr = ROWS ? g.s + (long long)t0 * g.s_b + (long long)k0 * 2 : g.s + (long long)t0 * 2 + (long long)k0 * g.s_b;
    const long long f_step = 64ll * g.f_b, s_step = ROWS ? ROWB : 64ll * g.s_b;
    // piece of a [k][row] tile that lies at place q: its k, and its rows as a multiple of eight behind the tile's first; rows beyond
    // the end repeat the last ones
    const int kk = tid >> 4, at = (tid & 15) ^ ((kk & 3) << 2);
    unsigned f_off[4], s_off[4];
    bool f_none[4], s_none[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = kk + j * 16;
        f_off[j] = (unsigned)k * (unsigned)g.f_b + (unsigned)min(at, (g.f_n - o0) / 8 - 1) * 16u;
        f_none[j] = k >= tail;
        if constexpr (ROWS) {
            const int r = (j * NT + tid) >> 3, pos = (tid & 7) ^ swz(r);
            s_off[j] = (unsigned)min(r, a.tokens - 1 - t0) * (unsigned)g.s_b + (unsigned)pos * 16u;
            s_none[j] = pos * 8 >= tail;
        } else {
            s_off[j] = (unsigned)k * (unsigned)g.s_b + (unsigned)min(at, (g.s_n - t0) / 8 - 1) * 16u;
            s_none[j] = k >= tail;
        }
    }
    int left = slabs;
    auto issue = [&](unsigned stage) {
        const unsigned to = ring + stage + (unsigned)wave * 1024u;
        if (--left > 0 || tail == 64) {
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma16_saddr(f_off[j], f_ptr, to + j * 4096u);
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma16_saddr(s_off[j], s_ptr, to + C::TILE + j * 4096u);
        } else {  // k that the last slab does not have
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma<16>(f_none[j] ? a.zeros : f_ptr + f_off[j], to + j * 4096u);
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma<16>(s_none[j] ? a.zeros : s_ptr + s_off[j], to + C::TILE + j * 4096u);
        }
        f_ptr += f_step;
        s_ptr += s_step;
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    const int kg = lane >> 5, lr = lane & 31;
    auto compute = [&](unsigned stage) {
        const char *tf = smem + stage, *ts = tf + C::TILE;
        uint4 ff[2][2], sf[2][2];
        auto load = [&](int ks, int set) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ff[set][i] = grad_frag(tf, ww * 2 + i, lane, 2 * ks + kg);
                sf[set][i] = ROWS ? read_frag<half_t, 128, FILL_VEC_K>(ts, wt * 64 + i * 32 + lr, ks, kg) : grad_frag(ts, wt * 2 + i, lane, 2 * ks + kg);
            }
        };
        load(0, 0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t < 3) load(t + 1, (t + 1) & 1);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) mfma_step<half_t>(acc[i][j], ff[t & 1][i], sf[t & 1][j]);
        }
    };
    issue(0);
    unsigned out = 0;
    for (int s = 0; s < slabs; ++s) {
        wait_vmcnt<0>();
        __syncthreads();
        if (s + 1 < slabs) issue(C::STAGE - out);
        compute(out);
        out = C::STAGE - out;
    }
    __syncthreads();
    float *w_tab = reinterpret_cast<float *>(smem), *b_tab = w_tab + C::ROWS_W, *x_tab = b_tab + C::ROWS_W;
    rows_tables<C>(a, o0, t0, w_tab, b_tab, x_tab, tid, NT);
    __syncthreads();
    if (g.parts > 1) {
        RowsArgs p = a;
        p.y = g.part + (size_t)z * grad_part(a.tokens, a.outs);
        rows_behind<P>(p, acc, o0, t0, ww, wt, lane, w_tab, b_tab, x_tab, smem + P::TABLE + wave * 32 * P::PITCH);
    } else {
        rows_behind<C>(a, acc, o0, t0, ww, wt, lane, w_tab, b_tab, x_tab, smem + C::TABLE + wave * 32 * C::PITCH);
    }
}

__global__ __launch_bounds__(GradTile<half_t>::NT) void grad_kernel(const GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int second = (int)blockIdx.x >= a.first, id = second ? (int)blockIdx.x - a.first : (int)blockIdx.x;
    if ((second ^ a.lead) == 0) grad_tile<true>(a.p[0], id, smem);
    else grad_tile<false>(a.p[1], id, smem);
}

// The parts' sums, in their order, rounded once: four values a thread.
struct GradJoin {
    const float *part[2];
    half_t *y[2];
    size_t n[2], values[2];  // fours of values (0: not in parts), values
    int parts[2];
};
__global__ __launch_bounds__(256) void grad_join_kernel(const GradJoin a) {
    size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int o = i >= a.n[0];
    if (o) i -= a.n[0];
    if (i >= a.n[o]) return;
    const float4 *p = reinterpret_cast<const float4 *>(a.part[o]) + i;
    float4 s = p[0];
    for (int k = 1; k < a.parts[o]; ++k) {
        const float4 v = p[(size_t)k * a.n[o]];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    typedef half_t h4 __attribute__((ext_vector_type(4)));
    const h4 v = h4{(half_t)s.x, (half_t)s.y, (half_t)s.z, (half_t)s.w};
    if (4 * i + 4 <= a.values[o]) {
        reinterpret_cast<h4 *>(a.y[o])[i] = v;
    } else {
        for (int e = 0; 4 * i + e < a.values[o]; ++e) a.y[o][4 * i + e] = v[e];
    }
}

// Microseconds of the launch with k of the two products in so many parts: a workgroup takes 0.95 a slab while it shares its compute
// unit with another, 0.7 alone, and 4 for the rest; what remains behind the long ones is half of a short one in the mean.  Parts cost
// their sums, written and read at 5 TB/s, and a launch.
static float grad_cost(const int (&tiles)[2], const int (&slabs)[2], const double (&mb)[2], const int (&parts)[2]) {
    const int cu = state().num_cu;
    float work = 0, longest = 0, shortest = 1e9f, extra = 0;
    long groups = 0;
    for (int i = 0; i < 2; ++i) groups += (long)tiles[i] * parts[i];
    const float slab = groups > cu ? 0.95f : 0.7f;
    for (int i = 0; i < 2; ++i) {
        if (!tiles[i]) continue;
        const int chunk = (slabs[i] + parts[i] - 1) / parts[i];
        const float one = chunk * slab + 4.f;
        work += one * tiles[i] * parts[i];
        longest = one > longest ? one : longest;
        shortest = one < shortest ? one : shortest;
        if (parts[i] > 1) extra += (float)(mb[i] * 8e-6 * parts[i] / 5.0);
    }
    const float spread = work / (2 * cu) + 0.5f * shortest;
    return (spread > longest ? spread : longest) + (extra > 0 ? extra + 4.f : 0.f);
}

int gated_products(const half_t *x, const half_t *w, const half_t *dh, half_t *dw, half_t *dx, int ns, int in, int rows, int cols, int pitch) {
    static bool ready = false;
    constexpr int RING = GradTile<half_t>::RING;
    if (!ready) {
        if (!hip_ok(hipFuncSetAttribute(reinterpret_cast<const void *>(grad_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, RING), "hipFuncSetAttribute"))
            return 2;
        ready = true;
    }
    GradArgs a = {};
    half_t *y[2] = {dx, dw};
    const int n[2] = {ns, rows}, k[2] = {rows, ns};
    int tiles[2], slabs[2], parts[2] = {1, 1};
    double values[2];
    for (int i = 0; i < 2; ++i) {
        tiles[i] = y[i] ? (in + 127) / 128 * ((n[i] + 127) / 128) : 0;
        slabs[i] = (k[i] + 63) / 64;
        values[i] = (double)n[i] * in;
    }
    float best = 1e30f;
    for (int u = 1; u <= 32 && (u == 1 || (tiles[0] && u * 4 <= slabs[0])); u *= 2)
        for (int v = 1; v <= 32 && (v == 1 || (tiles[1] && v * 4 <= slabs[1])); v *= 2) {
            const int p[2] = {u, v};
            const float c = grad_cost(tiles, slabs, values, p);
            if (c < best) {
                best = c;
                parts[0] = u;
                parts[1] = v;
            }
        }
    GradJoin j = {};
    size_t floats = 0;
    for (int i = 0; i < 2; ++i) {
        GradProd &p = a.p[i];
        p.out.y = y[i];
        p.out.outs = in;
        p.out.tokens = n[i];
        p.out.zeros = static_cast<const char *>(state().zeros);
        p.out.tiles_w = (in + 127) / 128;
        p.out.tiles_t = (n[i] + 127) / 128;
        p.f = reinterpret_cast<const char *>(i ? x : w);
        p.s = reinterpret_cast<const char *>(dh);
        p.k = k[i];
        p.f_b = cols * 2;
        p.s_b = pitch * 2;
        p.f_n = cols;
        p.s_n = pitch;
        p.chunk = (slabs[i] + parts[i] - 1) / parts[i];
        p.parts = (slabs[i] + p.chunk - 1) / p.chunk;
        if (p.parts > 1) floats += (size_t)p.parts * grad_part(n[i], in);
    }
    if (floats) {
        float *ws = workspace(floats * sizeof(float));
        if (!ws) return 2;
        for (int i = 0; i < 2; ++i) {
            if (a.p[i].parts == 1) continue;
            a.p[i].part = ws;
            j.part[i] = ws;
            j.y[i] = y[i];
            j.values[i] = (size_t)n[i] * in;
            j.n[i] = grad_part(n[i], in) / 4;
            j.parts[i] = a.p[i].parts;
            ws += (size_t)a.p[i].parts * grad_part(n[i], in);
        }
    }
    a.lead = a.p[0].chunk >= a.p[1].chunk ? 0 : 1;
    const int groups[2] = {tiles[0] * a.p[0].parts, tiles[1] * a.p[1].parts};
    a.first = groups[a.lead];
    hipLaunchKernelGGL(grad_kernel, dim3(groups[0] + groups[1]), dim3(GradTile<half_t>::NT), RING, state().stream, a);
    if (floats) {
        const size_t fours = j.n[0] + j.n[1];
        hipLaunchKernelGGL(grad_join_kernel, dim3((unsigned)((fours + 255) / 256)), dim3(256), 0, state().stream, j);
    }
    return hip_ok(hipGetLastError(), "gated layer launch") ? 0 : 2;
}

void rows_copy(const void *w, size_t n_w, const void *x, size_t n_x, void *to, int bytes, int pitch) {
    rows_copies(static_cast<const char *>(w), n_w, static_cast<const char *>(x), n_x, static_cast<char *>(to), bytes, pitch);
}

}  // namespace ptl
