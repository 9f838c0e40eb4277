// Both products behind the gradients dh of a gated layer's pre-activations, in one launch: dx = dh W (k: the 2 n_out rows of W) and
// dW = dh^T x (k: the tokens).
// W and x are contiguous along the inputs, which are not k: their tiles lie in LDS as they come, [k][row].  Of dh, the second operand, dx
// takes rows of k and dW again [k][row].
//   * fp16: fragments, eight k of one row, are read from [k][row] tiles with the transposing reads.  A tile has 256 bytes of a k side by
//     side; a fragment's reads touch eight k at the same 64 of them, a quarter of the banks: the 64-byte blocks of row k are therefore
//     exchanged by k % 4 (on the way in, where a lane chooses which piece it loads).  fp32: a value is a dword, and a fragment four reads
//     of 32 neighbours each.
//   * fp16: large layers take tiles of 256 x 128 and three slabs, one workgroup a compute unit: a fragment's way out of LDS costs half of what
//     the matrix instructions take, and what comes in on top a third less than with 128 x 128.  Smaller ones those, with two workgroups a
//     compute unit, one of which stores or waits while the other multiplies.  fp32: 128 x 64,
//     three (its instructions take sixteen times as long: smaller tiles cost nothing and leave less of the chip idle; 128 x 128 were 5 to 30 %
//     slower).  The two products' tiles differ in length (2 n_out against the number of tokens): the longer ones come first in the grid and the
//     shorter ones fill up behind them.
//   * Where that leaves compute units idle k is cut into parts, each with sums of its own in fp32, which another launch adds up.
// fp16, 2048 tokens, 2048 -> 5632: 185 us (1020 TFLOP/s; with the gradients of the pre-activations 210), as a dense layer's call 245;
// 256 tokens of the same layer 58 and 82, 64 tokens 31 and 49.  fp32, 2048 tokens, 1024 -> 2816: 391 us (121 TFLOP/s) and 461.
// Rows that are no whole 16-byte pieces come as copies (rows_copy(), gate_back_kernel): fp16, 2047 -> 5631 252 us with them.
// fp16: loads, fragments and matrix instructions follow each other one by one, a slab's last step behind its barrier (gated 229 -> 225 us).
// Tried: slabs of 32 k, four of them in flight, instead of two of 64: 3 to 8 % longer.
#include "ptl_rows_mm.inc"

namespace ptl {

template <typename OUT, int XR, int FW>  // tiles of FW inputs by XR rows of the other operand
struct GradTile {
    typedef OUT Out;
    typedef f32x16 Acc;
    static constexpr RowsAfter AFTER_SUMS = ROWS_SCALED;
    static constexpr bool GATED = false;
    static constexpr int ROWS_W = FW, ROWS_X = XR, WM = 64, WN = XR / 2, FM = 2, FN = XR / 64, OC = 64, PITCH = OC * (int)sizeof(OUT) + 16, GROUPS = 1;
    static constexpr int NT = 2 * FW, NS = FW == 256 ? 3 : 2, HALF = 128 * ROWB, TILE = FW * ROWB, STAGE = TILE + XR * ROWB, RING = NS * STAGE;
    static constexpr int TABLE = (2 * ROWS_W + ROWS_X) * 4;
    static_assert(TABLE + FW / 32 * 32 * PITCH <= RING, "what follows the sums fits the ring");
};

struct GradProd {
    RowsArgs out;       // y, outs (the inputs), tokens (rows of the second operand), tiles; no scales and biases
    const char *f, *s;  // first operand: k rows of outs values; second one: its rows of k values, or k rows of them
    int k, f_b, s_b;    // k, bytes of a row of either
    int f_n, s_n;       // rows that have values of their own in [k][row] tiles: whole eights
    int parts, chunk;   // k in parts of so many slabs, each with its own sums in fp32 (part) where there are more than one
    int high;           // parts of s; the others, the same k again, are of `low`
    const char *low;
    float *part;
};
struct GradArgs {
    GradProd p[2];  // dx, dW
    int first, lead;  // workgroups of the product that comes first, and which one that is
    int tiles;        // ... of both; behind them: of db
    const float *shares;
    void *db;
    int rows, n_shares;
};

// 16 bytes of a row (eight k; fp32: four) of a 32-row fragment from a [k][row] tile; chunk: k / 8, k / 4.
template <typename T, int XR>
__device__ inline uint4 grad_frag(const char *tile, int block, int lane, int chunk) {
    if constexpr (sizeof(T) == 4) {
        const unsigned *q = reinterpret_cast<const unsigned *>(tile) + chunk * 4 * XR + block * 32 + (lane & 31);
        return make_uint4(q[0], q[XR], q[2 * XR], q[3 * XR]);
    }
    static_assert(sizeof(T) == 4 || XR == 128, "blocks are exchanged over 256 bytes");
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
template <typename T, int XR, int FW, bool ROWS>
__device__ inline void grad_tile(const GradProd &g, int id, char *smem) {
    typedef GradTile<T, XR, FW> C;
    typedef GradTile<float, XR, FW> P;
    constexpr int NT = C::NT, ES = (int)sizeof(T), VEC = 16 / ES, KS = ROWB / ES;  // k of a slab
    constexpr int PER = 128 / VEC, XPER = XR / VEC, LX = XR * 8 / NT, FN = C::FN;      // pieces of a k's rows, loads of a thread for the second tile
    const RowsArgs &a = g.out;
    const int tiles = a.tiles_w * a.tiles_t, z = id / tiles, k0 = (z < g.high ? z : z - g.high) * g.chunk * KS, k_n = min(g.k - k0, g.chunk * KS);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave & 1, ww = wave >> 1;
    int tw, tt;
    rows_place(a, id - z * tiles, tw, tt);
    const int o0 = tw * FW, t0 = tt * XR, slabs = (k_n + KS - 1) / KS, tail = k_n - (slabs - 1) * KS;
    const unsigned ring = (unsigned)(uintptr_t)(lds_char *)smem;
    const char *f_ptr = g.f + (long long)o0 * ES + (long long)k0 * g.f_b;
    const char *s_ptr = (z < g.high ? g.s : g.low) + (ROWS ? (long long)t0 * g.s_b + (long long)k0 * ES : (long long)t0 * ES + (long long)k0 * g.s_b);
    const long long f_step = (long long)KS * g.f_b, s_step = ROWS ? ROWB : (long long)KS * g.s_b;
    // piece of a [k][row] tile that lies at place q: its k, and its rows as a multiple of VEC behind the tile's first; rows beyond
    // the end repeat the last ones
    auto place = [&](int q, int per) { return ES == 2 ? q % per ^ ((q / per & 3) << 2) : q % per; };
    unsigned f_off[4], s_off[LX];
    bool f_none[4], s_none[LX];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        constexpr int HALF = C::HALF / 16;  // (a wide tile is two narrow ones, one behind the other)
        const int q = (j * NT + tid) % HALF, k = q / PER;
        f_off[j] = (unsigned)k * (unsigned)g.f_b + (unsigned)min(place(q, PER) + (j * NT + tid) / HALF * PER, (g.f_n - o0) / VEC - 1) * 16u;
        f_none[j] = k >= tail;
    }
#pragma unroll
    for (int j = 0; j < LX; ++j) {
        if constexpr (ROWS) {
            const int r = (j * NT + tid) >> 3, pos = (tid & 7) ^ swz(r);
            s_off[j] = (unsigned)min(r, a.tokens - 1 - t0) * (unsigned)g.s_b + (unsigned)pos * 16u;
            s_none[j] = pos * VEC >= tail;
        } else {
            const int q = j * NT + tid, k = q / XPER;
            s_off[j] = (unsigned)k * (unsigned)g.s_b + (unsigned)min(place(q, XPER), (g.s_n - t0) / VEC - 1) * 16u;
            s_none[j] = k >= tail;
        }
    }
    int left = slabs;
    auto issue = [&](unsigned stage) {
        const unsigned to = ring + stage + (unsigned)wave * 1024u;
        if (--left > 0 || tail == KS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma16_saddr(f_off[j], f_ptr, to + j * NT * 16u);
#pragma unroll
            for (int j = 0; j < LX; ++j) lds_dma16_saddr(s_off[j], s_ptr, to + C::TILE + j * NT * 16u);
        } else {  // k that the last slab does not have
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_dma<16>(f_none[j] ? a.zeros : f_ptr + f_off[j], to + j * NT * 16u);
#pragma unroll
            for (int j = 0; j < LX; ++j) lds_dma<16>(s_none[j] ? a.zeros : s_ptr + s_off[j], to + C::TILE + j * NT * 16u);
        }
        f_ptr += f_step;
        s_ptr += s_step;
    };
    f32x16 acc[2][FN];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    const int kg = lane >> 5, lr = lane & 31;
    uint4 ff[2][2], sf[2][FN];  // fragments of a step and of the next
    auto first = [&](unsigned stage, int ks, int i) { ff[ks & 1][i] = grad_frag<T, 128>(smem + stage + (ww >> 1) * C::HALF, (ww & 1) * 2 + i, lane, 2 * ks + kg); };
    auto other = [&](unsigned stage, int ks, int j) {
        const char *ts = smem + stage + C::TILE;
        sf[ks & 1][j] = ROWS ? read_frag<half_t, XR, FILL_VEC_K>(ts, (wt * FN + j) * 32 + lr, ks, kg) : grad_frag<T, XR>(ts, wt * FN + j, lane, 2 * ks + kg);
    };
    auto load = [&](unsigned stage, int ks) {
#pragma unroll
        for (int i = 0; i < 2; ++i) first(stage, ks, i);
#pragma unroll
        for (int j = 0; j < FN; ++j) other(stage, ks, j);
    };
    if constexpr (ES == 2) {
        // step t of what is in registers, while those of step `to` are read from `from` and loads d0 .. d0 + PER_STEP - 1 of a slab go to `into`
        // (d0 < 0: none): one by one between the matrix instructions.  (Two slabs at a time in LDS: all loads in the first step, since they
        // are needed a slab later; three: over the four of them.)
        static_assert(FN == 2, "four matrix instructions a step");
        constexpr int NS = C::NS, L = 4 + LX, PER_STEP = NS == 2 ? L : (L + 3) / 4;
        auto step = [&](int t, unsigned from, int to, int d0, unsigned into) {
            const unsigned at = ring + into + (unsigned)wave * 1024u;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                if (m & 1) first(from, to, m >> 1);
                else other(from, to, m >> 1);
                if (d0 >= 0) {
#pragma unroll
                    for (int j = d0 + m * PER_STEP / 4; j < d0 + (m + 1) * PER_STEP / 4; ++j) {
                        if (j >= L) break;
                        if (j < 4) lds_dma16_saddr(f_off[j], f_ptr, at + j * NT * 16u);
                        else lds_dma16_saddr(s_off[j - 4], s_ptr, at + C::TILE + (j - 4) * NT * 16u);
                    }
                }
                mfma_step<T>(acc[m >> 1][m & 1], ff[t & 1][m >> 1], sf[t & 1][m & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Slab s lies in place s % NS.  Its barrier lies in front of its last step, whose fragments are in registers by then: its place takes
        // slab s + NS.
        auto next = [](unsigned stage) { return stage + C::STAGE == C::RING ? 0u : stage + C::STAGE; };
        unsigned in = 0, out = 0;
        for (int s = 0; s < NS; ++s) {
            if (s < slabs) issue(in);
            in = next(in);
        }
        if (slabs >= NS) wait_vmcnt<(NS - 1) * L>();
        else wait_vmcnt<0>();
        __syncthreads();
        load(0, 0);
        step(0, 0, 1, -1, 0);
        step(1, 0, 2, -1, 0);
        step(2, 0, 3, -1, 0);
        int s = 0;
        for (; s + NS < slabs - (tail == KS ? 0 : 1); ++s) {  // (slab s + NS is a whole one)
            wait_vmcnt<(NS - 2) * L>();
            __syncthreads();
            const unsigned from = next(out);
            step(3, from, 0, 0, out);
            step(0, from, 1, PER_STEP < L ? PER_STEP : -1, out);
            step(1, from, 2, 2 * PER_STEP < L ? 2 * PER_STEP : -1, out);
            step(2, from, 3, 3 * PER_STEP < L ? 3 * PER_STEP : -1, out);
            f_ptr += f_step;
            s_ptr += s_step;
            --left;
            out = from;
        }
        for (; s + 1 < slabs; ++s) {
            if (s + NS <= slabs) wait_vmcnt<(NS - 2) * L>();
            else wait_vmcnt<0>();
            __syncthreads();
            if (s + NS < slabs) issue(out);
            const unsigned from = next(out);
            step(3, from, 0, -1, 0);
            step(0, from, 1, -1, 0);
            step(1, from, 2, -1, 0);
            step(2, from, 3, -1, 0);
            out = from;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) mfma_step<T>(acc[m >> 1][m & 1], ff[1][m >> 1], sf[1][m & 1]);
    } else {
        issue(0);
        unsigned out = 0;
        for (int s = 0; s < slabs; ++s) {
            wait_vmcnt<0>();
            __syncthreads();
            if (s + 1 < slabs) issue(C::STAGE - out);
            load(out, 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t < 3) load(out, t + 1);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) mfma_step<T>(acc[i][j], ff[t & 1][i], sf[t & 1][j]);
            }
            out = C::STAGE - out;
        }
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

template <typename T, int XR, int FW>
__global__ __launch_bounds__((GradTile<T, XR, FW>::NT)) void grad_kernel(const GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    if ((int)blockIdx.x >= a.tiles) {
        typedef GradTile<T, XR, FW> C;
        static_assert(sizeof(LongSum<T>) * 1024 <= C::RING, "fits the ring");
        row_shares_of<T, C::NT>(a.shares, static_cast<T *>(a.db), a.rows, a.n_shares, (int)blockIdx.x - a.tiles, reinterpret_cast<LongSum<T>(*)[32]>(smem));
        return;
    }
    const int second = (int)blockIdx.x >= a.first, id = second ? (int)blockIdx.x - a.first : (int)blockIdx.x;
    if ((second ^ a.lead) == 0) grad_tile<T, XR, FW, true>(a.p[0], id, smem);
    else grad_tile<T, XR, FW, false>(a.p[1], id, smem);
}

// The parts' sums, in their order, rounded once: four values a thread.
template <typename T>
struct GradJoin {
    const float *part[2];
    T *y[2];
    size_t n[2], values[2];  // fours of values (0: not in parts), values
    int parts[2], high[2];
};
template <typename T>
__global__ __launch_bounds__(256) void grad_join_kernel(const GradJoin<T> a) {
    size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int o = i >= a.n[0];
    if (o) i -= a.n[0];
    if (i >= a.n[o]) return;
    const float4 *p = reinterpret_cast<const float4 *>(a.part[o]) + i;
    float4 s = p[0];
    float4 low = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 1; k < a.parts[o]; ++k) {
        const float4 v = p[(size_t)k * a.n[o]];
        float4 &t = k < a.high[o] ? s : low;
        t.x += v.x;
        t.y += v.y;
        t.z += v.z;
        t.w += v.w;
    }
    s = make_float4(fmaf(low.x, 1.f / GRAD_LOW, s.x), fmaf(low.y, 1.f / GRAD_LOW, s.y), fmaf(low.z, 1.f / GRAD_LOW, s.z), fmaf(low.w, 1.f / GRAD_LOW, s.w));
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 v = t4{(T)s.x, (T)s.y, (T)s.z, (T)s.w};
    if (4 * i + 4 <= a.values[o]) {
        reinterpret_cast<t4 *>(a.y[o])[i] = v;
    } else {
        for (int e = 0; 4 * i + e < a.values[o]; ++e) a.y[o][4 * i + e] = v[e];
    }
}

// Microseconds of the launch with k of the two products in so many parts.  fp16: a workgroup takes 0.95 a slab while it shares its compute
// unit with another, 0.7 alone, and 4 for the rest; what remains behind the long ones is half of a short one in the mean.  fp32: a slab
// and tile is 0.67 of a compute unit, 1.18 to a workgroup alone, the rest of a workgroup two slabs, what remains behind 1.7 times a
// short one (fitted to 14 layers with 20 choices each: 7 % off in the mean, the choice 1.05 times the best in the mean, 1.11 at most).
// Parts cost their sums, written and read at 5 TB/s, and a launch.
static float grad_cost(const int (&tiles)[2], const int (&slabs)[2], const double (&values)[2], const int (&parts)[2], bool fp32, int wide) {
    const int cu = state().num_cu;
    const float rest = fp32 ? 1.8f : 0.f;
    float work = 0, longest = 0, shortest = 1e9f, extra = 0, groups = 0;
    for (int i = 0; i < 2; ++i) groups += (float)tiles[i] * parts[i];
    const float slab = fp32 ? 1.f : groups > cu ? 0.95f : 0.7f;
    for (int i = 0; i < 2; ++i) {
        if (!tiles[i]) continue;
        const float one = (slabs[i] + parts[i] - 1) / parts[i] * slab + (fp32 ? rest : 4.f);
        work += one * tiles[i] * parts[i];
        longest = one > longest ? one : longest;
        shortest = one < shortest ? one : shortest;
        if (parts[i] > 1) extra += (float)(values[i] * 8e-6 * parts[i] / 5.0);
    }
    if (fp32) {
        const float beside = groups < 3.f * cu ? groups / cu : 3.f, alone = 0.67f * beside > 1.18f ? 0.67f * beside : 1.18f;
        const float spread = 0.67f * (work / cu + 1.7f * shortest), chain = longest * (groups <= 3.f * cu ? alone : 1.18f);
        return (spread > chain ? spread : chain) + (extra > 0 ? 0.72f * extra + 3.5f : 0.f);
    }
    const float spread = work / ((wide == 128 ? 2 : 1) * cu) + 0.5f * shortest;
    return (spread > longest ? spread : longest) + (extra > 0 ? extra + 4.f : 0.f);
}

template <typename T>
struct GradSizes {
    static constexpr int XR = sizeof(T) == 4 ? 64 : 128, KS = ROWB / (int)sizeof(T);
};
// Slabs of k of product i, of a part, and parts.
template <typename T>
static void grad_cut(int i, int parts, int ns, int rows, int &chunk, int &high) {
    const int slabs = ((i ? ns : rows) + GradSizes<T>::KS - 1) / GradSizes<T>::KS;
    chunk = (slabs + parts - 1) / parts;
    high = (slabs + chunk - 1) / chunk;
}

template <typename T, int FW>
static bool grad_ready() {
    static bool ready = false;
    constexpr int XR = GradSizes<T>::XR;
    if (!ready)
        ready = hip_ok(hipFuncSetAttribute(reinterpret_cast<const void *>(grad_kernel<T, XR, FW>), hipFuncAttributeMaxDynamicSharedMemorySize, GradTile<T, XR, FW>::RING),
                       "hipFuncSetAttribute");
    return ready;
}

// In tiles of so many inputs, the parts of least cost and what their sums take.
template <typename T>
static GradParts grad_plan(int wide, bool dw, bool dx, bool low, int ns, int in, int rows) {
    constexpr int XR = GradSizes<T>::XR, KS = GradSizes<T>::KS;
    GradParts p = {wide, {1, 1}, 0};
    const bool wanted[2] = {dx, dw};
    const int n[2] = {ns, rows}, k[2] = {rows, ns};
    int tiles[2], slabs[2];
    double values[2];
    for (int i = 0; i < 2; ++i) {
        tiles[i] = wanted[i] ? (in + wide - 1) / wide * ((n[i] + XR - 1) / XR) : 0;
        slabs[i] = (k[i] + KS - 1) / KS;
        values[i] = (double)n[i] * in;
    }
    float best = 1e30f;
    for (int u = 1; u <= 32 && (u == 1 || (tiles[0] && u * 4 <= slabs[0])); u *= 2)
        for (int v = 1; v <= 32 && (v == 1 || (tiles[1] && v * 4 <= slabs[1])); v *= 2) {
            const int parts[2] = {u, v};
            const float c = grad_cost(tiles, slabs, values, parts, sizeof(T) == 4, wide);
            if (c < best) {
                best = c;
                p.parts[0] = u;
                p.parts[1] = v;
            }
        }
    for (int i = 0; i < 2; ++i) {
        int chunk, high;
        grad_cut<T>(i, p.parts[i], ns, rows, chunk, high);
        const size_t parts = low && wanted[i] ? 2 * high : high;
        if (parts > 1) p.bytes += parts * grad_part(n[i], in) * sizeof(float);
    }
    return p;
}
template <typename T>
int gated_products_plan(GradParts &p, GradParts &less, bool dw, bool dx, bool low, int ns, int in, int rows) {
    p = less = grad_plan<T>(128, dw, dx, low, ns, in, rows);
    if constexpr (sizeof(T) == 2) {
        // Of 30 layers in fp16 (256 to 8192 tokens, 256 to 8192 inputs and outputs) tiles of 256 inputs take 0.94 times as long from 16 GFLOP on
        // (0.89 to 1.03) and below 1.01 (0.99 to 1.05): one workgroup a compute unit shares what two would read, but fewer of them fill the chip
        // less evenly.  Half as many tiles of a layer of few inputs may want their k in more parts, whose sums take more memory (7385 tokens,
        // 256 -> 3752 gated 129 us and 30 MB, 153 and none).
        if (2.0 * ns * in * rows * (dw + dx) >= 16e9) p = grad_plan<T>(256, dw, dx, low, ns, in, rows);
        if (p.bytes <= less.bytes) less = p;
    }
    const bool wide = p.wide == 256 || less.wide == 256, narrow = p.wide == 128 || less.wide == 128;
    return (!narrow || grad_ready<T, 128>()) && (!wide || grad_ready<T, sizeof(T) == 2 ? 256 : 128>()) ? 0 : 2;
}

template <typename T>
int gated_products(const GradParts &parts, float *ws, const T *x, const T *w, const T *dh, const T *low, T *dw, T *dx, int ns, int in, int rows, int cols,
                   int pitch, const float *shares, T *db, int n_shares) {
    constexpr int XR = GradSizes<T>::XR;
    GradArgs a = {};
    T *y[2] = {dx, dw};
    const int n[2] = {ns, rows}, k[2] = {rows, ns};
    GradJoin<T> j = {};
    for (int i = 0; i < 2; ++i) {
        GradProd &p = a.p[i];
        p.out.y = y[i];
        p.out.outs = in;
        p.out.tokens = n[i];
        p.out.zeros = static_cast<const char *>(state().zeros);
        p.out.tiles_w = (in + parts.wide - 1) / parts.wide;
        p.out.tiles_t = (n[i] + XR - 1) / XR;
        p.f = reinterpret_cast<const char *>(i ? x : w);
        p.s = reinterpret_cast<const char *>(dh);
        p.k = k[i];
        p.f_b = cols * (int)sizeof(T);
        p.s_b = pitch * (int)sizeof(T);
        p.f_n = cols;
        p.s_n = pitch;
        grad_cut<T>(i, parts.parts[i], ns, rows, p.chunk, p.high);
        p.low = reinterpret_cast<const char *>(low);
        p.parts = low && y[i] ? 2 * p.high : p.high;
        if (p.parts == 1) continue;
        p.part = ws;
        j.part[i] = ws;
        j.y[i] = y[i];
        j.values[i] = (size_t)n[i] * in;
        j.n[i] = grad_part(n[i], in) / 4;
        j.parts[i] = p.parts;
        j.high[i] = p.high;
        ws += (size_t)p.parts * grad_part(n[i], in);
    }
    a.lead = a.p[0].chunk >= a.p[1].chunk ? 0 : 1;
    int groups[2];
    for (int i = 0; i < 2; ++i) groups[i] = y[i] ? a.p[i].out.tiles_w * a.p[i].out.tiles_t * a.p[i].parts : 0;
    a.first = groups[a.lead];
    a.tiles = groups[0] + groups[1];
    a.shares = shares;
    a.db = db;
    a.rows = rows;
    a.n_shares = n_shares;
    const int all = a.tiles + (db ? (rows + 31) / 32 : 0);
    auto launch = [&](auto wide) {
        typedef GradTile<T, XR, decltype(wide)::value> C;
        hipLaunchKernelGGL((grad_kernel<T, XR, decltype(wide)::value>), dim3(all), dim3(C::NT), C::RING, state().stream, a);
    };
    if (parts.wide == 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, sizeof(T) == 2 ? 256 : 128>{});
    if (parts.bytes) {
        const size_t fours = j.n[0] + j.n[1];
        hipLaunchKernelGGL((grad_join_kernel<T>), dim3((unsigned)((fours + 255) / 256)), dim3(256), 0, state().stream, j);
    }
    return hip_ok(hipGetLastError(), "gated layer launch") ? 0 : 2;
}

template int gated_products_plan<half_t>(GradParts &, GradParts &, bool, bool, bool, int, int, int);
template int gated_products_plan<float>(GradParts &, GradParts &, bool, bool, bool, int, int, int);
template int gated_products<half_t>(const GradParts &, float *, const half_t *, const half_t *, const half_t *, const half_t *, half_t *, half_t *, int, int, int, int,
                                    int, const float *, half_t *, int);
template int gated_products<float>(const GradParts &, float *, const float *, const float *, const float *, const float *, float *, float *, int, int, int, int, int,
                                   const float *, float *, int);

void rows_copy(const void *w, size_t n_w, const void *x, size_t n_x, void *to, int bytes, int pitch) {
    rows_copies(static_cast<const char *>(w), n_w, static_cast<const char *>(x), n_x, static_cast<char *>(to), bytes, pitch);
}

}  // namespace ptl
