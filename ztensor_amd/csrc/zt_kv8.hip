// Rotary positions, and the int8 paged cache of keys and values: its writer,
// its dequantizer, and the pages' bookkeeping.  The attention that reads it is
// in zt_attn.hip.
//
// All of it moves bytes: a page holds, for each head, page x Dp codes of keys
// [token][dim] and as many of values [dim][token] (the order in which the
// attention's two products read them), and one fp32 scale of each.
#include <algorithm>
#include <limits>
#include <type_traits>

#include "zt_kv8.h"

namespace zt {

constexpr int kThreads = 256;

// ------------------------------------------------------------------- rotary

struct RopeArgs {
    Rows in[2], out[2];
    Turn turn;
    int tokens, dim;
    int units;       // of one head
    int all;         // of one token
    int per_block;   // tokens that a workgroup takes (1 where a token fills more than one)
    int chunks;      // workgroups that such a token takes
};

// One unit of 2 V values a thread.
template <class T, int V>
__device__ __forceinline__ void rope_block(const RopeArgs& g, int block) {
    const int group = g.chunks == 1 ? block : block / g.chunks;
    const int i = (block - group * g.chunks) * kThreads + threadIdx.x;
    if (i >= g.per_block * g.all) return;
    const int tl = g.per_block == 1 ? 0 : i / g.all, r = i - tl * g.all;
    const long t = (long)group * g.per_block + tl;
    if (t >= g.tokens) return;
    int h = r / g.units;
    const int u = r - h * g.units;
    const int w = h >= g.in[0].heads;
    h -= w ? g.in[0].heads : 0;
    const Rows &x = g.in[w], &y = g.out[w];
    float a[V], b[V];
    int first, second;
    turned<T, V>((const T*)x.p + t * x.token + h * x.head, u, g.turn.positions[t], g.turn, a, b, first, second);
    T* o = (T*)y.p + t * y.token + h * y.head;
    store_values<T, V>(o + first, a);
    store_values<T, V>(o + second, b);
}

// (a, b) -> (a c - b s, b c + a s): each value once in and once out, so bytes
// bound it.  A thread has 16 bytes of each half of its pairs where the strides
// allow it, and a workgroup the units of one token (of several, where a token
// fills less), so that one row of the table serves neighbouring threads.
// 4099 tokens of 72 heads of 128 fp16: 152 MB in 30.6 us, 4.97 TB/s, what a copy
// reaches; one token: 2.5 us, the launch.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs g) {
    rope_block<T, V>(g, blockIdx.x);
}

// The launch of n operands, and the units' size: V.
__host__ inline long rope_blocks(RopeArgs& g, int n, int V) {
    const int heads = g.in[0].heads + (n > 1 ? g.in[1].heads : 0);
    g.units = g.turn.half / V + (g.dim - 2 * g.turn.half) / (2 * V);
    g.all = heads * g.units;
    g.per_block = g.all >= kThreads ? 1 : kThreads / g.all;
    g.chunks = ceil_div(g.per_block * g.all, kThreads);
    return (long)ceil_div(g.tokens, g.per_block) * g.chunks;
}

// The widest V that all operands allow: 16 bytes of fp16 or fp32, 4 values, else one by one.
__host__ inline int rope_width(const zt_rows* const* r, int n, int dim, int half, int type) {
    const int widths[2] = {8, 4};
    for (int v : widths) {
        bool ok = units_fit(v, dim, half) && (v == 4 || type == ZT_F16);
        for (int i = 0; i < n && ok; i++) ok = rows_vector(*r[i], v, type);
        if (ok) return v;
    }
    return 1;
}

// -------------------------------------------------------- rotary, normed heads

struct NormArgs {
    RopeArgs r;  // (its `all`: chunks of heads of one token)
    HeadNorm norm[2];
    int lanes;  // of one head: a power of two
};

// g.lanes lanes have kHeads heads of one token, whose weights and angles are the
// same: those are read once, and the heads' loads wait together.  Bytes bound it:
// 4099 tokens, 64 + 4 heads of 128 of which 64 dims are turned, fp16, 144 MB in 30
// us, 4.8 TB/s, 26 where half of it is in the Infinity Cache (one head at a time
// 42); one token 3.8 us, the launch and the chain from its position to the angles.
constexpr int kHeads = 4;
template <class T, int V, Pairs P>
__device__ __forceinline__ void norm_block(const NormArgs& g, int block) {
    constexpr int N = kHeadUnits<V>;
    const int l = threadIdx.x & (g.lanes - 1);
    const long item = ((long)block * kThreads + threadIdx.x) / g.lanes, t = item / g.r.all;
    if (t >= g.r.tokens) return;
    int chunk = (int)(item - t * g.r.all);
    const int chunks = (g.r.in[0].heads + kHeads - 1) / kHeads, which = chunk >= chunks;
    chunk -= which ? chunks : 0;
    const Rows &x = g.r.in[which], &y = g.r.out[which];
    const HeadNorm& norm = g.norm[which];
    const int h0 = chunk * kHeads, n = min(kHeads, x.heads - h0);
    float a[kHeads][N][V], b[kHeads][N][V], w[N][2][V], cs[N][2][V];
    int first[N], second[N];
    const int pos = g.r.turn.half ? g.r.turn.positions[t] : 0;
#pragma unroll
    for (int h = 0; h < kHeads; h++)  // (past the last head: that one again)
        load_head<T, V, N, P>((const T*)x.p + t * x.token + (h0 + min(h, n - 1)) * x.head, l, g.lanes, g.r.units, g.r.turn, a[h], b[h], first, second);
#pragma unroll
    for (int k = 0; k < N; k++) {
        load_weights<V>(norm, first[k], w[k][0]);
        load_weights<V>(norm, second[k], w[k][1]);
        load_angles<V>(l + k * g.lanes, pos, g.r.turn, cs[k][0], cs[k][1]);
    }
#pragma unroll
    for (int h = 0; h < kHeads; h++) {
        const float r = head_factor<V, N>(l, g.lanes, g.r.units, norm, a[h], b[h]);
        T* o = (T*)y.p + t * y.token + (h0 + h) * y.head;
#pragma unroll
        for (int k = 0; k < N; k++) {
            if (h >= n || l + k * g.lanes >= g.r.units) continue;
            scale_unit<V>(r, w[k][0], a[h][k]);
            scale_unit<V>(r, w[k][1], b[h][k]);
            turn_by<V, P>(l + k * g.lanes, g.r.turn, cs[k][0], cs[k][1], a[h][k], b[h][k]);
            store_values<T, V>(o + first[k], a[h][k]);
            store_values<T, V>(o + second[k], b[h][k]);
        }
    }
}

template <class T, int V, Pairs P>
__global__ __launch_bounds__(kThreads) void norm_kernel(NormArgs g) {
    norm_block<T, V, P>(g, blockIdx.x);
}

// The launch of n operands whose heads are normed.
__host__ inline long norm_blocks(NormArgs& g, int n, int V) {
    g.r.units = g.r.turn.half / V + (g.r.dim - 2 * g.r.turn.half) / (2 * V);
    g.r.all = ceil_div(g.r.in[0].heads, kHeads) + (n > 1 ? ceil_div(g.r.in[1].heads, kHeads) : 0);
    g.lanes = head_lanes(g.r.units);
    return ((long)g.r.tokens * g.r.all * g.lanes + kThreads - 1) / kThreads;
}

__host__ inline bool norm_ok(const zt_head_norm* n) {
    return n && n->eps > 0 && n->eps <= std::numeric_limits<double>::max() && (((uintptr_t)n->q | (uintptr_t)n->k) & 3) == 0;
}

}  // namespace zt

using namespace zt;

ZT_EXPORT int zt_norm_rope(const zt_rows* in, const zt_rows* out, int n, const zt_head_norm* norm, const int* positions,
                           const float* table, int tokens, int head_dim, int rot_dim, int max_pos, int type, int flags,
                           zt_stream_t stream) {
    if (!in || !out || n < 1 || n > 2 || !norm_ok(norm) || tokens < 0 || head_dim < 2 || head_dim % 2 || head_dim > 256 ||
        !type_ok(type) || (flags & ~ZT_ROPE_INTERLEAVED) ||
        (table && (rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim || max_pos < 1)))
        return kInvalid;
    const zt_rows* all[4];
    for (int i = 0; i < n; i++) {
        if (in[i].heads != out[i].heads || in[i].heads > (1 << 20) / head_dim) return kInvalid;
        all[2 * i] = in + i;
        all[2 * i + 1] = out + i;
    }
    if (tokens == 0) return 0;
    for (int i = 0; i < 2 * n; i++)
        if (!rows_ok(*all[i], type)) return kInvalid;
    if (table && (!positions || ((uintptr_t)positions & 3) || ((uintptr_t)table & 3))) return kInvalid;
    NormArgs g{};
    for (int i = 0; i < n; i++) {
        g.r.in[i] = rows_of(in[i]);
        g.r.out[i] = rows_of(out[i]);
    }
    g.r.turn = {positions, table, table ? rot_dim / 2 : 0, max_pos, flags};
    g.r.tokens = tokens;
    g.r.dim = head_dim;
    g.norm[0] = {norm->q, norm->eps, 1.0 / head_dim};
    g.norm[1] = {norm->k, norm->eps, 1.0 / head_dim};
    const int v = rope_width(all, 2 * n, head_dim, g.r.turn.half, type);
    const long blocks = norm_blocks(g, n, v);
    if (blocks >= 1l << 31) return kInvalid;
    auto run = [&](auto kernel) { kernel<<<blocks, kThreads, 0, stream>>>(g); };
    auto with = [&](auto pairs) {
        constexpr Pairs P = decltype(pairs)::value;
        if (type == ZT_F32)
            v == 4 ? run(norm_kernel<float, 4, P>) : run(norm_kernel<float, 1, P>);
        else
            v == 8 ? run(norm_kernel<_Float16, 8, P>) : v == 4 ? run(norm_kernel<_Float16, 4, P>) : run(norm_kernel<_Float16, 1, P>);
    };
    flags & ZT_ROPE_INTERLEAVED ? with(std::integral_constant<Pairs, Pairs::INTERLEAVED>{}) : with(std::integral_constant<Pairs, Pairs::HALVES>{});
    return (int)hipGetLastError();
}

ZT_EXPORT int zt_rope(const zt_rows* in, const zt_rows* out, int n, const int* positions, const float* table, int tokens,
                      int head_dim, int rot_dim, int max_pos, int type, int flags, zt_stream_t stream) {
    if (!in || !out || n < 1 || n > 2 || tokens < 0 || head_dim < 2 || head_dim % 2 || rot_dim < 2 || rot_dim % 2 ||
        rot_dim > head_dim || max_pos < 1 || !type_ok(type) || (flags & ~(ZT_ROPE_INTERLEAVED | ZT_ROPE_INVERSE)))
        return kInvalid;
    const zt_rows* all[4];
    for (int i = 0; i < n; i++) {
        if (in[i].heads != out[i].heads || in[i].heads > (1 << 20) / head_dim) return kInvalid;
        all[2 * i] = in + i;
        all[2 * i + 1] = out + i;
    }
    if (tokens == 0) return 0;
    for (int i = 0; i < 2 * n; i++)
        if (!rows_ok(*all[i], type)) return kInvalid;
    if (!positions || !table || ((uintptr_t)positions & 3) || ((uintptr_t)table & 3)) return kInvalid;
    RopeArgs g{};
    for (int i = 0; i < n; i++) {
        g.in[i] = rows_of(in[i]);
        g.out[i] = rows_of(out[i]);
    }
    g.turn = {positions, table, rot_dim / 2, max_pos, flags};
    g.tokens = tokens;
    g.dim = head_dim;
    const int v = rope_width(all, 2 * n, head_dim, rot_dim / 2, type);
    const long blocks = rope_blocks(g, n, v);
    if (blocks >= 1l << 31) return kInvalid;
    if (type == ZT_F32) {
        if (v == 4)
            rope_kernel<float, 4><<<blocks, kThreads, 0, stream>>>(g);
        else
            rope_kernel<float, 1><<<blocks, kThreads, 0, stream>>>(g);
    } else if (v == 8) {
        rope_kernel<_Float16, 8><<<blocks, kThreads, 0, stream>>>(g);
    } else if (v == 4) {
        rope_kernel<_Float16, 4><<<blocks, kThreads, 0, stream>>>(g);
    } else {
        rope_kernel<_Float16, 1><<<blocks, kThreads, 0, stream>>>(g);
    }
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------- append

namespace zt {

struct AppendArgs {
    Kv8 c;
    Rows x[2];  // keys, values
    const long* slots;
    Turn turn;  // half == 0: keys as they are
    HeadNorm norm;  // of the keys, where the kernel norms them
    int lanes;      // that share a key for that
    int tokens;
    int windows;  // of 64 tokens
    // workgroups that a window's pages are dealt out to, for one head of keys or of values, and those of the last window
    // (no more than its tokens); where that is one, it takes the first `first` of them, and `helpers` share the further ones
    // of every groups-th window
    int turns, last, first, groups, helpers;
    long blocks;
};

// The tokens of one page: n of them, from token t on.
struct Run {
    int t, n, page, off;
    bool fresh;  // one of them is the page's first
    // tokens and places one after the other, from t and `off` on; else as listed: tokens from t on, and their places
    bool dense;
    const int* listed;
    const uint8_t* places;
    __device__ __forceinline__ int token(int i) const { return t + (dense ? i : listed[i]); }
    __device__ __forceinline__ int place(int i) const { return dense ? off + i : places[i]; }
};

// A run's tokens into their page: its new scale, and its codes by way of an image
// of it in LDS.
template <class T, int V, bool VALUES, bool NORM, Pairs P>
__device__ __forceinline__ void append_page(const AppendArgs& g, const Run& run, int head, int tid, uint32_t* image, float* red, float* factors) {
    const Kv8& c = g.c;
    const Rows& x = g.x[VALUES];
    Turn turn = g.turn;
    if (VALUES) turn.half = 0;
    const int units = units_of<V>(c.dim, turn.half);
    const int n = run.n;
    const T* rows = (const T*)x.p + (long)head * x.head;
    float m = 0.0f;
    bool bad = false;
    auto look = [&](const float (&a)[V], const float (&b)[V]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            m = fmaxf(m, fmaxf(fabsf(a[j]), fabsf(b[j])));
            bad |= !(fabsf(a[j]) <= kMaxFloat) || !(fabsf(b[j]) <= kMaxFloat);
        }
    };
    auto unit = [&](int tl, int u, int t, float (&a)[V], float (&b)[V], int& first, int& second) __attribute__((always_inline)) {
        const int pos = turn.half ? turn.positions[t] : 0;
        load_unit<T, V, P>(rows + (long)t * x.token, u, turn, a, b, first, second);
        if constexpr (NORM) {
            float w[2][V];
            load_weights<V>(g.norm, first, w[0]);
            load_weights<V>(g.norm, second, w[1]);
            scale_unit<V>(factors[tl], w[0], a);
            scale_unit<V>(factors[tl], w[1], b);
        }
        turn_unit<V, P>(u, pos, turn, a, b);
    };
    // Normed keys: lanes share a row, and kHeld rows' loads wait together.
    constexpr int N = kHeadUnits<V>, kHeld = NORM ? 2 : 1;
    float ha[kHeld][N][V], hb[kHeld][N][V];
    int first_of[N], second_of[N];
    const int shift = NORM ? __builtin_ctz(g.lanes) : 0, l = tid & ((1 << shift) - 1), at_once = kThreads >> shift, mine = tid >> shift;
    if constexpr (NORM) {
        float w[N][2][V];
        for (int i0 = mine; i0 < n + mine; i0 += kHeld * at_once) {
            float cs[kHeld][N][2][V];
            int pos[kHeld];
#pragma unroll
            for (int e = 0; e < kHeld; e++) {
                if (e && i0 - mine + e * at_once >= n) break;  // (the same for the workgroup)
                const int t = run.token(min(i0 + e * at_once, n - 1));
                pos[e] = turn.half ? turn.positions[t] : 0;
                load_head<T, V, N, P>(rows + (long)t * x.token, l, g.lanes, units, turn, ha[e], hb[e], first_of, second_of);
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                load_weights<V>(g.norm, first_of[k], w[k][0]);
                load_weights<V>(g.norm, second_of[k], w[k][1]);
#pragma unroll
                for (int e = 0; e < kHeld; e++) {
                    if (e && i0 - mine + e * at_once >= n) break;
                    load_angles<V>(l + k * g.lanes, pos[e], turn, cs[e][k][0], cs[e][k][1]);
                }
            }
#pragma unroll
            for (int e = 0; e < kHeld; e++) {
                if (e && i0 - mine + e * at_once >= n) break;
                const float r = head_factor<V, N>(l, g.lanes, units, g.norm, ha[e], hb[e]);
                if (l == 0 && i0 + e * at_once < n) factors[i0 + e * at_once] = r;
#pragma unroll
                for (int k = 0; k < N; k++) {
                    scale_unit<V>(r, w[k][0], ha[e][k]);
                    scale_unit<V>(r, w[k][1], hb[e][k]);
                    turn_by<V, P>(l + k * g.lanes, turn, cs[e][k][0], cs[e][k][1], ha[e][k], hb[e][k]);
                    if (i0 + e * at_once < n && l + k * g.lanes < units) look(ha[e][k], hb[e][k]);
                }
            }
        }
    } else {
        for (int i = tid; i < n * units; i += kThreads) {
            const int tl = i / units, u = i - tl * units;
            float a[V], b[V];
            int first, second;
            unit(tl, u, run.token(tl), a, b, first, second);
            look(a, b);
        }
    }
    block_peak(m, bad, red);

    float* scales = VALUES ? c.v_scale : c.k_scale;
    const long at = (long)run.page * c.heads + head;
    const bool fresh = run.fresh;
    const float had = fresh ? 0.0f : scales[at];
    const float now = bad || had != had ? __builtin_nanf("") : fmaxf(had, m * (1.0f / 127.0f));
    const bool grown = now > had, whole = fresh || grown;
    u32x4* codes = reinterpret_cast<u32x4*>((VALUES ? c.v : c.k) + c.at(run.page, head));
    u32x4* image4 = reinterpret_cast<u32x4*>(image);
    // 16 bytes each: all of the page, or, of keys of a page that goes on with its scale, the new tokens' rows
    const int row = c.dp / 16, pieces = whole ? c.bytes() / 16 : n * row;
    auto piece = [&](int i) { return whole ? i : run.dense ? run.off * row + i : run.place(i / row) * row + i % row; };
    const float ratio = grown ? had / now : 0.0f;
    if (grown && !fresh) {
        for (int i = tid; i < pieces; i += kThreads) {
            u32x4 w = codes[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t o = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o |= ((uint32_t)(int)rintf((float)(int8_t)(w[j] >> 8 * e) * ratio) & 0xFFu) << 8 * e;
                w[j] = o;
            }
            image4[i] = w;
        }
    } else if (whole || !VALUES) {  // zeros where nothing new comes; of a page that goes on, its new keys' rows
        for (int i = tid; i < pieces; i += kThreads) image4[piece(i)] = (u32x4){0, 0, 0, 0};
    }
    __syncthreads();  // (the scale has been read by everybody, too)

    int8_t* bytes = reinterpret_cast<int8_t*>(image);
    const float step = now > 0.0f ? now : 1.0f;  // 1 for a NaN, whose codes nobody takes for values
    auto write = [&](int place, const float (&a)[V], const float (&b)[V], int first, int second) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int p = code_of(a[j], step), q = code_of(b[j], step);
            if (VALUES) {
                bytes[(first + j) * c.page + place] = (int8_t)p;
                bytes[(second + j) * c.page + place] = (int8_t)q;
            } else {
                bytes[place * c.dp + first + j] = (int8_t)p;
                bytes[place * c.dp + second + j] = (int8_t)q;
            }
        }
    };
    if (NORM && n <= kHeld * at_once) {
#pragma unroll
        for (int e = 0; e < kHeld; e++)
#pragma unroll
            for (int k = 0; k < N; k++)
                if (mine + e * at_once < n && l + k * g.lanes < units)
                    write(run.place(mine + e * at_once), ha[e][k], hb[e][k], first_of[k], second_of[k]);
    } else {
        for (int i = tid; i < n * units; i += kThreads) {
            const int tl = i / units, u = i - tl * units;
            float a[V], b[V];
            int first, second;
            unit(tl, u, run.token(tl), a, b, first, second);
            write(run.place(tl), a, b, first, second);
        }
    }
    __syncthreads();

    if (whole || !VALUES) {
        for (int i = tid; i < pieces; i += kThreads) codes[piece(i)] = image4[piece(i)];
    } else {
        int8_t* out = reinterpret_cast<int8_t*>(codes);
        for (int i = tid; i < c.dim * n; i += kThreads) {
            const int d = i / n, to = d * c.page + run.place(i - d * n);
            out[to] = bytes[to];
        }
    }
    if (tid == 0) scales[at] = now;
    __syncthreads();  // the image is free again
}

// The page of a slot; none (-1) of one outside the cache.
__device__ __forceinline__ int page_of(const Kv8& c, long slot) {
    return slot >= 0 && slot < (long)c.pages << c.shift ? (int)(slot >> c.shift) : -1;
}

struct Found {
    int dense;  // tokens from the run's first on, one after the other
    int end;    // the first token of another page
    int last;   // the last token of this one's
    int count;  // of a list
    int fresh;
};

// The tokens on the page of token t, whose slot is s: up to the first that is on
// another page, without those that are left out.
__device__ __forceinline__ Run run_from(const AppendArgs& g, int t, long s, int tid, Found& found, int* listed, uint8_t* places) {
    const Kv8& c = g.c;
    const int left = g.tokens - t;
    Run run{t, 0, (int)(s >> c.shift), (int)(s & (c.page - 1)), false, true, listed, places};
    const int most = min(c.page - run.off, left);
    if (tid == 0) found = {most, left, 0, 0, 0};
    __syncthreads();
    auto look = [&](int i, long x, bool first) {  // token t + i, of the 64 of this wave, has slot x
        const int p = i < left ? page_of(c, x) : -1, from = i - (tid & 63);
        const uint64_t other = __ballot(p >= 0 && p != run.page), same = __ballot(p == run.page);
        const uint64_t gap = first ? __ballot(i < most && x != s + i) : 0;
        if ((tid & 63) == 0) {
            if (gap) atomicMin(&found.dense, from + __builtin_ctzll(gap));
            if (other) atomicMin(&found.end, from + __builtin_ctzll(other));
            if (same) atomicMax(&found.last, from + 63 - __builtin_clzll(same));
        }
    };
    look(tid, tid < left ? g.slots[t + tid] : -1, true);
    __syncthreads();
    // (a page that ends the step, or is followed by many tokens that are left out)
    constexpr int kAhead = 8;
    for (int i0 = kThreads; i0 < left && found.end >= i0; i0 += kAhead * kThreads) {
        long x[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; e++) x[e] = i0 + e * kThreads + tid < left ? g.slots[(long)t + i0 + e * kThreads + tid] : -1;
        __syncthreads();  // everybody has seen that the run goes on
#pragma unroll
        for (int e = 0; e < kAhead; e++) look(i0 + e * kThreads + tid, x[e], false);
        __syncthreads();
    }
    run.n = found.dense;
    run.fresh = run.off == 0;
    const int end = min(found.end, found.last + 1);
    if (end <= run.n) return run;
    // some of its tokens come after a gap: a list of all
    run.dense = false;
    for (int i0 = 0; i0 < end; i0 += kThreads) {
        const long x = i0 + tid < end ? g.slots[(long)t + i0 + tid] : -1;
        const bool mine = page_of(c, x) == run.page;
        const uint64_t all = __ballot(mine);
        int at = 0;
        if ((tid & 63) == 0 && all) at = atomicAdd(&found.count, __builtin_popcountll(all));
        at = __shfl(at, 0) + __builtin_popcountll(all & ((1ull << (tid & 63)) - 1));
        if (mine && at < c.page) {  // (more would be a slot that comes twice)
            listed[at] = i0 + tid;
            places[at] = (uint8_t)(x & (c.page - 1));
            if ((x & (c.page - 1)) == 0) found.fresh = 1;
        }
    }
    __syncthreads();
    run.n = min(found.count, c.page);
    run.fresh = found.fresh;
    return run;
}

// What a workgroup helps with, of each of its waves: the tokens that begin pages, and their slots.  A wave looks at kLooks
// windows at a time, and has a helper's part of each one's at most 64 pages.
constexpr int kLooks = 4;
struct Jobs {
    long slot[4][16 * kLooks];
    int token[4][16 * kLooks];
    int n[4];
};

// A page's scale s' = max(s, amax / 127), its codes rint(c s / s') where it grew,
// new ones rint(x / s'): one workgroup has a page of one head, keys or values,
// whole, since all of its codes wait for one maximum.  It reads its new rows
// twice (the second time from L2), and puts the codes together in LDS: values
// lie token-minor, and go out as whole 16 bytes instead of one byte a line.
// No atomics on memory, and no order among workgroups.
//
// A workgroup looks at a window of 64 tokens: those whose page is not that of the
// one before (tokens that are left out do not come between) begin a page's tokens.
// It takes every turns-th of them, each with all that follow on its page; or
// (HELP) the first few, and the call's first workgroups also take their part of
// what crowded windows have besides: page i of the k-th window of a group is helper
// (61 k + i) % helpers', which spreads pages evenly however many a window has.  q's
// rotation rides along as more workgroups, instead of a launch of its own.
//
// One token for each of 64 sequences (8 heads of 128, pages of 64, fp32): 10.4
// us, where a page that grows is read and written; a workgroup waits for its
// slots, its rows, their largest, the scale and the codes one after the other.
// Prompts of 1955 tokens in all (fp16, 32 + 8 heads of 128, pages of 16): 17.1 us.
//
// Normed keys: a row is dealt out to lanes that share its sum of squares, two
// rows at a time (four: 3218 tokens of prompts 30.4 us instead of 31.0, but 48
// sequences' tokens 12.0 instead of 10.3, for code that most of them skip).  A run
// that is as short as that stays in registers, others' factors are kept in LDS
// for the second reading.
template <class T, int V, int VQ, class Q, Pairs P, bool HELP>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs g, Q q) {
    constexpr bool NORM = std::is_same_v<Q, NormArgs>;
    extern __shared__ __align__(16) uint32_t image[];  // of one page and head
    __shared__ float factors[NORM ? 128 : 1];
    __shared__ float red[4];
    __shared__ Found found;
    __shared__ int listed[128];
    __shared__ uint8_t places[128];
    if (blockIdx.x >= g.blocks) {
        if constexpr (NORM)
            norm_block<T, VQ, P>(q, blockIdx.x - g.blocks);
        else
            rope_block<T, VQ>(q, blockIdx.x - g.blocks);
        return;
    }
    const Kv8& c = g.c;
    int b = blockIdx.x;
    const int values = b & 1, head = (b >> 1) % c.heads;
    b = (b >> 1) / c.heads;
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto lower = [&](uint64_t bits) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bits, 0)); };  // of lanes before this one
    auto slot = [&](long t) { return t >= 0 && t < g.tokens ? g.slots[t] : -1l; };
    // of 64 tokens, whose slots are `here` (and `before` that of the one before them), those that begin a page and are wanted
    // by that page's number among these
    auto begun = [&](long from, long here, long before, auto wanted) __attribute__((always_inline)) {
        const int page = page_of(c, here);
        const uint64_t stored = __ballot(page >= 0), below = stored & ((1ull << lane) - 1);
        if (!stored) return (uint64_t)0;
        int last = page_of(c, before);  // the page of the last token before these that is stored
        for (long t = from - 2; last < 0 && t >= 0; t -= 64) {
            const int p = page_of(c, slot(t - lane));
            const uint64_t any = __ballot(p >= 0);
            if (any) last = __shfl(p, __builtin_ctzll(any));
        }
        const int prior = __shfl(page, below ? 63 - __builtin_clzll(below) : lane);
        const bool begins = page >= 0 && page != (below ? prior : last);
        const int i = lower(__ballot(begins));
        return (uint64_t)__ballot(begins && wanted(i));
    };
    auto append = [&](int t, long s) __attribute__((always_inline)) {
        int tid = threadIdx.x;
        // (worked out for each page, not held in registers meanwhile: eight waves a SIMD instead of seven; normed keys', which
        // have more to work out, are four anyway)
        if constexpr (!NORM) asm volatile("" : "+v"(tid));
        const Run run = run_from(g, t, s, tid, found, listed, places);
        if (values)
            append_page<T, V, true, false, P>(g, run, head, tid, image, red, factors);
        else
            append_page<T, V, false, NORM, P>(g, run, head, tid, image, red, factors);
    };
    if constexpr (!HELP) {
        int turn = 0, windows = g.windows;  // all windows' first workgroups come first
        if (b >= g.last * windows) {
            turn = g.last;
            b -= turn * windows--;
        }
        const int row = b / windows, from = (b - row * windows) * 64;
        turn += row;
        const long here = slot(from + lane), behind = slot((long)from - 1);
        uint64_t todo = begun(from, here, behind, [&](int) { return true; });
        for (int left = turn; todo; todo &= todo - 1) {
            if (left-- > 0) continue;
            left = g.turns - 1;
            const int i = __builtin_ctzll(todo);
            append(from + i, __shfl(here, i));
        }
    } else {
        __shared__ Jobs jobs;
        const long own = b < g.windows ? 64l * b : -64;
        const long here = slot(own + lane), behind = slot(own - 1);
        int group = 0, help = 0, count = 0;  // the windows that it helps with
        if (b < g.groups * g.helpers) {
            help = b / g.groups;
            group = b - help * g.groups;
            count = (g.windows - group + g.groups - 1) / g.groups;
        }
        uint64_t todo = 0;
        for (int k0 = 0;; k0 += 4 * kLooks) {
            asm volatile("" : "+v"(lane));  // (what depends on it is worked out here, not held in registers while pages are written)
            auto from = [&](int e) { return 64l * (group + (long)(k0 + kLooks * wave + e) * g.groups); };
            long x[kLooks];
            if (k0 < count) {
#pragma unroll
                for (int e = 0; e < kLooks; e++) x[e] = slot(from(e) + lane);
            }
            if (k0 == 0) todo = begun(own, here, behind, [&](int i) { return i < g.first; });
            int w = 4, n = 0;
            if (k0 < count) {
                uint32_t more = 0;  // windows with more than `first` tokens that are not on the page of the one before
#pragma unroll
                for (int e = 0; e < kLooks; e++) {
                    const int page = page_of(c, x[e]), before = __shfl_up(page, 1);
                    if (__builtin_popcountll(__ballot(page >= 0 && (lane == 0 || page != before))) > g.first) more |= 1u << e;
                }
                for (; more; more &= more - 1) {
                    const int e = __builtin_ctz(more);
                    const uint32_t k = k0 + kLooks * wave + e;
                    const long at = slot(from(e) + lane);
                    const uint64_t all = begun(from(e), at, slot(from(e) - 1), [&](int i) { return i >= g.first && (61 * k + i) % (uint32_t)g.helpers == (uint32_t)help; });
                    if (all >> lane & 1) {
                        const int j = n + lower(all);
                        jobs.token[wave][j] = (int)from(e) + lane;
                        jobs.slot[wave][j] = at;
                    }
                    n += __builtin_popcountll(all);
                }
                if (lane == 0) jobs.n[wave] = n;
                __syncthreads();
                w = n = 0;
            }
            for (;;) {
                int t;
                long s;
                if (todo) {
                    const int i = __builtin_ctzll(todo);
                    todo &= todo - 1;
                    t = (int)own + i;
                    s = __shfl(here, i);
                } else {
                    while (w < 4 && n == __builtin_amdgcn_readfirstlane(jobs.n[w])) {
                        w++;
                        n = 0;
                    }
                    if (w == 4) break;
                    t = __builtin_amdgcn_readfirstlane(jobs.token[w][n]);
                    s = jobs.slot[w][n++];
                }
                append(t, (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(s >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)s)));
            }
            if (k0 + 4 * kLooks >= count) break;
            __syncthreads();  // nobody reads the list any more
        }
    }
}

}  // namespace zt

template <Pairs P, class Q>
static int launch_append(const AppendArgs& g, const Q& q, long blocks, int type, int width, int q_width, hipStream_t stream) {
    if (blocks >= 1l << 31) return kInvalid;
    const int lds = g.c.bytes();
    auto run = [&](auto kernel) { kernel<<<blocks, kThreads, lds, stream>>>(g, q); };
    auto with = [&](auto help) {
        constexpr bool H = decltype(help)::value;
        if (type == ZT_F32) {
            if (width == 4)
                q_width == 4 ? run(append_kernel<float, 4, 4, Q, P, H>) : run(append_kernel<float, 4, 1, Q, P, H>);
            else
                q_width == 4 ? run(append_kernel<float, 1, 4, Q, P, H>) : run(append_kernel<float, 1, 1, Q, P, H>);
        } else if (width == 4) {
            q_width == 8 ? run(append_kernel<_Float16, 4, 8, Q, P, H>) : q_width == 4 ? run(append_kernel<_Float16, 4, 4, Q, P, H>) : run(append_kernel<_Float16, 4, 1, Q, P, H>);
        } else {
            q_width == 8 ? run(append_kernel<_Float16, 1, 8, Q, P, H>) : q_width == 4 ? run(append_kernel<_Float16, 1, 4, Q, P, H>) : run(append_kernel<_Float16, 1, 1, Q, P, H>);
        }
    };
    g.helpers ? with(std::true_type{}) : with(std::false_type{});
    return (int)hipGetLastError();
}

static int append(const zt_kv8_cache* cache, const zt_rows* k, const zt_rows* v, const long* slots, const zt_rows* q,
                  const zt_rows* q_out, const zt_head_norm* norm, const int* positions, const float* table, int tokens,
                  int rot_dim, int max_pos, int type, int flags, hipStream_t stream) {
    if (!cache || !kv8_ok(*cache) || !k || !v || tokens < 0 || tokens >= 1l << 30 || !type_ok(type) || (flags & ~ZT_ROPE_INTERLEAVED) ||
        (q == nullptr) != (q_out == nullptr) || (q && !table && !norm))
        return kInvalid;
    const int dim = cache->head_dim, half = table ? rot_dim / 2 : 0;
    if (table && (rot_dim < 2 || rot_dim % 2 || rot_dim > dim || max_pos < 1)) return kInvalid;
    if (k->heads != cache->kv_heads || v->heads != cache->kv_heads) return kInvalid;
    if (q && (q->heads != q_out->heads || q->heads > (1 << 20) / dim)) return kInvalid;
    if (tokens == 0) return 0;
    const zt_rows* all[4] = {k, v, q, q_out};
    const int n = q ? 4 : 2;
    for (int i = 0; i < n; i++)
        if (!rows_ok(*all[i], type)) return kInvalid;
    if (!slots || ((uintptr_t)slots & 7) || (table && (!positions || ((uintptr_t)positions & 3) || ((uintptr_t)table & 3))))
        return kInvalid;
    // 4 values at a time for keys and values (values are not turned: 8 divide the head, a unit of 4 pairs), q as wide as it allows
    const int width = units_fit(4, dim, half) && rows_vector(*k, 4, type) && rows_vector(*v, 4, type) ? 4 : 1;
    const int q_width = q ? rope_width(all + 2, 2, dim, half, type) : 1;
    AppendArgs g{};
    g.c = kv8_of(*cache);
    g.x[0] = rows_of(*k);
    g.x[1] = rows_of(*v);
    g.slots = slots;
    g.turn = {positions, table, half, max_pos, flags};
    g.tokens = tokens;
    g.windows = ceil_div(tokens, 64);
    // A workgroup for each token (a batch's next tokens, each on a page of its own) as long as all are surely at work at a
    // time; then as many for 64 tokens as that is, if at least five, else as twice that is (us, fp16, with q, four heads for
    // each of keys, pages of 16; 8 heads, single tokens of 65, 128, 200, 1024 and 2048 sequences 10.7, 12.9, 15.7, 47 and 90;
    // with 64 for 64 tokens 14.7, 15.2 and 25, with eight 59 and 93, with four 57 and 106).  One that finds no page to begin
    // costs its launch and its look at 64 slots, and prompts begin few.  So where twice would be few, too, there is one, which
    // takes the pages that a prompt begins there, and as many as are surely at work at a time share the others (pages of 64;
    // us with these, with eight in any case, and with one alone: a prompt of 16000 tokens 97, 131 and 94; 8192 sequences'
    // single tokens 492, 492 and 614; 300 of them before a prompt of 8000 58, 84 and 200; 4096 255, with 1792 workgroups that
    // share, some of which begin when others have ended, 349).
    const long pairs = 2l * cache->kv_heads, most = norm ? 1024 : 1536, once = most / (pairs * g.windows);
    if (pairs * g.windows <= (norm ? 256 : 512)) {
        g.turns = pairs * tokens <= most ? 64 : (int)std::min(64l, once >= 5 ? once : 2 * most / (pairs * g.windows));
        g.last = std::min(g.turns, tokens - 64 * (g.windows - 1));
        g.blocks = pairs * ((long)g.windows * g.turns - (g.turns - g.last));
    } else {
        g.first = std::max(64 / g.c.page + 1, 4);
        const int all = std::max(8, (int)(most / pairs));
        // enough groups for one look at each one's windows, and for all helpers; at least six of these in each
        g.groups = std::min({g.windows, all / 6, std::max(ceil_div(g.windows, 4 * kLooks), ceil_div(all, 64))});
        g.helpers = std::min(64, all / g.groups);
        g.blocks = pairs * std::max((long)g.windows, (long)g.groups * g.helpers);
    }
    RopeArgs r{};
    r.turn = g.turn;
    r.tokens = tokens;
    r.dim = dim;
    if (q) {
        r.in[0] = rows_of(*q);
        r.out[0] = rows_of(*q_out);
    }
    if (!norm) {
        const long more = q ? rope_blocks(r, 1, q_width) : 0;
        return launch_append<Pairs::FLAGS>(g, r, g.blocks + more, type, width, q_width, stream);
    }
    g.norm = {norm->k, norm->eps, 1.0 / dim};
    g.lanes = head_lanes(half / width + (dim - 2 * half) / (2 * width));
    NormArgs m{r, {{norm->q, norm->eps, 1.0 / dim}, {}}, 1};
    const long more = q ? norm_blocks(m, 1, q_width) : 0;
    if (flags & ZT_ROPE_INTERLEAVED) return launch_append<Pairs::INTERLEAVED>(g, m, g.blocks + more, type, width, q_width, stream);
    return launch_append<Pairs::HALVES>(g, m, g.blocks + more, type, width, q_width, stream);
}

ZT_EXPORT int zt_kv8_append(const zt_kv8_cache* cache, const zt_rows* k, const zt_rows* v, const long* slots,
                            const zt_rows* q, const zt_rows* q_out, const int* positions, const float* table, int tokens,
                            int rot_dim, int max_pos, int type, int flags, zt_stream_t stream) {
    return append(cache, k, v, slots, q, q_out, nullptr, positions, table, tokens, rot_dim, max_pos, type, flags, stream);
}

ZT_EXPORT int zt_kv8_append_norm(const zt_kv8_cache* cache, const zt_rows* k, const zt_rows* v, const long* slots,
                                 const zt_rows* q, const zt_rows* q_out, const zt_head_norm* norm, const int* positions,
                                 const float* table, int tokens, int rot_dim, int max_pos, int type, int flags,
                                 zt_stream_t stream) {
    if (!norm_ok(norm)) return kInvalid;
    return append(cache, k, v, slots, q, q_out, norm, positions, table, tokens, rot_dim, max_pos, type, flags, stream);
}

// ------------------------------------------------------------------ dequant

namespace zt {

// code * scale: a byte in and four out, so the stores bound it.  One page and
// head of keys or of values a workgroup, 4 values a store.  Values go through
// LDS, in rows 4 bytes longer than a page so that neighbouring dims of one token
// lie in different banks.  64 pages of 64 tokens x 8 heads of 128: 42 MB in 10.5
// us, 4 TB/s.
__global__ __launch_bounds__(kThreads) void dequant_kernel(Kv8 c, const int* pages, float* keys, float* values) {
    __shared__ uint32_t image[256 * (128 + 4) / 4];
    const int is_v = blockIdx.x & 1, head = (blockIdx.x >> 1) % c.heads, i = (blockIdx.x >> 1) / c.heads;
    const int p = pages[i];
    const bool held = c.holds(p);
    float* out = (is_v ? values : keys) + ((long)i * c.heads + head) * c.page * c.dim;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>((is_v ? c.v : c.k) + (held ? c.at(p, head) : 0));
    const float scale = held ? (is_v ? c.v_scale : c.k_scale)[(long)p * c.heads + head] : __builtin_nanf("");
    const int row = is_v ? c.page / 4 : 0;
    if (is_v && held) {
        for (int j = threadIdx.x; j < c.dim * row; j += kThreads) image[j / row * (row + 1) + j % row] = codes[j];
    }
    __syncthreads();
    const int8_t* bytes = reinterpret_cast<const int8_t*>(image);
    const int quads = c.dim / 4;
    for (int j = threadIdx.x; j < c.page * quads; j += kThreads) {
        const int t = j / quads, d = (j - t * quads) * 4;
        float o[4];
        if (is_v) {
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (float)bytes[(d + e) * (c.page + 4) + t] * scale;
        } else {
            const uint32_t w = held ? codes[(t * c.dp + d) / 4] : 0;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (float)(int8_t)(w >> 8 * e) * scale;
        }
        store16(out + (long)t * c.dim + d, o);
    }
}

}  // namespace zt

ZT_EXPORT int zt_kv8_dequant(const zt_kv8_cache* cache, const int* pages, int n, float* keys, float* values,
                             zt_stream_t stream) {
    if (!cache || !kv8_ok(*cache) || n < 0) return kInvalid;
    if (n == 0) return 0;
    if (!pages || !keys || !values || (((uintptr_t)pages | (uintptr_t)keys | (uintptr_t)values) & 3)) return kInvalid;
    const long blocks = 2l * n * cache->kv_heads;
    if (blocks >= 1l << 31) return kInvalid;
    dequant_kernel<<<blocks, kThreads, 0, stream>>>(kv8_of(*cache), pages, keys, values);
    return (int)hipGetLastError();
}

// --------------------------------------------------------------------- plan

namespace zt {

struct PlanArgs {
    const int *kv_lens, *add, *table, *free_pages, *free_count;
    int requests, width, free_capacity, shift, tokens;
    int *table_out, *positions, *q_start, *kv_lens_out, *free_count_out;
    long* slots;
};

struct Request {
    int held, add, have, need;  // tokens held and added, pages held and wanted
    bool fits;
};

__device__ __forceinline__ Request request(const PlanArgs& g, int r) {
    Request q;
    q.held = max(0, g.kv_lens[r]);
    q.add = max(0, g.add[r]);
    const long end = (long)q.held + q.add, room = (1l << g.shift) - 1;
    q.fits = end <= min((long)g.width << g.shift, 0x7FFFFFFFl);
    q.have = (int)((q.held + room) >> g.shift);
    q.need = q.fits ? (int)((end + room) >> g.shift) - q.have : 0;
    return q;
}

// The workgroup's sum of v, in every thread.
__device__ __forceinline__ long block_sum(long v, long* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// Prefix sums of what the requests add and want.  A few loads that wait for each
// other are all of its time (8 requests 3.5 us, 512 of 4.5 MB in all 6.0): one
// launch, instead of sums and then their use.
//
// Workgroup r: request r's row, tokens and length.  Each sums up what the
// requests before it add and want by itself (a few loads a thread: no second
// launch, no order among the workgroups).  The last one has the tokens past
// the last request's, and what is left of the free list: a request that wants
// pages gets them if the wants up to its own are there, so once one does not,
// no later one does, and the largest sum that is there has been given away.
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs g) {
    __shared__ long red[4];
    const int r = blockIdx.x;
    const int free = min(max(0, *g.free_count), g.free_capacity);
    long before = 0, wanted = 0;
    for (int i = threadIdx.x; i < r; i += kThreads) {
        const Request q = request(g, i);
        before += q.add;
        wanted += q.need;
    }
    before = block_sum(before, red);
    wanted = block_sum(wanted, red);
    if (r < g.requests) {
        const Request q = request(g, r);
        const bool done = q.fits && (q.need == 0 || wanted + q.need <= free);
        const int* row = g.table + (long)r * g.width;
        int* out = g.table_out + (long)r * g.width;
        const int* fresh = g.free_pages + (free - 1 - wanted + q.have);  // read at -j: page j of the row, if it is new
        for (int j = threadIdx.x; j < g.width; j += kThreads)
            out[j] = done && j >= q.have && j < q.have + q.need ? fresh[-j] : row[j];
        for (long i = threadIdx.x; i < q.add && before + i < g.tokens; i += kThreads) {
            const long pos = q.held + i;
            const int j = (int)(pos >> g.shift);
            const int page = !done ? -1 : j >= q.have ? fresh[-j] : row[j];
            g.slots[before + i] = page < 0 ? -1 : ((long)page << g.shift) + (pos & ((1l << g.shift) - 1));
            g.positions[before + i] = (int)pos;
        }
        if (threadIdx.x == 0) {
            g.q_start[r] = (int)min(before, 0x7FFFFFFFl);
            g.kv_lens_out[r] = done ? q.held + q.add : q.held;
        }
        return;
    }
    for (long i = before + threadIdx.x; i < g.tokens; i += kThreads) {
        g.slots[i] = -1;
        g.positions[i] = 0;
    }
    __shared__ int sums[2][kThreads];
    __shared__ int given;
    if (threadIdx.x == 0) {
        g.q_start[r] = (int)min(before, 0x7FFFFFFFl);
        given = 0;
    }
    int base = 0;
    for (int i0 = 0; i0 < g.requests; i0 += kThreads) {  // running sums, 256 requests at a time
        const int i = i0 + (int)threadIdx.x, need = i < g.requests ? request(g, i).need : 0;
        int upto = need, at = 0;
        sums[0][threadIdx.x] = upto;
        __syncthreads();
        for (int o = 1; o < kThreads; o <<= 1, at ^= 1) {
            upto += (int)threadIdx.x >= o ? sums[at][threadIdx.x - o] : 0;
            sums[at ^ 1][threadIdx.x] = upto;
            __syncthreads();
        }
        if (need > 0 && base + upto <= free) atomicMax(&given, base + upto);
        base += sums[at][kThreads - 1];
        __syncthreads();
    }
    if (threadIdx.x == 0) *g.free_count_out = free - given;
}

}  // namespace zt

ZT_EXPORT int zt_kv8_plan(const int* kv_lens, const int* add, const int* table, int requests, int width,
                          const int* free_pages, const int* free_count, int free_capacity, int page_tokens, int tokens,
                          int* table_out, long* slots, int* positions, int* q_start, int* kv_lens_out,
                          int* free_count_out, zt_stream_t stream) {
    if (requests < 0 || width < 1 || tokens < 0 || free_capacity < 0 || !page_tokens_ok(page_tokens) ||
        (long)requests * width >= (1l << 31) - 256 || requests >= 1 << 24)
        return kInvalid;
    if (requests && (!kv_lens || !add || !table || !table_out || !kv_lens_out)) return kInvalid;
    if ((free_capacity && !free_pages) || !free_count || !free_count_out || !q_start || (tokens && (!slots || !positions)))
        return kInvalid;
    const void* ints[] = {kv_lens,   add,       table,   free_pages,  free_count,
                          table_out, positions, q_start, kv_lens_out, free_count_out};
    for (const void* p : ints)
        if ((uintptr_t)p & 3) return kInvalid;
    if ((uintptr_t)slots & 7) return kInvalid;
    // what one workgroup writes the others do not read (a table's row has one workgroup: it may be written in place)
    const long row = 4l * requests, rows = row * width;
    const Bytes in[] = {{kv_lens, row}, {add, row}, {free_pages, 4l * free_capacity}, {free_count, 4}, {table, rows}};
    const Bytes out[] = {{slots, 8l * tokens},  {positions, 4l * tokens}, {q_start, row + 4},
                         {kv_lens_out, row}, {free_count_out, 4},      {table_out, rows}};
    for (const Bytes& o : out) {
        for (const Bytes& i : in)
            if (o.meets(i) && !(o.p == table_out && i.p == table && table_out == table)) return kInvalid;
        for (const Bytes& other : out)
            if (&other < &o && o.meets(other)) return kInvalid;
    }
    PlanArgs g{kv_lens,  add,     table,     free_pages, free_count, requests,    width,         free_capacity, __builtin_ctz(page_tokens),
               tokens,   table_out, positions, q_start,  kv_lens_out, free_count_out, slots};
    plan_kernel<<<requests + 1, kThreads, 0, stream>>>(g);
    return (int)hipGetLastError();
}
