// Attention over the int8 paged cache: o = sum_j w_j v_j / sum_j w_j with w_j =
// 2^(f q.k_j - m), m a running maximum of the scores and f = scale log2(e) times
// the scale of the keys' page; one pass over the tokens, sums in fp32.
//
// Few rows (a batch's next tokens) read their sequences' codes once, and bytes
// bound them; the rows of a prompt read each tile many times, and the products
// and exponentials do.  So there are two kernels, and a third that joins what
// several waves have of one row.  A call whose requests have at most 64 rows of a
// key/value head (tokens x the group of its q heads) is the first kernel's, which
// reads a tile for 16 or 32 of them; in a call of longer ones those of up to 64
// still are, and the others' rows are the second's, up to 128 at a time.
#include <algorithm>
#include <cmath>

#include "zt_kv8.h"

namespace zt {

struct AttnArgs {
    Kv8 c;
    Rows q, out;
    const int *table, *kv_lens, *q_start;
    const float* scale;
    int requests, width, tokens, window, group;
    float unit, unit_lo;  // log2(e) / sqrt(dim) in two parts: a score's factor where no scale is given
};

// ------------------------------------------------- few rows: a long axis split

// Workgroups of one request and head along its tokens, and the tiles of 64
// tokens that each takes (the last one: all that are left).
struct Split {
    int splits, tiles;
};

struct Work {
    AttnArgs a;
    int most;    // requests of up to so many rows (a row: a token and one of the heads of a group) are the few kernel's
    int shares;  // waves of the few kernel
    int empties; // workgroups of a key/value head for the rows of no request
    bool single; // each takes whole heads
    Split many;
    int qtiles;  // workgroups along the rows of the other kernel
    int vec;     // q and out in pieces of 4 values
    long others; // rows of sums that the few kernel has room for; the other kernel's follow
    long places; // of both
    int most_parts;  // of a row
    float* part;   // [][dp]: sums of a row over some of its tokens, not yet divided,
    float2* stat;  // and their (maximum, sum of weights)
    int2* parts;   // [tokens][q heads]: of each row, the place of its first part's sums, and how many parts there are
    // the place of a row's sums in the other kernel's
    __device__ __forceinline__ long many_at(int split, int t, int h) const {
        return others + ((long)split * a.tokens + t) * a.q.heads + h;
    }
};

// 8 codes as fp16, exact: each byte, its sign bit turned over, goes under the
// byte of 1024's exponent, which makes 1024 + 128 + code.
__device__ __forceinline__ half8v codes8(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t k = 0x64646464u;
    const u32x4 w = {__builtin_amdgcn_perm(k, a, 0x04010400u), __builtin_amdgcn_perm(k, a, 0x04030402u),
                     __builtin_amdgcn_perm(k, b, 0x04010400u), __builtin_amdgcn_perm(k, b, 0x04030402u)};
    const _Float16 o = (_Float16)1152.0f;
    return __builtin_bit_cast(half8v, w) - (half8v){o, o, o, o, o, o, o, o};
}

__device__ __forceinline__ float4v mfma(half8v a, half8v b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

constexpr float kNone = -__builtin_inff();
constexpr float kNothing = -kMaxFloat;  // of a base: below all finite scores, and none of its own differences is not a number
constexpr float kWeightBits = 10.0f, kSumBits = 4.0f;
constexpr float kLog2e = 1.44269504088896340736f, kLog2eLo = (float)(1.44269504088896340736 - (double)kLog2e);

// What makes a product of a query and a key a score in units of log 2, to 48
// bits: an error in it is one of every score in the same direction, and grows
// with them.  fp16 rows take the first 24 (lo stays out): a score of 100 is then
// off by 2^-17, far below the 11 bits that its weight is held in.
struct Factor {
    float hi, lo;
};
__device__ __forceinline__ Factor factor_of(const AttnArgs& g) {
    if (!g.scale) return {g.unit, g.unit_lo};
    const float s = *g.scale, hi = s * kLog2e;
    return {hi, __builtin_fmaf(s, kLog2eLo, __builtin_fmaf(s, kLog2e, -hi))};
}
// The same times a page's scale: hi above 0, and for fp32 rows lo, above 0 too
// (so that both take -inf to -inf).
template <bool SPLIT>
__device__ __forceinline__ Factor times(const Factor& f, float ks) {
    Factor r;
    r.hi = f.hi * ks;
    r.hi = r.hi < 1e-30f ? 1e-30f : r.hi;  // (not a number: stays that)
    r.lo = 0.0f;
    if (SPLIT) {
        r.hi = __uint_as_float(__float_as_uint(r.hi) - 1);
        r.lo = fmaxf(__builtin_fmaf(f.lo, ks, __builtin_fmaf(f.hi, ks, -r.hi)), 1e-37f);
    }
    return r;
}

// 16 values of one row from dim d on, fp32; past the head's size and of no row: 0.
template <class T>
__device__ __forceinline__ void load16(const T* row, int d, int dim, bool vec, float (&v)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        float x[4] = {0, 0, 0, 0};
        if (row && d + e < dim) {  // dim is a multiple of 8
            if (vec) {
                load_values<T, 4>(row + d + e, x);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = (float)row[d + e + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) v[e + i] = x[i];
    }
}

template <class T>
__device__ __forceinline__ void store4(T* row, int d, int dim, bool vec, const float (&v)[4]) {
    if (d >= dim) return;
    if (vec) {
        store_values<T, 4>(row + d, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) row[d + i] = (T)v[i];
    }
}

// The rows of a request and the tokens that they see, by the device's lengths.
struct Span {
    int start, n, len;  // first row, rows, tokens
    int tile0, tile1;   // tiles of 64 tokens that any row sees
};
__device__ __forceinline__ int row_bound(const AttnArgs& g, int r) { return min(max(0, g.q_start[r]), g.tokens); }
// The first token that token i of a request's n sees.  (Lengths and windows may be up to 2^31 - 1: what may pass that is
// a long, or unsigned.)
__device__ __forceinline__ int first_seen(const AttnArgs& g, int len, int n, int i) {
    return g.window > 0 ? (int)max(0l, (long)len - n + i + 1 - g.window) : 0;
}
__device__ __forceinline__ int tiles_up_to(int token) { return (int)(((unsigned)token + 63) >> 6); }
__device__ __forceinline__ Span span_of(const AttnArgs& g, int r) {
    Span s;
    s.start = row_bound(g, r);
    s.n = row_bound(g, r + 1) - s.start;
    const long most = (long)g.width << g.c.shift;
    // (rows that q does not have are the last ones of their request: what only they would see is as good as not there)
    const long cut = max(0, g.q_start[r + 1]) - (long)(s.start + s.n);
    s.len = g.c.pages ? (int)max(0l, min((long)max(0, g.kv_lens[r]), most) - max(0l, cut)) : 0;
    s.tile0 = first_seen(g, s.len, s.n, 0) >> 6;
    s.tile1 = max(tiles_up_to(s.len), s.tile0 + 1);  // (one where there is nothing to see: it gives zeros)
    return s;
}

// Splits that so many tiles fill.
__device__ __forceinline__ int splits_of(const Split& f, int tiles) {
    return min(f.splits, max(1, (tiles + f.tiles - 1) / f.tiles));
}

// Row `row` of a request and key/value head as this lane's operands: dims 64 d
// + 16 (lane / 16) .. +16 of each d, fp32 rows in two parts after a power of
// two; factor: what a product of it is to be multiplied by for a score in
// units of log 2; hi: it sees tokens before that (0: no such row).
template <class T, int DN>
__device__ __forceinline__ void load_query(const Work& f, const Span& sp, int kv, int row, int rows, const Factor& scale,
                                           half8v (&q)[DN][2], half8v (&ql)[DN][2], Factor& factor, int& hi) {
    constexpr bool SPLIT = sizeof(T) == 4;
    const AttnArgs& g = f.a;
    const int i = row / g.group, h = kv * g.group + row - i * g.group, quad = (threadIdx.x & 63) >> 4;
    const bool there = row < rows;
    hi = there ? sp.len - sp.n + i + 1 : 0;
    const T* x = there ? (const T*)g.q.p + (long)(sp.start + i) * g.q.token + (long)h * g.q.head : nullptr;
    float v[DN][16];
    float m = 0.0f;
#pragma unroll
    for (int d = 0; d < DN; d++) {
        load16<T>(x, 64 * d + 16 * quad, g.c.dim, f.vec, v[d]);
#pragma unroll
        for (int e = 0; e < 16; e++) m = fmaxf(m, finite(fabsf(v[d][e])));
    }
    int e2 = 0;
    if (SPLIT) e2 = scale_exponent(max_step<16>(max_step<32>(m)));
    const bool negative = scale.hi < 0.0f;
    factor = {ldexpf(fabsf(scale.hi), -e2), ldexpf(negative ? -scale.lo : scale.lo, -e2)};
    if (negative) {  // its sign goes to the query: a larger product is a larger score
#pragma unroll
        for (int d = 0; d < DN; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) v[d][e] = -v[d][e];
    }
#pragma unroll
    for (int d = 0; d < DN; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if constexpr (SPLIT) {
                float x8[8];
#pragma unroll
                for (int k = 0; k < 8; k++) x8[k] = ldexpf(v[d][8 * e + k], e2);
                split_hi_lo(x8, q[d][e], ql[d][e]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) q[d][e][k] = (_Float16)v[d][8 * e + k];
            }
        }
}

// The scale of a lane's values in a tile, and its logarithm: fp16 rows add it to
// a score, fp32 rows, which multiply a weight by the scale, need a whole number
// that is not below it.  Of nothing: -inf.
struct ValueScale {
    float by, log;
};
template <bool SPLIT>
__device__ __forceinline__ ValueScale value_scale(float vs) {
    if (SPLIT) return {vs, vs > 0.0f ? (float)__builtin_amdgcn_frexp_expf(vs) : kNone};
    return {vs, __builtin_amdgcn_logf(vs)};
}

// What the softmax of one row stands on.  Its sums have two units, each a power
// of two: l is in units of 2^base, base near the largest score so far, and o in
// units of 2^(unit - 10), unit near the largest product of a weight and its
// values' scale.  So fp16 has the weights that matter for o, whatever the scales
// of pages that the row gives no weight, or does not see.
struct Base {
    float base, unit;  // kNothing: nothing yet
    // the factor `by` of sums in o, for the unit of l
    __device__ __forceinline__ float o_in_l(float by) const {
        return ldexpf(by, (int)fminf(fmaxf(unit - base - kWeightBits, -1000.0f), 1000.0f));
    }
};

// Of a tile's 16 tokens in this lane, t on, what a row does not see: tokens that
// are not `there`, from hi on, or (window > 0) not among the last `window` before
// that.  Their scores become -inf; of a lane in which it sees none the scales may
// be anything, and are set aside.
__device__ __forceinline__ void mask_scores(float4v (&s)[4], Factor& fk, ValueScale& v, int t, bool there, int window, int hi) {
    hi -= t;
    const int lo = window > 0 ? hi - window : 0;
    if (!there || hi <= 0 || lo >= 16) {
        fk = {1.0f, 1e-37f};
        v = {1.0f, 1000.0f};  // (a logarithm that asks for nothing: see weights_of)
        hi = 0;
    }
#pragma unroll
    for (int k = 0; k < 16; k++)
        if (k < lo || k >= hi) s[k >> 2][k & 3] = kNone;
}

// The weights of a tile's 16 tokens in this lane for one row: scores s times fk
// in units of log 2, against a base that follows their maximum only when it is
// passed by more than 2^4 (most tiles move some row's maximum a little; so few
// of them change l and o, which stand already), and as the second product takes
// them, times the values' scale, against a unit that follows in the same way: at
// most 2^14 in fp16.  Scales of keys and values are not negative.
template <bool SPLIT, int N>
__device__ __forceinline__ void weights_of(const float4v (&s)[4], const Factor& fk, const ValueScale& v, Base& b, float& l,
                                           float4v (&o)[N], half8v (&p)[2], half8v (&pl)[2]) {
    float top = kNone;
#pragma unroll
    for (int k = 0; k < 16; k++) top = fmaxf(top, s[k >> 2][k & 3]);
    top *= fk.hi;
    const float most = top + v.log;
    if (__any(top > b.base + 4.0f || most > b.unit + 4.0f)) {  // (from nothing: to the first that is seen)
        auto follow = [](float& at, float x) {
            x = ceilf(max_step<16>(max_step<32>(x)));
            const bool up = x > at + 4.0f;
            const float keep = up ? __builtin_amdgcn_exp2f(at - x) : 1.0f;
            at = up ? x : at;
            return keep;
        };
        l *= follow(b.base, top);
        const float keep = follow(b.unit, most);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= keep;
    }
    const float from = b.base, unit = b.unit - kWeightBits;
    float sum = 0.0f;
    if constexpr (SPLIT) {
        float by = ldexpf(v.by, (int)fminf(from - unit, 1000.0f));
        by = by > 0x1p100f ? 0x1p100f : by;  // (of weights that are nothing: 0 times it is not to be NaN)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float x = s[2 * h + (k >> 2)][k & 3];
                const float z = __builtin_amdgcn_exp2f(__builtin_fmaf(x, fk.hi, __builtin_fmaf(x, fk.lo, -from)));
                sum += z;
                y[k] = z * by;
                // one value for both parts: fused into the conversion of one of them, the product would round to another
                // fp16 near a tie, and the parts would be off by its last bit
                asm("" : "+v"(y[k]));
            }
            split_hi_lo(y, p[h], pl[h]);
        }
    } else {
        // The scale in the exponent; fp16 holds 11 bits of a weight.  l adds the weights up as fp16 has them, so that their
        // rounding is the same above and below, but for pages whose scale is so far below that fp16 holds too little of
        // what they add to it: off by at most 2^-25 each where they are small, from 2^kSumBits on that is 2^-29 of l's unit
        // for a token, 2^-13 for 65536 of them.
        // (Of a row that has seen nothing, base and unit are the same: it does not ask for that.)
        const float at = v.log - unit, bits = v.log + kWeightBits + (from - b.unit);
        const half2v one = {(_Float16)1.0f, (_Float16)1.0f};
        const bool apart = __any(bits < kSumBits);
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            const half2v w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 2][k & 3], fk.hi, at)),
                              (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 2][(k & 3) + 1], fk.hi, at))};
            sum = __builtin_amdgcn_fdot2(w, one, sum, false);
            p[k >> 3][k & 7] = w[0];
            p[k >> 3][(k & 7) + 1] = w[1];
        }
        sum *= __builtin_amdgcn_exp2f(-bits);
        if (apart) {
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 2][k & 3], fk.hi, -from));
        }
    }
    l += sum;
}

// The page of a token, as the table has it (a load that nothing waits for until
// the page is needed; past the length: of the last token), and whether there is
// something to see there.
struct Pages {
    const int* row;
    int len, shift;
    __device__ __forceinline__ int operator()(unsigned token) const { return len > 0 ? row[min(token, (unsigned)len - 1) >> shift] : -1; }
    __device__ __forceinline__ bool seen(const Kv8& c, int page, unsigned token) const { return token < (unsigned)len && c.holds(page); }
};

// What a lane holds of a row, dims 16 i + 4 (lane / 16) .. +4: the result, or
// the sum that the other splits' are to be added to.
template <class T, int DN>
__device__ __forceinline__ void store_row(const Work& f, const Span& sp, int kv, int row, int rows, bool part, long at,
                                          const Base& b, float sum, const float4v (&o)[4 * DN]) {
    if (row >= rows) return;
    const AttnArgs& g = f.a;
    const int i = row / g.group, h = kv * g.group + row - i * g.group, quad = (threadIdx.x & 63) >> 4;
    const long t = sp.start + i;
    const float by = b.o_in_l(part ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum);
    if (part && quad == 0) f.stat[at] = make_float2(b.base, sum);
    T* out = (T*)g.out.p + t * g.out.token + (long)h * g.out.head;
#pragma unroll
    for (int k = 0; k < 4 * DN; k++) {
        const float4v x = o[k] * by;
        const int d = 16 * k + 4 * quad;
        if (part)
            *reinterpret_cast<float4v*>(f.part + at * g.c.dp + d) = x;
        else
            store4<T>(out, d, g.c.dim, f.vec, {x[0], x[1], x[2], x[3]});
    }
}

// The few kernel's work is a row of tiles: request after request, and of each
// request its column groups (of 16 CT rows) and key/value heads, each with the
// tiles of 64 tokens that the request sees, after a place for what it takes to
// begin.  Every wave takes an equal share of the row, wherever that begins and
// ends: sequences of any lengths keep all CUs busy to the end.  What a share
// holds of a head's tiles goes to `out` if it is all of them, else to the
// share's place for its first part or its last.
// That place counts as four tiles: 64 sequences of up to 8000 tokens, fp16, 89 us at one, 77 at two, 70 at four or
// seven; fp32 80, 70, 72 and 73.  Where the host knows of few tiles, a head's are one place: nothing is split, nothing
// to be joined.
constexpr int kBegin = 4;
__device__ __forceinline__ int begin_of(const Work& f) { return f.single ? 0 : kBegin; }
__device__ __forceinline__ int length_of(const Work& f, const Span& sp) { return f.single ? 1 : sp.tile1 - sp.tile0 + kBegin; }
__device__ __forceinline__ long places_of(const Work& f, const Span& sp, int rows_of_group) {
    const int rows = sp.n * f.a.group;
    if (sp.n <= 0 || rows > f.most) return 0;
    return (long)((rows + rows_of_group - 1) / rows_of_group) * f.a.c.heads * length_of(f, sp);
}

// Running sums over the lanes, the lane's own included.
__device__ __forceinline__ long wave_scan(long v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long x = __shfl_up(v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// A wave takes its share; up to 16 CT rows (tokens x the group's q heads) of one
// request and head are the columns of the products
//     S^T = K Q^T  (64 tokens x 16)   and   O^T += V^T P^T  (dims x 16),
// whose operands K and V^T come from the cache straight into registers, 16
// bytes a lane: the codes of a lane's tokens and dims are neighbours in both
// layouts, and a lane's scores of the first product are its weights in the
// second.  Row i of the first product's tile j is token 16 (i / 4) + 4 j + i % 4:
// lane (n, g) then holds tokens 16 g .. 16 g + 15 of column n, all on one page,
// and needs the values of just these.  The waves of a workgroup share nothing; a
// lane's queries lie in LDS for itself.
//
// Weights enter the second product times their page's scale over a power of two
// that keeps the row's largest such product so far in 2^8 to 2^14: fp16 then holds
// 32 bits below it.  fp32 rows: queries and weights in two fp16 parts (22 bits).
//
// The codes bound it: 64 sequences of up to 8000 tokens (8 heads of 128, fp32,
// pages of 32) 306 MB in 65 us, 4.7 TB/s, near the rate of a large copy; one of
// 40011 (fp16, pages of 64) 82 MB in 20.3 us, 4.0 TB/s, of which about 5 us are
// the launch and the chain from the lengths to the first codes; 37 tokens 8.9 us,
// all of it that chain.  fp32 rows of two columns keep 24 registers in memory at
// 128 dims, and fp32 rows 78, fp16 rows 25 at 256.
template <class T, int DN, int CT>
__device__ __forceinline__ void few_rows(const Work& f, int block, half8v* queries) {  // [4 waves][CT][DN][2][PARTS][64]
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int PARTS = SPLIT ? 2 : 1;
    const AttnArgs& g = f.a;
    const Kv8& c = g.c;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (f.shares + 3) / 4, share = block * 4 + wave;
    if (block >= blocks) {  // rows of no request: those before the first one's, and past the last one's
        const int kv = (block - blocks) % c.heads, upto = g.requests ? row_bound(g, 0) : 0;
        const int from = g.requests ? max(upto, row_bound(g, g.requests)) : 0, rows = upto + g.tokens - from;
        for (long row = (block - blocks) / c.heads; row < rows; row += f.empties) {
            const int t = (int)(row < upto ? row : from + row - upto);
            for (int i = threadIdx.x; i < g.group * c.dim; i += 256) {
                const int h = i / c.dim;
                if (i - h * c.dim == 0) f.parts[(long)t * g.q.heads + kv * g.group + h] = make_int2(0, 1);
                ((T*)g.out.p)[(long)t * g.out.token + (long)(kv * g.group + h) * g.out.head + i - h * c.dim] = (T)0.0f;
            }
        }
        return;
    }
    if (share >= f.shares) return;
    // the share, and the request of its first place; 64 requests' spans lie in the lanes at a time
    Span span{};
    long all = 0, before = 0, upto = 0, places = 0;
    auto load_spans = [&](int r0) {
        span = Span{};
        if (r0 + lane < g.requests) span = span_of(g, r0 + lane);
        places = places_of(f, span, 16 * CT);
        upto = wave_scan(places);
    };
    for (int r0 = 0; r0 < g.requests; r0 += 64) {
        load_spans(r0);
        all += __shfl(upto, 63);
    }
    const long each = (all + f.shares - 1) / f.shares;
    long pos = share * each;
    const long end = min(all, pos + each);
    if (pos >= end) return;
    int r = 0, r0 = 0;
    for (;; r0 += 64) {
        if (g.requests > 64) load_spans(r0);
        const uint64_t past = __ballot(before + upto > pos);
        if (past) {
            const int l = __builtin_ctzll(past);
            r = r0 + l;
            before += __shfl(upto - places, l);
            break;
        }
        before += __shfl(upto, 63);
    }
    r = __builtin_amdgcn_readfirstlane(r);
    const Factor scale = factor_of(g);
    const int krow = (col >> 2) * 16 + (col & 3);  // this lane's token of a key tile, less 4 j

    while (pos < end) {
        if (r >= r0 + 64) {
            r0 += 64;
            load_spans(r0);
        }
        Span sp;
        sp.start = __builtin_amdgcn_readlane(span.start, r - r0);
        sp.n = __builtin_amdgcn_readlane(span.n, r - r0);
        sp.len = __builtin_amdgcn_readlane(span.len, r - r0);
        sp.tile0 = __builtin_amdgcn_readlane(span.tile0, r - r0);
        sp.tile1 = __builtin_amdgcn_readlane(span.tile1, r - r0);
        const int rows = sp.n * g.group, tiles = sp.tile1 - sp.tile0;
        const long mine = places_of(f, sp, 16 * CT);
        if (pos - before >= mine) {
            before += mine;
            r++;
            continue;
        }
        const int length = length_of(f, sp), begin = begin_of(f);
        const int seg = __builtin_amdgcn_readfirstlane((int)((pos - before) / length));
        const int at0 = __builtin_amdgcn_readfirstlane((int)(pos - before - (long)seg * length));
        const int at1 = (int)min(at0 + end - pos, (long)length);
        const int cg = seg / c.heads, kv = seg - cg * c.heads;
        const int into = max(0, at0 - begin), n = f.single ? tiles : at1 - begin - into;
        const int first = sp.tile0 + into, last = first + n;
        const long first_place = pos - at0 + begin;
        pos += at1 - at0;
        if (n <= 0) continue;
        const int parts = f.single ? 1 : (int)((first_place + tiles - 1) / each) - share + 1;  // (of the first part's share)
        const Pages page_of{g.table + (long)r * g.width, sp.len, c.shift};
        int pk = page_of(first * 64 + (col >> 2) * 16), pv = page_of(first * 64 + quad * 16);
        half8v* mine_q = queries + wave * (CT * DN * 2 * PARTS * 64);
        Factor factor[CT];
        int hi[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            half8v q[DN][2], ql[DN][2];
            load_query<T, DN>(f, sp, kv, (cg * CT + ct) * 16 + col, rows, scale, q, ql, factor[ct], hi[ct]);
#pragma unroll
            for (int d = 0; d < DN; d++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    mine_q[(((ct * DN + d) * 2 + h) * PARTS) * 64 + lane] = q[d][h];
                    if constexpr (SPLIT) mine_q[(((ct * DN + d) * 2 + h) * PARTS + 1) * 64 + lane] = ql[d][h];
                }
        }
        // every row of these columns sees tokens all_lo .. all_hi - 1
        const int row0 = cg * 16 * CT, row1 = min(rows, row0 + 16 * CT) - 1;
        const int all_hi = sp.len - sp.n + row0 / g.group + 1;
        const int all_lo = first_seen(g, sp.len, sp.n, row1 / g.group);

        float4v o[CT][4 * DN];
        Base m[CT];
        float l[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            m[ct] = {kNothing, kNothing};
            l[ct] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) o[ct][i] = (float4v){0, 0, 0, 0};
        }

        for (int tile = first; tile < last && c.pages; tile++) {
            const int t0 = tile * 64;
            int qlane = lane;
            asm volatile("" : "+v"(qlane));  // the queries are read from LDS for each tile: held, they cost 16 to 64 registers
            const bool seen = page_of.seen(c, pv, t0 + 16 * quad);
            const int at = seen ? pv : 0;
            const int8_t* kp = c.k + c.at(page_of.seen(c, pk, t0 + (col >> 2) * 16) ? pk : 0, kv) + (long)((t0 + krow) & (c.page - 1)) * c.dp + 16 * quad;
            const int8_t* vp = c.v + c.at(at, kv) + (long)col * c.page + ((t0 + 16 * quad) & (c.page - 1));
            u32x4 kw[4][DN], vw[4 * DN];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int d = 0; d < DN; d++) kw[j][d] = *reinterpret_cast<const u32x4*>(kp + 4 * j * c.dp + 64 * d);
            const float ks = c.k_scale[(long)at * c.heads + kv], vs = c.v_scale[(long)at * c.heads + kv];
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) vw[i] = *reinterpret_cast<const u32x4*>(vp + (long)16 * i * c.page);
            const bool whole = t0 <= all_hi - 64 && t0 >= all_lo && __all(seen);
            // the next tile's pages, while this one's codes are on their way
            pk = page_of(t0 + 64u + (col >> 2) * 16);
            pv = page_of(t0 + 64u + quad * 16);

            const ValueScale scales = value_scale<SPLIT>(vs);

            float4v s[CT][4];
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[ct][j] = (float4v){0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int d = 0; d < DN; d++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const half8v k8 = codes8(kw[j][d][2 * h], kw[j][d][2 * h + 1]);
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
#pragma unroll
                            for (int part = 0; part < PARTS; part++) s[ct][j] = mfma(k8, mine_q[(((ct * DN + d) * 2 + h) * PARTS + part) * 64 + qlane], s[ct][j]);
                        }
                    }

            half8v p[CT][2], pl[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                Factor fk = times<SPLIT>(factor[ct], ks);
                ValueScale v = scales;
                if (!whole) mask_scores(s[ct], fk, v, t0 + 16 * quad, seen, g.window, hi[ct]);
                weights_of<SPLIT>(s[ct], fk, v, m[ct], l[ct], o[ct], p[ct], pl[ct]);
            }
#pragma unroll
            for (int i = 0; i < 4 * DN; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8v v8 = codes8(vw[i][2 * h], vw[i][2 * h + 1]);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        o[ct][i] = mfma(v8, p[ct][h], o[ct][i]);
                        if constexpr (SPLIT) o[ct][i] = mfma(v8, pl[ct][h], o[ct][i]);
                    }
                }
        }

#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            l[ct] += __shfl_xor(l[ct], 16);
            l[ct] += __shfl_xor(l[ct], 32);
            const long at = ((long)share * 2 + (into == 0)) * (16 * CT) + 16 * ct + col;
            const int row = (cg * CT + ct) * 16 + col, i = row / g.group;
            if (into == 0 && row < rows && quad == 0)
                f.parts[(long)(sp.start + i) * g.q.heads + kv * g.group + row - i * g.group] = make_int2((int)at, parts);
            store_row<T, DN>(f, sp, kv, row, rows, n < tiles, at, m[ct], l[ct], o[ct]);
        }
    }
}

template <class T, int DN, int CT>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(Work f) {
    extern __shared__ __align__(16) half8v shared[];
    few_rows<T, DN, CT>(f, blockIdx.x, shared);
}

// ------------------------------------------------------------ prompts: tiled

// Columns of 16 rows that a wave of the tiled kernel holds.
template <int DN>
constexpr int kCols = DN <= 2 ? 2 : 1;
template <int DN>
constexpr int kRows = 64 * kCols<DN>;  // rows of a workgroup

// The workgroup's rows that `row` is among: the tiles that they see.
struct RowTiles {
    int row0, tile0, tile1;
};
template <int DN>
__device__ __forceinline__ RowTiles tiles_of(const AttnArgs& g, const Span& sp, int row) {
    RowTiles w;
    w.row0 = row / kRows<DN> * kRows<DN>;
    const int last = min(w.row0 + kRows<DN>, sp.n * g.group) - 1;
    w.tile0 = first_seen(g, sp.len, sp.n, w.row0 / g.group) >> 6;
    w.tile1 = max(tiles_up_to(max(0, sp.len - sp.n + last / g.group + 1)), w.tile0);
    return w;
}

// As the few kernel, with the roles of its operands and its numbers, but the
// rows of a prompt read a tile many times: four waves of 16 CT rows each share
// tiles of 64 tokens that they bring to LDS as fp16, decoded once for the
// workgroup's 64 CT rows, each fragment in the order of the lanes that read it
// (16 bytes a lane side by side, no bank conflicts).  The next tile's codes are
// on their way to registers while a tile is worked on, and go to the other
// buffer after it: one barrier a tile.
//
// Two workgroups a CU.  Three prompts (187 GFLOP, 32 heads over 8 of 128, fp16)
// 243 us, 0.77 PFLOP/s, one call after the other (290 for the first ones, before
// the clock has settled).  A tile of one wave is 64 matrix instructions (1024
// cycles) and some 360 of the vector unit (1800 cycles with the exponentials),
// which bounds it: 80 decode its share of the codes, 5 for each of its scores are
// the softmax's.  The last fifth of the time is a tail with half of the
// workgroups.  fp32 rows take twice the products in two fp16 parts: 364 us, 1.03
// PFLOP/s of them, with 38 registers kept in memory; at 256 dims those are 84, of
// fp16 rows 24.
template <class T, int DN>
__device__ __forceinline__ void many_rows(const Work& f, int b, half8v* tiles) {  // [2][FRAGS][64]
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int CT = kCols<DN>, FRAGS = 16 * DN;  // fragments of 64 lanes x 16 bytes in a buffer: keys', then values'
    const AttnArgs& g = f.a;
    const Kv8& c = g.c;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = b % c.heads;
    b /= c.heads;
    const int split = b % f.many.splits;
    b /= f.many.splits;
    const int r = b % g.requests, at = b / g.requests;  // (the longest rows of all requests first)
    const Span sp = span_of(g, r);
    const int rows = sp.n * g.group;
    if (sp.n <= 0 || rows <= f.most) return;
    const Factor scale = factor_of(g);
    const int krow = (col >> 2) * 16 + (col & 3);
    const Pages page_of{g.table + (long)r * g.width, sp.len, c.shift};

    // the later a row, the more tokens it sees: those first
    const int all = (rows + kRows<DN> - 1) / kRows<DN>;
    for (int qt = all - 1 - at; qt >= 0; qt -= f.qtiles) {
        const RowTiles w = tiles_of<DN>(g, sp, qt * kRows<DN>);
        const int ns = splits_of(f.many, w.tile1 - w.tile0);
        if (split >= ns) continue;
        const int first = w.tile0 + split * f.many.tiles, last = split == ns - 1 ? w.tile1 : first + f.many.tiles;

        half8v q[CT][DN][2], ql[CT][DN][2];
        Factor factor[CT];
        int hi[CT];
        const int row0 = w.row0 + wave * 16 * CT, row1 = min(rows, row0 + 16 * CT) - 1;
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
            load_query<T, DN>(f, sp, kv, row0 + 16 * ct + col, rows, scale, q[ct], ql[ct], factor[ct], hi[ct]);
        const int all_hi = sp.len - sp.n + row0 / g.group + 1;
        const int all_lo = first_seen(g, sp.len, sp.n, row1 / g.group);

        float4v o[CT][4 * DN];
        Base m[CT];
        float l[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            m[ct] = {kNothing, kNothing};
            l[ct] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) o[ct][i] = (float4v){0, 0, 0, 0};
        }

        // this wave's share of a tile: key tile j = wave (DN loads), values' dims 16 (DN wave + i) (DN loads)
        u32x4 kw[DN], vw[DN];
        float ks, vs;
        bool seen;
        // (a tile begins at a multiple of 64: what a lane adds to that stays in the page, or is taken modulo its tokens)
        const uint32_t page_bytes = (uint32_t)c.heads * c.bytes(), head_bytes = (uint32_t)kv * c.bytes();
        const uint32_t k_lane = ((krow + 4 * wave) & (c.page - 1)) * c.dp + 16 * quad + head_bytes;
        const uint32_t v_lane = (16 * DN * wave + col) * c.page + ((16 * quad) & (c.page - 1)) + head_bytes;
        auto fetch = [&](int tile, int pk, int pv) {
            const unsigned t0 = tile * 64u, in = t0 & (c.page - 1);
            seen = page_of.seen(c, pv, t0 + 16 * quad);
            const uint32_t p = seen ? pv : 0, q = page_of.seen(c, pk, t0 + (col >> 2) * 16) ? pk : 0;
            const int8_t* kp = c.k + ((uint64_t)q * page_bytes + (k_lane + in * c.dp));
            const int8_t* vp = c.v + ((uint64_t)p * page_bytes + (v_lane + in));
#pragma unroll
            for (int d = 0; d < DN; d++) {
                kw[d] = *reinterpret_cast<const u32x4*>(kp + 64 * d);
                vw[d] = *reinterpret_cast<const u32x4*>(vp + 16 * d * c.page);
            }
            const uint32_t at = p * c.heads + kv;
            ks = c.k_scale[at];
            vs = c.v_scale[at];
        };
        auto put = [&](int buffer) {
            half8v* to = tiles + buffer * FRAGS * 64 + lane;
#pragma unroll
            for (int d = 0; d < DN; d++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    to[((wave * DN + d) * 2 + h) * 64] = codes8(kw[d][2 * h], kw[d][2 * h + 1]);
                    to[(8 * DN + (wave * DN + d) * 2 + h) * 64] = codes8(vw[d][2 * h], vw[d][2 * h + 1]);
                }
        };
        int pk = page_of(first * 64 + (col >> 2) * 16), pv = page_of(first * 64 + quad * 16);
        __syncthreads();  // nobody reads the buffers of the rows before any more
        if (first < last) {
            fetch(first, pk, pv);
            pk = page_of(first * 64 + 64u + (col >> 2) * 16);
            pv = page_of(first * 64 + 64u + quad * 16);
            put(0);
        }
        __syncthreads();
        for (int tile = first, buffer = 0; tile < last; tile++, buffer ^= 1) {
            const int t0 = tile * 64;
            const float fs = ks, fvs = vs;
            const bool there = seen;
            const bool whole = t0 <= all_hi - 64 && t0 >= all_lo && __all(there);
            // (past the last tile: of the last token's page, for nobody)
            fetch(tile + 1, pk, pv);
            pk = page_of(t0 + 128u + (col >> 2) * 16);
            pv = page_of(t0 + 128u + quad * 16);
            const half8v* from = tiles + buffer * FRAGS * 64 + lane;

            const ValueScale scales = value_scale<SPLIT>(fvs);

            // four fragments ahead of the products that take them, sums that depend on each other 8 products apart
            half8v frag[2][4];
            auto keys = [&](int to, int k) {
#pragma unroll
                for (int j = 0; j < 4; j++) frag[to][j] = from[(j * 2 * DN + k) * 64];
            };
            auto values = [&](int to, int at) {
#pragma unroll
                for (int k = 0; k < 4; k++) frag[to][k] = from[(8 * DN + 4 * at + k) * 64];
            };
            __builtin_amdgcn_s_setprio(1);  // the other workgroup's wave has the vector unit meanwhile
            float4v s[CT][4];
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[ct][j] = (float4v){0, 0, 0, 0};
            keys(0, 0);
#pragma unroll
            for (int k = 0; k < 2 * DN; k++) {
                if (k + 1 < 2 * DN) keys((k + 1) & 1, k + 1); else values((k + 1) & 1, 0);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) s[ct][j] = mfma(frag[k & 1][j], q[ct][k >> 1][k & 1], s[ct][j]);
                if constexpr (SPLIT) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) s[ct][j] = mfma(frag[k & 1][j], ql[ct][k >> 1][k & 1], s[ct][j]);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 4 * CT * (SPLIT ? 2 : 1), 0);
            }
            __builtin_amdgcn_s_setprio(0);
            half8v p[CT][2], pl[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                Factor fk = times<SPLIT>(factor[ct], fs);
                ValueScale v = scales;
                if (!whole) mask_scores(s[ct], fk, v, t0 + 16 * quad, there, g.window, hi[ct]);
                weights_of<SPLIT>(s[ct], fk, v, m[ct], l[ct], o[ct], p[ct], pl[ct]);
            }
            put(buffer ^ 1);
#pragma unroll
            for (int j = 0; j < 2 * DN; j++) {
                if (j + 1 < 2 * DN) values((j + 1) & 1, j + 1);
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++)
                            o[ct][2 * j + e] = mfma(frag[j & 1][2 * e + h], p[ct][h], o[ct][2 * j + e]);
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int e = 0; e < 2; e++)
#pragma unroll
                            for (int ct = 0; ct < CT; ct++)
                                o[ct][2 * j + e] = mfma(frag[j & 1][2 * e + h], pl[ct][h], o[ct][2 * j + e]);
                    }
                }
            }
            __syncthreads();
        }

#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            l[ct] += __shfl_xor(l[ct], 16);
            l[ct] += __shfl_xor(l[ct], 32);
            const int row = row0 + 16 * ct + col, i = row / g.group;
            if (f.many.splits > 1 && split == 0 && row < rows && quad == 0)
                f.parts[(long)(sp.start + i) * g.q.heads + kv * g.group + row - i * g.group] = make_int2(0, ns);
            store_row<T, DN>(f, sp, kv, row, rows, ns > 1, f.many_at(split, sp.start + i, kv * g.group + row - i * g.group), m[ct],
                             l[ct], o[ct]);
        }
    }
}

// The other kernel's workgroups come last in the same launch: they are there while the tiled ones run out.
template <class T, int DN>
__global__ __launch_bounds__(256, 2) void attn_many_kernel(Work f, int tiled) {
    extern __shared__ __align__(16) half8v shared[];
    if ((int)blockIdx.x < tiled)
        many_rows<T, DN>(f, blockIdx.x, shared);
    else
        few_rows<T, DN, (DN <= 2 ? 2 : 1)>(f, blockIdx.x - tiled, shared);
}

// Joins what several waves or workgroups hold of a row, in their order: W waves
// a row and q head, 16 DN lanes x 4 dims a part, 4 W / DN parts at a time; then
// those sets' sums, all with maxima of their own.  One wave does for a batch,
// whose heads are split in few parts; of one long sequence there are hundreds.
// The rows: ROWS all of them, FEW up to each_n of each request, MANY as FEW, of
// the other kernel's.
//
// It reads the parts (512 bytes each at 128 dims) after where they are, two loads
// that wait for each other: the 64 rows of one long sequence, in 128 parts, 4.3
// us; 64 sequences' 2048 rows 4.8.
enum class Join { ROWS, FEW, MANY };
template <class T, int DN, int W>
__global__ __launch_bounds__(512) void attn_join_kernel(Work f, int rows_of_group, int each_n, Join which) {
    constexpr int G = W == 1 ? 4 / DN : 32 / DN;  // groups of 16 DN lanes
    constexpr int LANES = W == 1 ? 64 : 512, SETS = 512 / LANES;
    constexpr int LOADS = W == 1 ? 2 : 8;  // parts on their way at a time: where rows are many, waves do that
    __shared__ float4 part[SETS][G][16 * DN];
    __shared__ float2 stats[SETS][G];
    const AttnArgs& g = f.a;
    const int set = W == 1 ? threadIdx.x >> 6 : 0, tid = threadIdx.x & (LANES - 1);
    long b = (long)blockIdx.x * SETS + set;
    const int h = (int)(b % g.q.heads);
    b /= g.q.heads;
    int t = (int)b, to = min(t + 1, g.tokens), step_t = 1;
    if (which != Join::ROWS) {
        const int r = (int)(b / each_n);
        t = to = 0;
        if (r < g.requests) {
            const int start = row_bound(g, r), n = row_bound(g, r + 1) - start;
            if ((which == Join::MANY) == (n * g.group > f.most)) {
                t = start + (int)(b % each_n);
                to = start + n;
            }
        }
        step_t = each_n;
    }
    const int group = tid / (16 * DN), piece = tid % (16 * DN);
    for (; t < to; t += step_t) {
        const int2 of = f.parts[(long)t * g.q.heads + h];
        const int ns = of.y;
        if (ns <= 1 || ns > f.most_parts) continue;
        // the place of the first part, of the second, and on from there
        const long at0 = which == Join::MANY ? f.many_at(0, t, h) : of.x;
        const long at = which == Join::MANY ? f.many_at(1, t, h) : at0 + rows_of_group;
        const long step = which == Join::MANY ? at - at0 : 2l * rows_of_group;
        float top = kNone, l = 0.0f;
        float4 sum = make_float4(0, 0, 0, 0);
        if (group < G) {
            for (int s = group; s < ns; s += LOADS * G) {
                float2 st[LOADS];
                float4 x[LOADS];
#pragma unroll
                for (int e = 0; e < LOADS; e++) {
                    const int k = s + e * G;
                    const long place = k ? at + (long)(k - 1) * step : at0;
                    st[e] = make_float2(kNone, 0.0f);
                    x[e] = make_float4(0, 0, 0, 0);
                    if (k < ns && place >= 0 && place < f.places) {  // (a starts' array out of order may lead past them)
                        st[e] = f.stat[place];
                        x[e] = reinterpret_cast<const float4*>(f.part + place * g.c.dp)[piece];
                    }
                }
                float m = top;
#pragma unroll
                for (int e = 0; e < LOADS; e++) m = fmaxf(m, st[e].x);
                const float base = m == kNone ? 0.0f : m, old = __builtin_amdgcn_exp2f(top - base);
                top = m;
                l *= old;
                sum.x *= old;
                sum.y *= old;
                sum.z *= old;
                sum.w *= old;
#pragma unroll
                for (int e = 0; e < LOADS; e++) {
                    const float w = __builtin_amdgcn_exp2f(st[e].x - base);
                    l += st[e].y * w;
                    sum.x += x[e].x * w;
                    sum.y += x[e].y * w;
                    sum.z += x[e].z * w;
                    sum.w += x[e].w * w;
                }
            }
            part[set][group][piece] = sum;
            if (piece == 0) stats[set][group] = make_float2(top, l);
        }
        if (W > 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        if (tid < 16 * DN) {
            top = kNone;
            for (int k = 0; k < G; k++) top = fmaxf(top, stats[set][k].x);
            const float base = top == kNone ? 0.0f : top;
            l = 0.0f;
            sum = make_float4(0, 0, 0, 0);
            for (int k = 0; k < G; k++) {
                const float4 x = part[set][k][piece];
                const float w = __builtin_amdgcn_exp2f(stats[set][k].x - base);
                l += stats[set][k].y * w;
                sum.x += x.x * w;
                sum.y += x.y * w;
                sum.z += x.z * w;
                sum.w += x.w * w;
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            store4<T>((T*)g.out.p + (long)t * g.out.token + (long)h * g.out.head, 4 * piece, g.c.dim, f.vec,
                      {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv});
        }
        if (W > 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
}

}  // namespace zt

using namespace zt;

static bool attn_ok(const zt_kv8_attn* a) {
    return a && kv8_ok(a->cache) && type_ok(a->type) && a->reserved == 0 && a->requests >= 0 && a->width >= 1 &&
           a->tokens >= 0 && a->max_q >= 0 && a->max_kv >= 0 && a->window >= 0 && a->q.heads >= 1 &&
           a->q.heads == a->out.heads && a->q.heads % a->cache.kv_heads == 0 && a->q.heads <= 1 << 16 &&
           (long)a->tokens * a->q.heads < (1l << 31) - 256 && (long)a->requests * a->width < (1l << 31);
}

// How a call is launched.
struct AttnPlan {
    int ct;  // column tiles of a wave of the few kernel
    int most, shares, qtiles, empties;
    int few_n, many_n;  // bounds of the tokens of one request
    bool single, wide;
    Split many;
    long others;
    long part, stat, parts;  // bytes of the parts' sums, and of where they are
    long places;
};

static AttnPlan attn_plan(const zt_kv8_attn* a) {
    AttnPlan p{};
    const int group = a->q.heads / a->cache.kv_heads, dp = (a->cache.head_dim + 63) & ~63;
    const long requests = std::max(1, a->requests), heads = a->cache.kv_heads;
    const long most = (long)std::min(a->max_q, a->tokens) * group;
    // up to 64 rows by the few kernel: 32 requests of 3000 tokens, 64 rows 88 us, by the other 97; 128 rows 124 and 103
    p.most = most <= 64 ? 0x7FFFFFFF : 64;
    // of more than 16 rows two columns of them share what is read of a tile (those requests, 32 rows: 66 us, one by one
    // 80); past 128 dims their sums would leave no registers
    p.ct = most > 16 && dp <= 128 ? 2 : 1;
    long kv = std::min((long)a->max_kv, (long)a->width * a->cache.page_tokens);
    if (a->window > 0) kv = std::min(kv, (long)a->window + a->max_q + 63);
    const long tiles = std::max(1l, (kv + 63) / 64);
    // A tile each as far as the bounds go, up to a wave for each SIMD: fewer leave some without work, each more makes
    // parts to be joined (one sequence of 40011 tokens 25.4 us, with 512 29.7, with 2048 28.1; 64 of up to 8000 69, 95
    // and 73).
    const long groups = (std::max(1l, std::min(most, 64l)) + 16 * p.ct - 1) / (16 * p.ct);
    p.single = tiles <= 2;
    p.shares = (int)std::min(1024l, requests * heads * groups * (p.single ? 1 : tiles + kBegin));
    // eight waves to join a row of more than 16 parts (one sequence of 40011 tokens, 128 parts: 25 us, with one 39), else
    // one (64 sequences 70 us, with eight 81)
    p.wide = p.shares > 16 * requests * heads * groups;
    // Any row may be of no request (a batch padded to a graph's size): a workgroup zeroes one in 0.3 us (8 heads, group
    // 4), so one for 16 rows, up to about the card's 1024 in all (4096 padded rows 50 us, by one a head 1210).
    p.empties = (int)std::max(1l, std::min({(a->tokens + 15) / 16l, 64l, 1024 / heads}));
    p.others = 2l * p.shares * 16 * p.ct;
    p.many_n = std::max(1, std::min(a->max_q, a->tokens));
    p.few_n = std::max(1, std::min(p.many_n, 64 / group));
    p.many = {1, 1};
    if (most > 64) {
        p.qtiles = ceil_div(most, dp <= 128 ? 128 : 64);
        // Along the tokens where that is less time: a tile of 128 rows and dims is 2.2 us while the card's 512 workgroups
        // are not passed, the parts are written and read at 4.5 TB/s, a launch 4 us.  (32 heads over 8 of 128, fp16, one
        // sequence: 100 tokens onto 4000 41 us in 16 splits, 120 whole; 1000 onto 4000 127 in two, 150 whole; 700 from
        // the beginning 40 in two, 32 whole.)
        const long have = requests * heads * p.qtiles;
        const double tile = 2.2 * dp / (dp <= 128 ? 128 : 256), part = 8.0 * a->tokens * a->q.heads * dp / 4.5e6;
        long splits = 1;
        double least = 0;
        for (long s = 1; s <= std::max(1l, std::min(512 / have, tiles / 4)); s++) {
            const double us = (double)((tiles + s - 1) / s) * tile + (s > 1 ? 4 + s * part : 0);
            if (s == 1 || us < least) {
                least = us;
                splits = s;
            }
        }
        p.many.tiles = (int)((tiles + splits - 1) / splits);
        p.many.splits = (int)((tiles + p.many.tiles - 1) / p.many.tiles);
    }
    const long all = p.others + (p.many.splits > 1 ? (long)p.many.splits * a->tokens * a->q.heads : 0);
    p.stat = (all * 8 + 15) & ~15l;
    p.part = all * dp * 4;
    p.places = all;
    p.parts = ((long)a->tokens * a->q.heads * 8 + 15) & ~15l;
    return p;
}

template <class T, int DN>
static int launch(const Work& f, const AttnPlan& p, hipStream_t stream) {
    const long tiled = (long)p.qtiles * p.many.splits * f.a.c.heads * f.a.requests;
    const int few = (f.shares + 3) / 4 + f.a.c.heads * f.empties;
    if (tiled + few >= 1l << 31) return kInvalid;
    constexpr int column = DN * 2 * (sizeof(T) / 2) * 4096;  // LDS of the few kernel, at most 64 KB in all
    if (tiled) {
        static std::atomic<uint64_t> raised{0};
        constexpr int lds = 2 * 16 * DN * 1024;
        static_assert(lds >= column * (DN <= 2 ? 2 : 1));
        if constexpr (lds > 65536) {
            const hipError_t rc = raise_lds((const void*)attn_many_kernel<T, DN>, lds, raised);
            if (rc != hipSuccess) return (int)rc;
        }
        attn_many_kernel<T, DN><<<(unsigned)(tiled + few), 256, lds, stream>>>(f, (int)tiled);
    } else if (p.ct == 2) {
        if constexpr (DN <= 2) attn_few_kernel<T, DN, 2><<<few, 256, 2 * column, stream>>>(f);
    } else {
        attn_few_kernel<T, DN, 1><<<few, 256, column, stream>>>(f);
    }
    const auto join = [&](Join which, int each, bool wide) {
        each = (int)std::min((long)each, std::max(1l, ((1l << 31) - 1) / (std::max(1l, (long)f.a.requests) * f.a.q.heads)));
        const long rows = which == Join::ROWS ? (long)f.a.tokens * f.a.q.heads : (long)f.a.requests * each * f.a.q.heads;
        if (wide)
            attn_join_kernel<T, DN, 8><<<(unsigned)rows, 512, 0, stream>>>(f, 16 * p.ct, each, which);
        else
            attn_join_kernel<T, DN, 1><<<(unsigned)((rows + 7) / 8), 512, 0, stream>>>(f, 16 * p.ct, each, which);
    };
    if (f.a.requests && !p.single) join(p.qtiles ? Join::FEW : Join::ROWS, p.few_n, p.wide);
    if (f.a.requests && p.many.splits > 1) join(Join::MANY, p.many_n, false);
    return (int)hipGetLastError();
}

ZT_EXPORT long zt_kv8_attention_workspace_bytes(const zt_kv8_attn* a) {
    if (!attn_ok(a)) return -1;
    const AttnPlan p = attn_plan(a);
    return p.part + p.stat + p.parts;
}

ZT_EXPORT int zt_kv8_attention(const zt_kv8_attn* a, void* workspace, long workspace_bytes, zt_stream_t stream) {
    if (!attn_ok(a)) return kInvalid;
    if (a->tokens == 0) return 0;
    if (!rows_ok(a->q, a->type) || !rows_ok(a->out, a->type) || !a->q_start ||
        (a->requests && (!a->table || !a->kv_lens)) ||
        (((uintptr_t)a->table | (uintptr_t)a->kv_lens | (uintptr_t)a->q_start | (uintptr_t)a->scale) & 3))
        return kInvalid;
    const AttnPlan p = attn_plan(a);
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.part + p.stat + p.parts) return kInvalid;
    const double unit = 1.44269504088896340736 / std::sqrt((double)a->cache.head_dim);
    const AttnArgs g{kv8_of(a->cache), rows_of(a->q), rows_of(a->out), a->table, a->kv_lens, a->q_start, a->scale,
                     a->requests,      a->width,      a->tokens,       a->window, a->q.heads / a->cache.kv_heads,
                     (float)unit,      (float)(unit - (double)(float)unit)};
    const Work f{g,        p.most, p.shares, p.empties, p.single, p.many, p.qtiles, rows_vector(a->q, 4, a->type) && rows_vector(a->out, 4, a->type),
                 p.others, p.places, std::max(p.shares, p.many.splits), (float*)workspace, (float2*)((char*)workspace + p.part),
                 (int2*)((char*)workspace + p.part + p.stat)};
    const bool f32 = a->type == ZT_F32;
    switch (g.c.dp) {
        case 64: return f32 ? launch<float, 1>(f, p, stream) : launch<_Float16, 1>(f, p, stream);
        case 128: return f32 ? launch<float, 2>(f, p, stream) : launch<_Float16, 2>(f, p, stream);
        case 192: return f32 ? launch<float, 3>(f, p, stream) : launch<_Float16, 3>(f, p, stream);
        default: return f32 ? launch<float, 4>(f, p, stream) : launch<_Float16, 4>(f, p, stream);
    }
}
