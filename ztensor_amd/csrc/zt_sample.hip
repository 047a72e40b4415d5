// A token from the logits: temperature, top-k, top-p, min-p, given uniforms.
#include <algorithm>

#include "zt_kv8.h"

namespace zt {

constexpr int kSampleThreads = 1024;

struct SampleArgs {
    const void* logits;
    long row_stride;
    int rows, vocab;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    long* token;
    float* logprob;
};

// fp32 as unsigned whole numbers of the same order; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}

template <class T>
__device__ __forceinline__ float logit(const T* row, int i) {
    const float z = (float)row[i];
    return z != z ? -__builtin_inff() : z;
}

// Weights of a row: its largest value, the temperature, and 1 / temperature
// rounded to nearest (0: divide).
struct Scores {
    float top, temperature, by;
    __device__ __forceinline__ Scores(float top_, float t) : top(top_), temperature(t), by(t > 1e-30f && t < 1e30f ? 1.0f / t : 0.0f) {}
    // (z - top) / temperature, rounded to nearest: a quotient from the rounded
    // reciprocal and one correction by its remainder is the rounded one
    // (Markstein), where nothing over- or underflows: below -80 it is divided, and
    // what is tiny has the exponential 1 whatever its last bit.
    __device__ __forceinline__ float quotient(float z) const {
#pragma clang fp contract(off)
        const float a = z - top, q = a * by;
        if (__builtin_expect(!(q > -80.0f) || by == 0.0f, 0)) return a / temperature;
        return __builtin_fmaf(__builtin_fmaf(-q, temperature, a), by, q);
    }
    // exp of it, and that in units of 2^-40
    __device__ __forceinline__ uint64_t weight(float z, float& w) const {
        w = z == top ? 1.0f : expf(quotient(z));
        const float x = w * 256.0f;  // kFix = 2^8 2^32: the whole part, then 32 bits more, all exact
        const uint32_t hi = (uint32_t)x, lo = (uint32_t)((x - (float)hi) * 4294967296.0f);
        return (uint64_t)hi << 32 | lo;
    }
    __device__ __forceinline__ uint64_t weight(float z) const {
        float w;
        return weight(z, w);
    }
};

struct Scan {
    uint64_t part[kSampleThreads / 64];
};

// x + (x of the lane that a DPP move takes it from; 0 where none)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t add_moved(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, true);
    return x + ((uint64_t)hi << 32 | lo);
}

// Running sums in the order of the threads: v becomes the sum before the
// thread's own, the result is the sum of all.  In a wave by moves of 1, 2, 4 and
// 8 lanes in rows of 16, then each row's last to the rows after it; across the
// 16 waves every thread adds up the waves' sums.
__device__ __forceinline__ uint64_t block_scan(uint64_t& v, Scan& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t x = v;
    x = add_moved<0x111, 0xF>(x);
    x = add_moved<0x112, 0xF>(x);
    x = add_moved<0x114, 0xF>(x);
    x = add_moved<0x118, 0xF>(x);
    x = add_moved<0x142, 0xA>(x);  // lanes 15 and 47 to the next row
    x = add_moved<0x143, 0xC>(x);  // lane 31 to the upper two
    __syncthreads();
    if (lane == 63) s.part[wave] = x;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSampleThreads / 64; i++) {
        const uint64_t p = s.part[i];
        before += i < wave ? p : 0;
        all += p;
    }
    v = before + x - v;
    return all;
}

struct Prefix {
    uint32_t key;    // tokens of a larger key are in
    int equal;       // and so many of this key, by index
    uint64_t mass;   // of all of them
};

// A row's settings, those that are not numbers or out of range as off.
struct Settings {
    float temperature, top_p, min_p;
    uint64_t k;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& g, int b) {
    // loads without branches, all on their way at once: of an array that is not there, u's in its place
    const float* none = g.u + b;
    const float t = *(g.temperature ? g.temperature + b : none), p = *(g.top_p ? g.top_p + b : none);
    const float m = *(g.min_p ? g.min_p + b : none);
    const int k = *(g.top_k ? g.top_k + b : (const int*)none);
    Settings s;
    s.temperature = g.temperature ? t : 1.0f;
    const bool greedy = !(s.temperature > 0.0f);
    if (greedy) s.temperature = 1.0f;
    s.k = greedy ? 1 : !g.top_k || k <= 0 || k > g.vocab ? g.vocab : k;
    s.top_p = g.top_p && p < 1.0f ? p : 1.0f;
    s.min_p = g.min_p && m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    return s;
}

// The weight that the kept tokens before the last have to reach: at least 1.
__device__ __forceinline__ uint64_t goal_of(float top_p, uint64_t mass) {
    const double d = ceil((double)top_p * (double)mass);
    return d > 1.0 ? (uint64_t)d : 1;
}

// Where in the kept weights the uniform falls.
__device__ __forceinline__ uint64_t aim_of(float u, uint64_t mass) {
    const uint64_t x = (uint64_t)fmax(0.0, (double)u * (double)mass);
    return x < mass ? x : mass - 1;
}

struct Digits {
    unsigned counts[256];
    unsigned long long masses[256];
    Prefix found;
};

// A whole row by one workgroup, which reads it again in every pass: two radix
// selections of 8 bits a pass, one by number and one by weight.  Slow, and for
// every row: those with more tokens in one bin than the list below has room for.
template <class T>
__device__ __forceinline__ void sample_row(const SampleArgs& g, int b, const Scores& sc, const Settings& st, Scan& scan, Digits& dg) {
    const int tid = threadIdx.x, V = g.vocab;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    uint64_t want = st.k;  // the weights fall with the logits: those of min_p or more are the first so many, too
    if (st.min_p > 0.0f) {
        uint64_t n = 0;
        for (int i = tid; i < V; i += kSampleThreads) {
            float w;
            sc.weight(logit(row, i), w);
            n += !(w < st.min_p);
        }
        const uint64_t all = block_scan(n, scan);
        want = min(want, all);
    }
    // the least prefix of at least `want` tokens, then of at least `goal` weight
    Prefix p{0, 0, 0};
    for (int by_mass = 0; by_mass < 2; by_mass++) {
        uint64_t goal = want;
        if (by_mass) {
            if (st.top_p == 1.0f) break;
            goal = goal_of(st.top_p, p.mass);
            if (goal >= p.mass) break;
        }
        uint32_t prefix = 0;
        uint64_t cnt = 0, mass = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) {
                dg.counts[tid] = 0;
                dg.masses[tid] = 0;
            }
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const float z = logit(row, i);
                const uint32_t key = key_of(z);
                if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                const uint64_t f = sc.weight(z);
                atomicAdd(&dg.counts[(key >> shift) & 255], 1u);
                atomicAdd(&dg.masses[(key >> shift) & 255], (unsigned long long)f);
            }
            __syncthreads();
            int d = 255;  // every thread walks down the digits
            for (; d > 0; d--) {
                if ((by_mass ? mass + dg.masses[d] : cnt + dg.counts[d]) >= goal) break;
                mass += dg.masses[d];
                cnt += dg.counts[d];
            }
            prefix |= (uint32_t)d << shift;
            if (shift == 0 && tid == 0) {
                const uint64_t each = dg.counts[d] ? dg.masses[d] / dg.counts[d] : 0;  // equal keys weigh the same
                uint64_t e = by_mass ? (each ? (goal - mass + each - 1) / each : dg.counts[d]) : goal - cnt;
                e = min(max(e, (uint64_t)1), (uint64_t)dg.counts[d]);
                dg.found = {prefix, (int)e, mass + e * each};
            }
        }
        __syncthreads();
        p = dg.found;
    }
    // the token: runs of 1024 in order of the index
    const uint64_t aim = aim_of(g.u[b], p.mass);
    uint64_t done = 0, equal = 0;
    for (int i0 = 0; i0 < V; i0 += kSampleThreads) {
        const int i = i0 + tid;
        const float z = i < V ? logit(row, i) : -__builtin_inff();
        const uint32_t key = key_of(z);
        const bool own = i < V && key == p.key;
        uint64_t same = own;
        const uint64_t sames = block_scan(same, scan);
        const uint64_t f = i < V && (key > p.key || (own && equal + same < (uint64_t)p.equal)) ? sc.weight(z) : 0;
        uint64_t before = f;
        const uint64_t all = block_scan(before, scan);
        if (f && done + before <= aim && aim < done + before + f) {
            g.token[b] = i;
            g.logprob[b] = (float)log((double)f / (double)p.mass);
        }
        done += all;
        equal += sames;
        if (done > aim) break;
    }
}

// ---------------------------------------------------------- rows in four steps

// A row is split among workgroups: (1) its largest and smallest value, and the
// largest of up to 4096 groups of its tokens; (2) how many tokens, or what
// weight of them, as its cuts need it, are in each of 1024 bins of (top - z);
// (3) the bins in which the cuts fall are known, so each workgroup sums up what
// is certainly kept of its part and lists the tokens of these bins; (4) one
// workgroup sorts the listed ones and picks the token.  A small top-k needs no
// bins of all tokens: those of k groups' largest values and above hold at least
// k tokens, and few more.  Every sum is of whole numbers, so the order of the
// atomics leaves no trace.
//
// The logits are read three times, from the Infinity Cache after the first: 128
// rows of 100003 fp32 (51 MB) take 10.4 us in (1), the rate of a copy, 16.6 in
// (2), bound by LDS atomics and exponentials, 24 in (3), 5 of them until its cuts
// are known, and 20 in (4), most of it the sort of up to 2048 tokens; (4) keeps 6
// registers in memory.  One row, 50 tokens to sort: 3.5, 2.5, 8.5 and 8.1 us,
// chains of a few loads, sums over a workgroup, and launches.
constexpr int kBins = kSampleThreads;
constexpr int kSplits = 64;    // most workgroups of a row
constexpr int kWaves = kSampleThreads / 64;
constexpr int kParts = kSplits * kWaves;  // its parts: neighbours, one wave's
constexpr int kListed = 2048;
constexpr float kSpan = 27.8f;  // past it a weight is below 2^-40: exp(-27.73)

// Where the cuts fall.
struct Cut {
    uint64_t n, before;  // tokens that stay by number; those in the bins before bin0
    uint64_t whole;      // the weight of the first n, where there is no need to rank for it
    int bin0, bin1;      // the bins in which the n-th token is looked for; bin0 > bin1: it ends bin1
    int lo, hi;          // those in which the last kept token is; lo > hi: it ends bin hi
};

struct RowWork {
    unsigned long long mass[kBins];
    unsigned long long list[kListed];  // key and, falling, index: the order of the tokens
    unsigned long long sure[kParts];   // weight of a part's tokens in the bins before the cut
    Cut cut;
    float top[kSplits], low[kSplits];
    unsigned count[kBins];
    unsigned listed, spare;
};

// How the rows are split, and where what their workgroups leave lies.
struct Parts {
    RowWork* work;
    float* tops;  // [rows][groups]
    int splits, part, seg;
    int lanes;    // of a group
    int groups;   // of a row
};

// What a row's cuts need.
struct Needs {
    bool few;      // the first k are listed, all of them
    bool counted;  // the bins' numbers, for a larger k
    bool weighed;  // the bins' weights, for a cut by weight
};
__device__ __forceinline__ Needs needs_of(const SampleArgs& g, const Parts& w, const Settings& st) {
    Needs n;
    n.few = g.vocab <= kListed || st.k <= (uint64_t)min(kListed / 2, w.groups / 4);
    n.counted = !n.few && st.k < (uint64_t)g.vocab;
    n.weighed = !n.few && st.top_p < 1.0f;
    return n;
}

__device__ __forceinline__ unsigned long long order_of(uint32_t key, int i) {
    return (unsigned long long)key << 32 | (0xFFFFFFFFu - (unsigned)i);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

// The bins of a row: by its largest value, the scale that spreads what has a
// weight over all of them.
struct Bins {
    float top, by;
    __device__ __forceinline__ int of(float z) const {
        const float d = z == top ? 0.0f : top - z;  // falls as z grows
        return (int)fminf(d * by, (float)(kBins - 1));  // (inf * 0, -inf beside values all alike: the last)
    }
};

__device__ __forceinline__ Bins bins_of(const RowWork& w, int splits, float temperature) {
    float top = -__builtin_inff(), low = __builtin_inff();
    const int lane = threadIdx.x & 63;
    if (lane < splits) {
        top = w.top[lane];
        low = w.low[lane];
    }
    top = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(top))))));
    low = -max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(-low))))));
    const float span = fminf(kSpan * temperature, top - low);
    return {top, span > 0.0f ? (float)kBins / span : 0.0f};
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_top_kernel(SampleArgs g, Parts parts) {
    __shared__ float tops[kSampleThreads / 64], lows[kSampleThreads / 64];
    const int splits = parts.splits, part = parts.part;
    const int b = blockIdx.x / splits, s = blockIdx.x - b * splits, tid = threadIdx.x;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    float top = -__builtin_inff(), low = __builtin_inff();
    const int to = min(g.vocab, (s + 1) * part);
#pragma unroll 4
    for (int i = s * part + tid; i < to; i += kSampleThreads) {
        const float z = logit(row, i);
        top = fmaxf(top, z);
        low = fminf(low, z > -__builtin_inff() ? z : low);
    }
    {
        // lanes that differ in the upper bits of their number in a row of 16 are a group
        float m = top;
        if (parts.lanes >= 2) m = max_step<8>(m);
        if (parts.lanes >= 4) m = max_step<4>(m);
        if (parts.lanes >= 8) m = max_step<2>(m);
        if (parts.lanes >= 16) m = max_step<1>(m);
        const int each = 16 / parts.lanes, in = tid & 15;
        if (in < each) parts.tops[(long)b * parts.groups + s * (kSampleThreads / parts.lanes) + (tid >> 4) * each + in] = m;
    }
    top = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(top))))));
    low = -max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(-low))))));
    if ((tid & 63) == 0) {
        tops[tid >> 6] = top;
        lows[tid >> 6] = low;
    }
    RowWork& w = parts.work[b];
    if (s == 0) {
        w.mass[tid] = 0;
        w.count[tid] = 0;
        if (tid == 0) w.listed = 0;
    }
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSampleThreads / 64; i++) {
            top = fmaxf(top, tops[i]);
            low = fminf(low, lows[i]);
        }
        w.top[s] = top;
        w.low[s] = low;
    }
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs g, Parts parts) {
    __shared__ unsigned long long mass[kBins];
    __shared__ unsigned count[kBins];
    const int splits = parts.splits, part = parts.part;
    const int b = blockIdx.x / splits, s = blockIdx.x - b * splits, tid = threadIdx.x;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    RowWork& w = parts.work[b];
    const Settings st = settings_of(g, b);
    const Bins bins = bins_of(w, splits, st.temperature);
    if (!(bins.top > -__builtin_inff())) return;
    const Needs need = needs_of(g, parts, st);
    if (!need.counted && !need.weighed) return;
    mass[tid] = 0;
    count[tid] = 0;
    __syncthreads();
    const int to = min(g.vocab, (s + 1) * part);
    const Scores sc(bins.top, st.temperature);
    constexpr int kAhead = 4;
    for (int i0 = s * part + tid; i0 < to; i0 += kSampleThreads * kAhead) {
        float z[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) z[k] = logit(row, min(i0 + kSampleThreads * k, to - 1));
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            if (i0 + kSampleThreads * k >= to) continue;
            const int bin = bins.of(z[k]);
            if (need.counted) atomicAdd(&count[bin], 1u);
            if (need.weighed) {
                float x;
                const uint64_t f = sc.weight(z[k], x);
                if (f && x >= st.min_p) atomicAdd(&mass[bin], (unsigned long long)f);
            }
        }
    }
    __syncthreads();
    if (count[tid]) atomicAdd(&w.count[tid], count[tid]);
    if (mass[tid]) atomicAdd(&w.mass[tid], mass[tid]);
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_list_kernel(SampleArgs g, Parts parts) {
    __shared__ Scan scan;
    __shared__ Cut cut;
    __shared__ unsigned long long list[kListed];
    __shared__ unsigned listed, at;
    const int splits = parts.splits, part = parts.part;
    const int b = blockIdx.x / splits, s = blockIdx.x - b * splits, tid = threadIdx.x;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    RowWork& w = parts.work[b];
    const Settings st = settings_of(g, b);
    const Bins bins = bins_of(w, splits, st.temperature);
    if (!(bins.top > -__builtin_inff())) return;
    const Needs need = needs_of(g, parts, st);

    if (tid == 0) {
        cut = {st.k, 0, 0, kBins, kBins - 1, kBins, kBins - 1};  // all stay
        if (need.few) cut = {st.k, 0, 0, 0, kBins - 1, 0, kBins - 1};
        listed = 0;
    }
    __syncthreads();
    uint64_t own_f = 0, f0 = 0;
    if (need.few && g.vocab > kListed) {
        // the bins from which the k-th of the groups' largest values is up hold k tokens or more
        __shared__ unsigned count[kBins];
        count[tid] = 0;
        __syncthreads();
        for (int i = tid; i < parts.groups; i += kSampleThreads)
            atomicAdd(&count[bins.of(parts.tops[(long)b * parts.groups + i])], 1u);
        __syncthreads();
        const uint64_t own_n = count[tid];
        uint64_t n0 = own_n;
        block_scan(n0, scan);
        if (n0 < st.k && st.k <= n0 + own_n) cut.bin1 = cut.hi = tid;
    }
    if (need.weighed) {
        own_f = f0 = w.mass[tid];
        const uint64_t all = block_scan(f0, scan);
        if (tid == 0) cut.whole = all;
    }
    if (need.counted) {
        const uint64_t own_n = w.count[tid];
        uint64_t n0 = own_n;
        block_scan(n0, scan);
        if (n0 < st.k && st.k <= n0 + own_n) {
            const bool inside = st.k < n0 + own_n && (!need.weighed || own_f);  // tokens without weight need no ranks
            cut.before = n0;
            cut.whole = f0 + own_f;
            cut.bin1 = cut.hi = tid;
            cut.bin0 = cut.lo = inside ? tid : tid + 1;
        }
    }
    __syncthreads();
    if (need.weighed) {
        // the weight of the first n is between that of the bins before bin1 and that with it
        const int bin1 = cut.bin1;
        const bool inside = cut.bin0 <= bin1;
        const uint64_t whole = cut.whole, less = inside ? w.mass[bin1] : 0;
        const uint64_t from = goal_of(st.top_p, whole - less), upto = goal_of(st.top_p, whole);
        __syncthreads();
        if (f0 < from && from <= f0 + own_f) cut.lo = tid;
        if (f0 < upto && upto <= f0 + own_f) cut.hi = tid;
        __syncthreads();
    }
    const int lo = cut.lo, hi = cut.hi, bin0 = cut.bin0, bin1 = cut.bin1;
    if (s == 0 && tid == 0) w.cut = cut;

    // each wave its part
    const Scores sc(bins.top, st.temperature);
    const int wave = tid >> 6, from = s * part + wave * parts.seg, to = min(g.vocab, from + parts.seg);
    uint64_t sure = 0;
    constexpr int kAhead = 8;  // values on their way at a time
    for (int i0 = from + (tid & 63); i0 < to; i0 += 64 * kAhead) {
        float z[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) z[k] = logit(row, min(i0 + 64 * k, to - 1));
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + 64 * k, bin = bins.of(z[k]);
            const bool counts = bin < lo, ranks = (bin >= lo && bin <= hi) || (bin >= bin0 && bin <= bin1);
            if (i >= to || !(counts || ranks)) continue;
            float x;
            const uint64_t f = sc.weight(z[k], x);
            sure += counts && x >= st.min_p ? f : 0;
            if (ranks && f) {  // tokens without weight are the last in any order
                const unsigned n = atomicAdd(&listed, 1u);
                if (n < kListed) list[n] = order_of(key_of(z[k]), i);
            }
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sure += __shfl_xor(sure, o);
    if ((tid & 63) == 0) w.sure[s * kWaves + wave] = sure;
    __syncthreads();
    const unsigned n = listed;
    if (n == 0) return;
    if (tid == 0) at = atomicAdd(&w.listed, n);
    __syncthreads();
    for (unsigned i = tid; i < min(n, (unsigned)kListed); i += kSampleThreads)
        if (at + i < kListed) w.list[at + i] = list[i];
}

// Falling order of n2 values, a power of two up to 2 kSampleThreads, by compare
// and exchange over strides that halve.  At strides up to 64 a wave's pairs are
// its own 128 values: no barrier between such steps.
__device__ __forceinline__ void sort_falling(unsigned long long* v, int n2) {
    const int t = threadIdx.x;
    for (int size = 2; size <= n2; size <<= 1)
        for (int stride = size >> 1; stride >= 1; stride >>= 1) {
            if (t < n2 / 2) {
                const int i = 2 * t - (t & (stride - 1)), j = i + stride;
                const unsigned long long a = v[i], b = v[j];
                if ((a < b) != ((i & size) != 0)) {
                    v[i] = b;
                    v[j] = a;
                }
            }
            if (stride > 64 || (stride == 1 && (size > 64 || size == n2)))
                __syncthreads();
            else
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_pick_kernel(SampleArgs g, Parts parts) {
    constexpr int kTurns = kListed / kSampleThreads;
    __shared__ Scan scan;
    __shared__ union {
        unsigned long long order[kListed];
        Digits digits;
    } u;
    __shared__ unsigned long long part_mass[kParts], least;
    __shared__ int chosen;
    __shared__ uint64_t chosen_before;
    const int b = blockIdx.x, tid = threadIdx.x, seg = parts.seg;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    const RowWork& w = parts.work[b];
    // everything that may be wanted is on its way before any of it is waited for
    const Cut cut = w.cut;
    const int listed = (int)min(w.listed, 0x7FFFFFFFu);
    const uint64_t sure = tid < parts.splits * kWaves ? w.sure[tid] : 0;
    unsigned long long mine[kTurns];
#pragma unroll
    for (int e = 0; e < kTurns; e++) mine[e] = w.list[tid + e * kSampleThreads];
    const float u01 = g.u[b];
    const Settings st = settings_of(g, b);
    const Bins bins = bins_of(w, parts.splits, st.temperature);
    if (!(bins.top > -__builtin_inff())) {
        if (tid == 0) {
            g.token[b] = -1;
            g.logprob[b] = __builtin_nanf("");
        }
        return;
    }
    const Scores sc(bins.top, st.temperature);
    if (listed > kListed) {
        sample_row<T>(g, b, sc, st, scan, u.digits);
        return;
    }
    part_mass[tid] = sure;
    if (tid == 0) least = ~0ull;
    uint64_t before = sure;
    const uint64_t above = block_scan(before, scan);
    uint64_t total = above;
    if (listed) {
        int n2 = 16;
        while (n2 < listed) n2 *= 2;
#pragma unroll
        for (int e = 0; e < kTurns; e++) {
            const int i = tid + e * kSampleThreads;
            if (i < n2) u.order[i] = i < listed ? mine[e] : 0;
        }
        __syncthreads();
        if (n2 <= 256) {
            // few: each counts those before it, four threads or more for one (128: 1 us less than by exchanges)
            const int each = min(64, kSampleThreads / n2), i = tid / each;
            const unsigned long long o = i < listed ? u.order[i] : 0;
            int rank = 0;
            for (int j = tid & (each - 1); j < n2; j += each) rank += u.order[j] > o;
            for (int x = 1; x < each; x <<= 1) rank += __shfl_xor(rank, x);
            __syncthreads();
            if (i < listed && (tid & (each - 1)) == 0) u.order[rank] = o;
            __syncthreads();
        } else {
            sort_falling(u.order, n2);
        }
        // this thread's tokens, neighbours in that order: their weights, and which cut they are listed for
        uint64_t f[kTurns];
        bool ranked[kTurns], weighed[kTurns], likely[kTurns];
        uint64_t rank = 0, all_f = 0;
#pragma unroll
        for (int e = 0; e < kTurns; e++) {
            const int i = tid * kTurns + e;
            const unsigned long long o = i < listed ? u.order[i] : 0;
            const float z = value_of((uint32_t)(o >> 32));
            const int bin = i < listed ? bins.of(z) : -1;
            ranked[e] = bin >= cut.bin0 && bin <= cut.bin1;
            weighed[e] = bin >= cut.lo && bin <= cut.hi;
            float x = 0.0f;
            f[e] = bin >= 0 ? sc.weight(z, x) : 0;
            likely[e] = x >= st.min_p;
            rank += ranked[e];
        }
        block_scan(rank, scan);
        // of those of bin0 .. bin1 only the first n
        bool in[kTurns];
        uint64_t first = 0;
#pragma unroll
        for (int e = 0; e < kTurns; e++) {
            in[e] = likely[e] && (!ranked[e] || cut.before + rank < cut.n);
            first += ranked[e] && in[e] ? f[e] : 0;
            rank += ranked[e];
            all_f += weighed[e] && in[e] ? f[e] : 0;
        }
        uint64_t goal = ~0ull;
        if (st.top_p < 1.0f) {
            // the weight of the first n
            uint64_t whole = cut.whole;
            first = block_scan(first, scan);
            if (cut.bin0 <= cut.bin1) whole = first + (cut.bin0 == 0 ? 0 : cut.whole - w.mass[cut.bin1]);
            goal = goal_of(st.top_p, whole);
        }
        uint64_t mass = all_f;
        block_scan(mass, scan);
        mass += above;
#pragma unroll
        for (int e = 0; e < kTurns; e++) {
            if (weighed[e] && in[e] && mass < goal) {
                const unsigned long long o = u.order[tid * kTurns + e];
                atomicAdd(&part_mass[(0xFFFFFFFFu - (unsigned)o) / (unsigned)seg], (unsigned long long)f[e]);
                atomicMin(&least, o);
            }
            mass += weighed[e] && in[e] ? f[e] : 0;
        }
        __syncthreads();
        before = part_mass[tid];
        total = block_scan(before, scan);
    }
    // the part in which the uniform falls, then its tokens in runs of 1024
    const uint64_t aim = aim_of(u01, total);
    if (part_mass[tid] && before <= aim && aim < before + part_mass[tid]) {
        chosen = tid;
        chosen_before = before;
    }
    __syncthreads();
    const int end = min(g.vocab, (chosen + 1) * seg);
    uint64_t done = chosen_before;
    for (int i0 = chosen * seg; i0 < end; i0 += kSampleThreads) {
        const int i = i0 + tid;
        uint64_t f = 0;
        if (i < end) {
            const float z = logit(row, i);
            const int bin = bins.of(z);
            if (bin < cut.lo || (bin <= cut.hi && order_of(key_of(z), i) >= least)) {
                float x;
                f = sc.weight(z, x);
                if (!(x >= st.min_p)) f = 0;
            }
        }
        uint64_t at = f;
        const uint64_t all = block_scan(at, scan);
        if (f && done + at <= aim && aim < done + at + f) {
            g.token[b] = i;
            g.logprob[b] = (float)log((double)f / (double)total);
        }
        done += all;
        if (done > aim) break;
    }
}

}  // namespace zt

using namespace zt;

static bool sample_ok(int rows, int vocab) { return rows >= 0 && vocab >= 1 && vocab <= 1 << 20; }

// Workgroups of a row: enough to fill the CUs twice, of 4096 tokens at least (4 a
// thread).
static Parts parts_of(int rows, int vocab) {
    Parts p{};
    const int most = std::max(1, std::min({512 / std::max(rows, 1), ceil_div(vocab, 4096), kSplits}));
    p.seg = ceil_div(ceil_div(vocab, most), kWaves);
    p.part = p.seg * kWaves;
    p.splits = ceil_div(vocab, p.part);
    p.lanes = 1;
    while (kSampleThreads / p.lanes * p.splits > 4096) p.lanes *= 2;
    p.groups = kSampleThreads / p.lanes * p.splits;
    return p;
}

ZT_EXPORT long zt_sample_workspace_bytes(int rows, int vocab) {
    if (!sample_ok(rows, vocab)) return -1;
    return (long)rows * ((long)sizeof(RowWork) + parts_of(rows, vocab).groups * 4l);
}

template <class T>
static void launch(const SampleArgs& g, void* work, hipStream_t stream) {
    Parts p = parts_of(g.rows, g.vocab);
    p.work = (RowWork*)work;
    p.tops = (float*)(p.work + g.rows);
    const int blocks = g.rows * p.splits;
    sample_top_kernel<T><<<blocks, kSampleThreads, 0, stream>>>(g, p);
    sample_bins_kernel<T><<<blocks, kSampleThreads, 0, stream>>>(g, p);
    sample_list_kernel<T><<<blocks, kSampleThreads, 0, stream>>>(g, p);
    sample_pick_kernel<T><<<g.rows, kSampleThreads, 0, stream>>>(g, p);
}

ZT_EXPORT int zt_sample(const void* logits, long row_stride, int rows, int vocab, int type, const float* u,
                        const float* temperature, const int* top_k, const float* top_p, const float* min_p, long* token,
                        float* logprob, void* workspace, long workspace_bytes, zt_stream_t stream) {
    if (!sample_ok(rows, vocab) || !type_ok(type)) return kInvalid;
    if (rows == 0) return 0;
    if (!logits || !u || !token || !logprob || ((uintptr_t)logits & (type == ZT_F16 ? 1 : 3)) || ((uintptr_t)token & 7) ||
        (((uintptr_t)u | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p |
          (uintptr_t)logprob) & 3) || !workspace || ((uintptr_t)workspace & 15) ||
        workspace_bytes < zt_sample_workspace_bytes(rows, vocab) || (long)rows * kSplits >= 1l << 31)
        return kInvalid;
    const SampleArgs g{logits, row_stride, rows, vocab, u, temperature, top_p, min_p, top_k, token, logprob};
    if (type == ZT_F32)
        launch<float>(g, workspace, stream);
    else
        launch<_Float16>(g, workspace, stream);
    return (int)hipGetLastError();
}
