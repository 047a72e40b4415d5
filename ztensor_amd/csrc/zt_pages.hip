// What a step over a drafted tree, and sequences that share pages, need besides
// attention: the tree's positions and masks, the path that the drawn tokens
// accept, its rows moved to the context's end, pages given back, shared and
// copied.  The cache's layout is zt_kv8.h's.
//
// All of it is bookkeeping, or a few codes: loads that wait for each other bound
// it, so each operator is one launch and its lengths stay on the device.
#include <algorithm>

#include "zt_kv8.h"

namespace zt {

constexpr int kThreads = 256;

// The rows of a request, by the device's starts, inside the step's.
struct RowSpan {
    int start, n;
    long all;  // the rows that its starts give it; those past the step's are not there
};
__device__ __forceinline__ RowSpan rows_of_request(const int* q_start, int r, int tokens) {
    RowSpan s;
    s.start = min(max(0, q_start[r]), tokens);
    const int end = max(0, q_start[r + 1]);
    s.n = max(0, min(end, tokens) - s.start);
    s.all = max(0l, (long)end - s.start);
    return s;
}

// Rows of no request, one for each call of `row`: those before the first one's and past the last one's.
template <class F>
__device__ __forceinline__ void rows_of_none(const int* q_start, int requests, int tokens, F row) {
    const int upto = requests ? min(max(0, q_start[0]), tokens) : 0;
    const int from = requests ? max(upto, min(max(0, q_start[requests]), tokens)) : 0;
    for (long i = threadIdx.x; i < (long)upto + tokens - from; i += blockDim.x) row((int)(i < upto ? i : from + i - upto));
}

// ----------------------------------------------------------------------- tree

struct TreeArgs {
    const int *parents, *kv_lens, *q_start;
    int requests, tokens, words, window;  // window: rows that a row sees, itself and those right above it (0: all)
    int* positions;
    uint64_t* mask;
};

// A row's parent, an earlier row of its request; anything else is none.
__device__ __forceinline__ int parent_of(int p, int row) { return p >= 0 && p < row ? p : -1; }

// A thread follows a row's parents, which go down, and writes the mask's words
// from the last to the first as they are left behind.  The parents of a request
// lie in LDS: a step up is one wait for that, not for memory.  8 trees of 12 rows
// 3.1 us, 128 of 48 4.3: the launch, and the starts before the parents.
__global__ __launch_bounds__(kThreads) void tree_kernel(TreeArgs g) {
    __shared__ int near[64 * ZT_TREE_WORDS];
    const int r = blockIdx.x;
    if (r >= g.requests) {
        rows_of_none(g.q_start, g.requests, g.tokens, [&](int t) {
            g.positions[t] = 0;
            for (int w = 0; w < g.words; w++) g.mask[(long)t * g.words + w] = 0;
        });
        return;
    }
    const RowSpan s = rows_of_request(g.q_start, r, g.tokens);
    const int* parents = g.parents + s.start;
    constexpr int kNear = 64 * ZT_TREE_WORDS;
    for (int i = threadIdx.x; i < min(s.n, kNear); i += kThreads) near[i] = parents[i];
    __syncthreads();
    const long context = (long)max(0, g.kv_lens[r]) - s.all;
    for (int i = threadIdx.x; i < s.n; i += kThreads) {
        uint64_t* out = g.mask + (long)(s.start + i) * g.words;
        uint64_t bits = 0;
        int w = g.words - 1, depth = 0;
        for (int at = i; at >= 0; depth++) {
            const int x = at >> 6;
            for (; w > x; w--) {
                out[w] = bits;
                bits = 0;
            }
            if (x == w && (g.window == 0 || depth < g.window)) bits |= 1ull << (at & 63);
            at = parent_of(at < kNear ? near[at] : parents[at], at);
        }
        for (; w >= 0; w--) {
            out[w] = bits;
            bits = 0;
        }
        g.positions[s.start + i] = (int)min(max(0l, context + depth - 1), 0x7FFFFFFFl);
    }
}

// --------------------------------------------------------------------- accept

struct AcceptArgs {
    const long *drafted, *drawn;
    const int *parents, *q_start;
    const long* slots;
    int requests, tokens;
    int *path, *kept, *last;
    long* token;
};

// One wave a request: from row 0 on, the first row whose parent this is and
// whose token was drawn here.  The rows lie in the lanes, so that a step of the
// path is one comparison and a ballot after the load of what was drawn.  8 trees
// of 12 rows 3.2 us, 128 of 48 6.0: a wait for each row of the path.
__global__ __launch_bounds__(64) void accept_kernel(AcceptArgs g) {
    const int r = blockIdx.x, lane = threadIdx.x;
    if (r >= g.requests) {
        rows_of_none(g.q_start, g.requests, g.tokens, [&](int t) { g.path[t] = -1; });
        return;
    }
    const RowSpan s = rows_of_request(g.q_start, r, g.tokens);
    const long* drafted = g.drafted + s.start;
    const long* drawn = g.drawn + s.start;
    int* path = g.path + s.start;
    int count = 0, at = 0;
    long want = -1;
    if (s.n > 0 && !(g.slots && g.slots[s.start] < 0)) {
        auto parent = [&](int i) { return g.parents ? parent_of(g.parents[s.start + i], i) : i - 1; };
        // 64 rows lie in the lanes
        int from = 0, mine = lane < s.n ? parent(lane) : -1;
        long has = lane < s.n ? drafted[lane] : -1;
        for (;;) {
            if (lane == 0) path[count] = at;
            count++;
            want = drawn[at];
            int next = -1;
            for (int i0 = at & ~63; next < 0 && i0 < s.n && want >= 0; i0 += 64) {
                const int i = i0 + lane;
                if (i0 != from) {
                    from = i0;
                    mine = i < s.n ? parent(i) : -1;
                    has = i < s.n ? drafted[i] : -1;
                }
                const uint64_t found = __ballot(mine == at && has == want && i > at);
                if (found) next = i0 + __builtin_ctzll(found);
            }
            if (next < 0) break;
            at = next;
        }
    }
    for (int i = count + lane; i < s.n; i += 64) path[i] = -1;
    if (lane == 0) {
        g.kept[r] = count;
        g.last[r] = count ? s.start + at : -1;
        g.token[r] = want;
    }
}

// -------------------------------------------------------------------- compact

// The buffers of caches of one shape.
constexpr int kLayers = 32;
struct Layers {
    int8_t *k[kLayers], *v[kLayers];
    float *k_scale[kLayers], *v_scale[kLayers];
};

struct CompactArgs {
    Kv8 c;  // sizes
    const int *table, *held, *q_start, *path, *kept;
    int requests, width, tokens;
    int* kv_lens_out;  // NULL: another launch writes them
};

// Where the codes of a page's places come from.
struct Sources {
    int page[128];  // -1: they stay
    uint8_t place[128];
    float scale[128];  // of that page
    uint8_t rows[128];  // the places that are written, in their order
};

// A code as this page takes it over: what it holds itself by the growth of its
// scale, what comes from another page by its value.
struct TakeOver {
    float ratio, step;  // ratio 1: the scale stays
    __device__ __forceinline__ int operator()(int code, bool far, float by) const {
        return far ? code_of((float)code * by, step) : ratio != 1.0f ? (int)rintf((float)code * ratio) : code;
    }
};
__device__ __forceinline__ int code_at(const u32x4& w, int k) { return (int8_t)(w[k >> 2] >> 8 * (k & 3)); }
__device__ __forceinline__ void set_code(u32x4& w, int k, int code) {
    w[k >> 2] = (w[k >> 2] & ~(0xFFu << 8 * (k & 3))) | ((uint32_t)code & 0xFFu) << 8 * (k & 3);
}
// The same where k is one for the wave, but not known to the compiler.
__device__ __forceinline__ int code_at_any(const u32x4& w, int k) {
    return (int8_t)((k & 8 ? k & 4 ? w[3] : w[2] : k & 4 ? w[1] : w[0]) >> 8 * (k & 3));
}
__device__ __forceinline__ void set_code_any(u32x4& w, int k, int code) {
    const uint32_t mask = 0xFFu << 8 * (k & 3), to = ((uint32_t)code & 0xFFu) << 8 * (k & 3);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (k >> 2 == i) w[i] = (w[i] & ~mask) | to;
}

// Values' places that come from the same 16 of the same page as the first of
// `left`, which they are taken from: loaded at once, a dim of all 16 a lane.
struct Sixteen {
    int page, piece;
    float scale;
    uint64_t places[2];
};
// (of place 64 half + lane: `from`'s values in a lane's registers, which others read without LDS's wait)
struct Lanes {
    int page[2], place[2];
    float scale[2];
    __device__ __forceinline__ int place_of(int half, uint64_t bits) const {
        return __builtin_amdgcn_readlane(place[half], __builtin_ctzll(bits));
    }
};
__device__ __forceinline__ Sixteen first_sixteen(const Lanes& from, uint64_t (&left)[2]) {
    const int z = __builtin_ctzll(left[0] ? left[0] : left[1]);
    Sixteen x{__builtin_amdgcn_readlane(left[0] ? from.page[0] : from.page[1], z),
              __builtin_amdgcn_readlane(left[0] ? from.place[0] : from.place[1], z) >> 4,
              __int_as_float(__builtin_amdgcn_readlane(__float_as_int(left[0] ? from.scale[0] : from.scale[1]), z)), {0, 0}};
#pragma unroll
    for (int half = 0; half < 2; half++) {
        x.places[half] = left[half] & __ballot(from.page[half] == x.page && from.place[half] >> 4 == x.piece);
        left[half] &= ~x.places[half];
    }
    return x;
}

// One wave: a request's rows of one head of keys or of values, page after page of
// those that they go to.  A row comes from behind the place that it goes to, and
// places are written in their order, each by the lane that has read what goes
// there (of values a lane has a dim of all places): nothing is written before it
// has been read.
//
// On its own page a code stays what it is; from another page its value comes,
// and the page's scale grows where that needs it, as the cache's writer has it.
//
// Loads that wait for each other bound it: starts and counts, the path, the pages,
// their scales, the codes.  Codes go in pieces of 16 bytes, of values those of 16
// places of a dim, however many of them are wanted (of 128 requests with trees of
// 48 rows, 8 heads of 128, pages of 16, two layers: 20.4 us; values' codes read one
// by one, lanes 16 bytes apart, 24.7; all codes one by one 139); 8 requests of 12
// rows, pages of 64: 5.9 us.
__global__ __launch_bounds__(64) void compact_kernel(CompactArgs g, Layers layers) {
    __shared__ Sources from;
    const Kv8& c = g.c;
    const int lane = threadIdx.x;
    int b = blockIdx.x;
    const int values = b & 1, head = (b >> 1) % c.heads;
    b = (b >> 1) / c.heads;
    const int r = b % g.requests, layer = b / g.requests;
    const RowSpan s = rows_of_request(g.q_start, r, g.tokens);
    const long base = max(0, g.held[r]);
    const int kept = min(max(0, g.kept[r]), s.n);
    if (g.kv_lens_out && layer == 0 && head == 0 && !values && lane == 0) g.kv_lens_out[r] = (int)min(base + kept, 0x7FFFFFFFl);
    int8_t* codes = values ? layers.v[layer] : layers.k[layer];
    float* scales = values ? layers.v_scale[layer] : layers.k_scale[layer];
    const int* row = g.table + (long)r * g.width;
    const long end = min(base + kept, (long)g.width << c.shift);
    for (long p = base >> c.shift; p << c.shift < end; p++) {
        const int page = row[p];
        uint64_t moved[2] = {0, 0}, far[2] = {0, 0};
        Lanes lanes;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int place = 64 * half + lane;
            const long at = (p << c.shift) + place;
            int src_page = -1;
            lanes.place[half] = 0;
            lanes.scale[half] = 0.0f;
            if (place < c.page && at >= base && at < end) {
                const int j = (int)(at - base), k = g.path[s.start + j];
                const long src = base + k;
                if (k > j && k < s.n && src < (long)g.width << c.shift) {
                    src_page = row[src >> c.shift];
                    if (!c.holds(src_page) || !c.holds(page)) src_page = -1;
                    lanes.place[half] = (int)(src & (c.page - 1));
                    if (src_page >= 0) lanes.scale[half] = scales[(long)src_page * c.heads + head];
                }
            }
            lanes.page[half] = src_page;
            if (place < c.page) {
                from.page[place] = src_page;
                from.place[place] = (uint8_t)lanes.place[half];
                from.scale[place] = lanes.scale[half];
            }
            moved[half] = __ballot(src_page >= 0);
            far[half] = __ballot(src_page >= 0 && src_page != page);
        }
        if (!(moved[0] | moved[1])) continue;
        __syncthreads();

        const long at = (long)page * c.heads + head;
        const float had = scales[at];
        float now = had;
        auto sixteen = [&](const Sixteen& x) { return reinterpret_cast<const u32x4*>(codes + c.at(x.page, head)) + x.piece; };
        if (far[0] | far[1]) {
            float m = 0.0f;
            bool bad = false;
            auto look = [&](int code, float by) {
                const float value = fabsf((float)code * by);
                m = fmaxf(m, value);
                bad |= !(value <= kMaxFloat);
            };
            uint64_t left[2] = {far[0], far[1]};
            while (!values && (left[0] | left[1])) {
                // four places at a time (the last ones again where there are fewer); of each 4 dims a lane
                uint32_t w[4];
                float by[4];
                int z = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int half = left[0] ? 0 : 1;
                    if (left[half]) {
                        z = 64 * half + __builtin_ctzll(left[half]);
                        left[half] &= left[half] - 1;
                    }
                    by[e] = from.scale[z];
                    w[e] = 0;
                    if (4 * lane < c.dp) w[e] = *reinterpret_cast<const uint32_t*>(codes + c.at(from.page[z], head) + from.place[z] * c.dp + 4 * lane);
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int k = 0; k < 4; k++) look((int8_t)(w[e] >> 8 * k), by[e]);
            }
            while (left[0] | left[1]) {
                const Sixteen x = first_sixteen(lanes, left);
                const u32x4* src = sixteen(x);
                int most = 0;  // (the largest product is the largest code's)
                for (int d = lane; d < c.dp; d += 64) {
                    const u32x4 w = src[d * (c.page / 16)];
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        for (uint64_t bits = x.places[half]; bits; bits &= bits - 1)
                            most = max(most, abs(code_at_any(w, lanes.place_of(half, bits) & 15)));
                }
                look(most, x.scale);
            }
            bad = __any(bad);
            m = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(m))))));
            now = bad || had != had ? __builtin_nanf("") : fmaxf(had, m * (1.0f / 127.0f));
        }
        const bool grown = now > had;
        const TakeOver take{grown ? had / now : 1.0f, now > 0.0f ? now : 1.0f};
        u32x4* out = reinterpret_cast<u32x4*>(codes + c.at(page, head));
        if (!values) {  // rows of dp codes, as many at a time as the lanes have
            int count = 0;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint64_t some = grown ? c.page - 64 * half >= 64 ? ~0ull : c.page <= 64 * half ? 0 : (1ull << (c.page - 64 * half)) - 1
                                            : moved[half];
                if (some >> lane & 1) from.rows[count + __builtin_popcountll(some & ((1ull << lane) - 1))] = (uint8_t)(64 * half + lane);
                count += __builtin_popcountll(some);
            }
            __syncthreads();
            const int per = c.dp / 16, rows = 64 / per, mine = lane / per, piece = lane - mine * per;
            for (int i = mine; i < count; i += rows) {
                if (mine >= rows) break;  // (of 192 dims 60 lanes)
                const int z = from.rows[i], src_page = from.page[z];
                const bool other = src_page >= 0 && src_page != page;
                u32x4 w = *(reinterpret_cast<const u32x4*>(codes + c.at(src_page < 0 ? page : src_page, head)) + (src_page < 0 ? z : from.place[z]) * per + piece);
                if (other || grown) {
                    const float by = other ? from.scale[z] : 0.0f;
#pragma unroll
                    for (int k = 0; k < 16; k++) set_code(w, k, take(code_at(w, k), other, by));
                }
                out[z * per + piece] = w;
            }
        } else {  // 16 places of a dim
            const int per = c.page / 16;
            for (int chunk = 0; chunk < per; chunk++) {
                const uint32_t some = (uint32_t)(moved[chunk >> 2] >> 16 * (chunk & 3)) & 0xFFFFu;
                if (!some && !grown) continue;
                for (int d = lane; d < c.dp; d += 64) {
                    u32x4 w = out[d * per + chunk];
                    if (grown) {
#pragma unroll
                        for (int k = 0; k < 16; k++) set_code(w, k, take(code_at(w, k), false, 0.0f));
                    }
                    const uint64_t bits16 = (uint64_t)some << 16 * (chunk & 3);
                    uint64_t left[2] = {chunk < 4 ? bits16 : 0, chunk < 4 ? 0 : bits16};
                    while (left[0] | left[1]) {
                        const Sixteen x = first_sixteen(lanes, left);
                        const u32x4 in = sixteen(x)[d * per];
#pragma unroll
                        for (int half = 0; half < 2; half++)
                            for (uint64_t bits = x.places[half]; bits; bits &= bits - 1)
                                set_code_any(w, __builtin_ctzll(bits) & 15, take(code_at_any(in, lanes.place_of(half, bits) & 15), x.page != page, x.scale));
                    }
                    out[d * per + chunk] = w;
                }
            }
        }
        if (lane == 0 && !(now == had)) scales[at] = now;
        __syncthreads();  // `from` is free again
    }
}

// ----------------------------------------------------------------------- copy

// Pages of all heads of one layer's keys or values lie in one piece: 16 KB of it
// a workgroup, whose loads wait together.  160 pages of 64 tokens, 8 heads of 128,
// 4 layers: 79 MB written (16 sources, read from the caches mostly) in 27.7 us, 2.8
// TB/s of writes; 4 pages of 16 4.1 us.  Bytes bound it.
constexpr int kCopyPieces = 4;
__global__ __launch_bounds__(kThreads) void copy_kernel(Kv8 c, Layers layers, const int* from, const int* to, int n, int chunks) {
    int b = blockIdx.x;
    const int chunk = b % chunks;
    b /= chunks;
    const int i = b % n, values = (b / n) & 1, layer = b / n >> 1;
    const int a = from[i], z = to[i];
    if (!c.holds(a) || !c.holds(z) || a == z) return;
    int8_t* codes = values ? layers.v[layer] : layers.k[layer];
    float* scales = values ? layers.v_scale[layer] : layers.k_scale[layer];
    const u32x4* src = reinterpret_cast<const u32x4*>(codes + c.at(a, 0));
    u32x4* dst = reinterpret_cast<u32x4*>(codes + c.at(z, 0));
    const int pieces = (int)((long)c.heads * c.bytes() / 16), first = chunk * kCopyPieces * kThreads + threadIdx.x;
    u32x4 w[kCopyPieces];
#pragma unroll
    for (int e = 0; e < kCopyPieces; e++)
        if (first + e * kThreads < pieces) w[e] = src[first + e * kThreads];
#pragma unroll
    for (int e = 0; e < kCopyPieces; e++)
        if (first + e * kThreads < pieces) dst[first + e * kThreads] = w[e];
    if (chunk == 0)
        for (int h = threadIdx.x; h < c.heads; h += kThreads) scales[(long)z * c.heads + h] = scales[(long)a * c.heads + h];
}

// ----------------------------------------------------------------------- trim

struct TrimArgs {
    const int *kv_lens, *keep;
    const int* table;
    int requests, width, shift, pages;
    int *free_pages, *refs, *table_out, *free_count_out;
    const int* free_count;
};

struct Gone {
    int first, end;  // pages of a request's row
};
__device__ __forceinline__ Gone gone_of(const TrimArgs& g, int r) {
    const long room = (1l << g.shift) - 1;
    auto pages = [&](int n) { return (int)min((long)g.width, (max(0, n) + room) >> g.shift); };
    Gone x{pages(g.keep[r]), pages(g.kv_lens[r])};
    x.end = max(x.first, x.end);
    return x;
}

constexpr int kTrimThreads = 1024;

// Running sums over the workgroup, a thread's own value included; `all` is the whole.
__device__ __forceinline__ int block_scan(int v, int* sums, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v, o);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < kTrimThreads / 64; w++) {
        if (w < wave) before += sums[w];
        all += sums[w];
    }
    return before + v;
}

// The first workgroup marks the pages that nobody holds any more in LDS, one bit
// each, and lists them in the order of their numbers, whatever the order in
// which they were found.  The others copy the rows of the table.  One workgroup,
// since the list has one end and one order: 8 requests 4.0 us, 128 4.3.
__global__ __launch_bounds__(kTrimThreads) void trim_kernel(TrimArgs g) {
    extern __shared__ uint32_t bits[];
    __shared__ int upto[kTrimThreads], sums[kTrimThreads / 64];
    if (blockIdx.x > 0) {
        const int r = blockIdx.x - 1;
        const Gone x = gone_of(g, r);
        for (int j = threadIdx.x; j < g.width; j += kTrimThreads) {
            const int p = g.table[(long)r * g.width + j];
            g.table_out[(long)r * g.width + j] = j >= x.first && j < x.end && (unsigned)p < (unsigned)g.pages ? -1 : p;
        }
        return;
    }
    const bool in_place = g.table_out == g.table;
    const int words = (g.pages + 31) >> 5;
    for (int i = threadIdx.x; i < words; i += kTrimThreads) bits[i] = 0;
    for (int r0 = 0; r0 < g.requests; r0 += kTrimThreads) {
        Gone x{0, 0};
        if (r0 + (int)threadIdx.x < g.requests) x = gone_of(g, r0 + threadIdx.x);
        int all;
        __syncthreads();
        upto[threadIdx.x] = block_scan(x.end - x.first, sums, all);  // (at most 2^31: the table's entries)
        __syncthreads();
        for (int i = threadIdx.x; i < all; i += kTrimThreads) {
            int lo = 0, hi = kTrimThreads - 1;  // the first request whose sum passes i
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (upto[mid] > i) hi = mid; else lo = mid + 1;
            }
            const Gone y = gone_of(g, r0 + lo);
            const long at = (long)(r0 + lo) * g.width + y.end - (upto[lo] - i);
            const int p = g.table[at];
            if ((unsigned)p >= (unsigned)g.pages) continue;
            if (in_place) g.table_out[at] = -1;
            if (!g.refs || atomicSub(&g.refs[p], 1) <= 0) atomicOr(&bits[p >> 5], 1u << (p & 31));
        }
    }
    __syncthreads();
    const int free = min(max(0, *g.free_count), g.pages), each = (words + kTrimThreads - 1) / kTrimThreads;
    const int w0 = min(words, (int)threadIdx.x * each), w1 = min(words, w0 + each);
    int mine = 0, all;
    for (int w = w0; w < w1; w++) mine += __builtin_popcount(bits[w]);
    int to = free + block_scan(mine, sums, all) - mine;
    for (int w = w0; w < w1; w++)
        for (uint32_t left = bits[w]; left; left &= left - 1, to++) {
            const int p = 32 * w + __builtin_ctz(left);
            if (to < g.pages) g.free_pages[to] = p;
            if (g.refs) g.refs[p] = 0;
        }
    if (threadIdx.x == 0) *g.free_count_out = min(g.pages, free + all);
}

// ----------------------------------------------------------------------- fork

struct ForkArgs {
    zt_kv8_fork_call a;
    int shift;
};

// What fork i does: the tokens of its source, and whether it takes a page.
struct Forked {
    int source, held;
    bool part;
};
__device__ __forceinline__ Forked forked(const ForkArgs& g, int i) {
    Forked f{g.a.source[i], 0, false};
    if ((unsigned)f.source >= (unsigned)g.a.rows) return f;
    const int held = g.a.kv_lens[f.source];
    f.held = held > 0 && held <= (long)g.a.width << g.shift ? held : 0;
    f.part = (f.held & ((1 << g.shift) - 1)) != 0 && (unsigned)g.a.target[i] < (unsigned)g.a.rows && f.source != g.a.target[i];
    return f;
}

// Workgroup r: row r of the table, which is a fork's or stays.  How many forks
// before it take a page it counts by itself, as the step's plan does: loads that
// wait for each other, no second launch.  A fork whose target an earlier one has
// takes none; whether there may be any, a bit of LDS for each row says (past 2^18
// rows two may share one: then the earlier forks are looked through for nothing).
// 4 forks of 500 tokens 4.0 us, 160 of 1500 6.6.
constexpr int kMet = 1 << 18;  // rows that have bits of their own
__global__ __launch_bounds__(kThreads) void fork_kernel(ForkArgs g) {
    extern __shared__ uint32_t met[];  // of min(rows, kMet) bits
    __shared__ int chosen, wanted, twice;
    const int r = blockIdx.x, free = min(max(0, *g.a.free_count), g.a.pages);
    if (threadIdx.x == 0) {
        chosen = r == g.a.rows ? 0 : g.a.n;
        wanted = twice = 0;
    }
    __syncthreads();
    if (r < g.a.rows)
        for (int i = threadIdx.x; i < g.a.n; i += kThreads)
            if (g.a.target[i] == r) atomicMin(&chosen, i);
    __syncthreads();
    const int i = chosen;
    const int* row = g.a.table + (long)r * g.a.width;
    int* out = g.a.table_out + (long)r * g.a.width;
    const bool itself = r < g.a.rows && i < g.a.n && g.a.source[i] == r;
    if (r < g.a.rows) {
        for (int k = threadIdx.x; k < g.a.n; k += kThreads)  // (a row that comes twice: the first of them)
            if (g.a.target[k] == r && (k != i || itself)) g.a.copy_from[k] = g.a.copy_to[k] = -1;
        if (i >= g.a.n || itself) {
            for (int j = threadIdx.x; j < g.a.width; j += kThreads) out[j] = row[j];
            if (threadIdx.x == 0) g.a.kv_lens_out[r] = g.a.kv_lens[r];
            return;
        }
    }
    // the pages that forks before this one take, or (of no row) all
    const int n = r < g.a.rows ? i : g.a.n;
    for (int k = threadIdx.x; 32 * k < min(g.a.rows, kMet); k += kThreads) met[k] = 0;
    __syncthreads();
    int mine = 0;
    for (int k = threadIdx.x; k < n; k += kThreads) {
        mine += forked(g, k).part;
        const int t = g.a.target[k];
        if ((unsigned)t < (unsigned)g.a.rows && atomicOr(&met[t % kMet / 32], 1u << (t & 31)) >> (t & 31) & 1) twice = 1;
    }
    __syncthreads();
    if (twice) {
        mine = 0;
        for (int k = threadIdx.x; k < n; k += kThreads) {
            bool first = forked(g, k).part;
            for (int e = 0; e < k && first; e++) first = g.a.target[e] != g.a.target[k];
            mine += first;
        }
    }
    if (mine) atomicAdd(&wanted, mine);
    __syncthreads();
    if (r == g.a.rows) {
        for (int k = threadIdx.x; k < n; k += kThreads)
            if ((unsigned)g.a.target[k] >= (unsigned)g.a.rows) g.a.copy_from[k] = g.a.copy_to[k] = -1;
        if (threadIdx.x == 0) *g.a.free_count_out = free - min(free, wanted);
        return;
    }
    const Forked f = forked(g, i);
    const bool done = f.held > 0 && (!f.part || wanted < free);
    const int full = f.held >> g.shift, fresh = done && f.part ? g.a.free_pages[free - 1 - wanted] : -1;
    const int* from = g.a.table + (long)(f.held ? f.source : r) * g.a.width;
    for (int j = threadIdx.x; j < g.a.width; j += kThreads) {
        int p = -1;
        if (done && j < full) {
            p = from[j];
            if ((unsigned)p < (unsigned)g.a.pages) atomicAdd(&g.a.refs[p], 1);
        }
        out[j] = done && f.part && j == full ? fresh : p;
    }
    if (threadIdx.x == 0) {
        g.a.kv_lens_out[r] = done ? f.held : 0;
        g.a.copy_from[i] = done && f.part ? from[full] : -1;
        g.a.copy_to[i] = fresh;
    }
}

}  // namespace zt

using namespace zt;

ZT_EXPORT int zt_kv8_tree_window(const int* parents, const int* kv_lens, const int* q_start, int requests, int tokens, int words,
                                 int window, int* positions, uint64_t* mask, zt_stream_t stream) {
    if (requests < 0 || requests >= 1 << 24 || tokens < 0 || words < 1 || words > ZT_TREE_WORDS || window < 0 || !q_start) return kInvalid;
    if (tokens == 0) return 0;
    if (!parents || !positions || !mask || (requests && !kv_lens) ||
        (((uintptr_t)parents | (uintptr_t)kv_lens | (uintptr_t)q_start | (uintptr_t)positions) & 3) || ((uintptr_t)mask & 7))
        return kInvalid;
    const Bytes in[] = {{parents, 4l * tokens}, {kv_lens, 4l * requests}, {q_start, 4l * requests + 4}};
    const Bytes out[] = {{positions, 4l * tokens}, {mask, 8l * tokens * words}};
    if (!apart(in, out)) return kInvalid;
    tree_kernel<<<requests + 1, kThreads, 0, stream>>>({parents, kv_lens, q_start, requests, tokens, words, window, positions, mask});
    return (int)hipGetLastError();
}

ZT_EXPORT int zt_kv8_tree(const int* parents, const int* kv_lens, const int* q_start, int requests, int tokens, int words,
                          int* positions, uint64_t* mask, zt_stream_t stream) {
    return zt_kv8_tree_window(parents, kv_lens, q_start, requests, tokens, words, 0, positions, mask, stream);
}

ZT_EXPORT int zt_tree_accept(const long* drafted, const long* drawn, const int* parents, const int* q_start,
                             const long* slots, int requests, int tokens, int* path, int* kept, int* last, long* token,
                             zt_stream_t stream) {
    if (requests < 0 || requests >= 1 << 24 || tokens < 0 || !q_start) return kInvalid;
    if (tokens == 0 && requests == 0) return 0;
    if ((tokens && (!drafted || !drawn || !path)) || (requests && (!kept || !last || !token)) ||
        (((uintptr_t)parents | (uintptr_t)q_start | (uintptr_t)path | (uintptr_t)kept | (uintptr_t)last) & 3) ||
        (((uintptr_t)drafted | (uintptr_t)drawn | (uintptr_t)slots | (uintptr_t)token) & 7))
        return kInvalid;
    const long row = 4l * requests, rows = 4l * tokens;
    const Bytes in[] = {{drafted, 2 * rows}, {drawn, 2 * rows}, {parents, parents ? rows : 0}, {q_start, row + 4}, {slots, slots ? 2 * rows : 0}};
    const Bytes out[] = {{path, rows}, {kept, row}, {last, row}, {token, 2 * row}};
    if (!apart(in, out)) return kInvalid;
    accept_kernel<<<requests + 1, 64, 0, stream>>>({drafted, drawn, parents, q_start, slots, requests, tokens, path, kept, last, token});
    return (int)hipGetLastError();
}

static bool caches_ok(const zt_kv8_cache* c, int n) {
    if (!c || n < 1 || n > 1 << 16) return false;
    for (int i = 0; i < n; i++)
        if (!kv8_ok(c[i]) || c[i].pages != c[0].pages || c[i].kv_heads != c[0].kv_heads || c[i].head_dim != c[0].head_dim ||
            c[i].page_tokens != c[0].page_tokens)
            return false;
    return true;
}

// The launches of caches, kLayers at a time.
template <class F>
static int for_layers(const zt_kv8_cache* caches, int n, F launch) {
    for (int at = 0; at < n; at += kLayers) {
        Layers l{};
        const int some = std::min(kLayers, n - at);
        for (int i = 0; i < some; i++) {
            l.k[i] = (int8_t*)caches[at + i].k;
            l.v[i] = (int8_t*)caches[at + i].v;
            l.k_scale[i] = caches[at + i].k_scale;
            l.v_scale[i] = caches[at + i].v_scale;
        }
        launch(l, some, at == 0);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

ZT_EXPORT int zt_kv8_compact(const zt_kv8_cache* caches, int layers, const int* table, int requests, int width,
                             const int* held, const int* q_start, const int* path, const int* kept, int tokens,
                             int* kv_lens_out, zt_stream_t stream) {
    if (!caches_ok(caches, layers) || requests < 0 || width < 1 || tokens < 0 || (long)requests * width >= 1l << 31)
        return kInvalid;
    if (requests == 0) return 0;
    if (!table || !held || !q_start || (tokens && !path) || !kept || !kv_lens_out ||
        (((uintptr_t)table | (uintptr_t)held | (uintptr_t)q_start | (uintptr_t)path | (uintptr_t)kept | (uintptr_t)kv_lens_out) & 3))
        return kInvalid;
    const long row = 4l * requests;
    const Bytes in[] = {{table, row * width}, {held, row}, {q_start, row + 4}, {path, 4l * tokens}, {kept, row}};
    const Bytes out[] = {{kv_lens_out, row}};
    if (!apart(in, out)) return kInvalid;
    const long blocks = 2l * caches->kv_heads * requests;
    if (blocks * std::min(layers, kLayers) >= 1l << 31) return kInvalid;
    return for_layers(caches, layers, [&](const Layers& l, int n, bool first) {
        const CompactArgs g{kv8_of(*caches), table, held, q_start, path, kept, requests, width, tokens, first ? kv_lens_out : nullptr};
        compact_kernel<<<(unsigned)(blocks * n), 64, 0, stream>>>(g, l);
    });
}

ZT_EXPORT int zt_kv8_copy(const zt_kv8_cache* caches, int layers, const int* from, const int* to, int n, zt_stream_t stream) {
    if (!caches_ok(caches, layers) || n < 0) return kInvalid;
    if (n == 0) return 0;
    if (!from || !to || (((uintptr_t)from | (uintptr_t)to) & 3)) return kInvalid;
    const Kv8 c = kv8_of(*caches);
    const int chunks = ceil_div((long)c.heads * c.bytes(), 16l * kThreads * kCopyPieces);
    if (2l * n * chunks * std::min(layers, kLayers) >= 1l << 31) return kInvalid;
    return for_layers(caches, layers, [&](const Layers& l, int some, bool) {
        copy_kernel<<<(unsigned)(2l * n * chunks * some), kThreads, 0, stream>>>(c, l, from, to, n, chunks);
    });
}

ZT_EXPORT int zt_kv8_trim(const int* kv_lens, const int* keep, const int* table, int requests, int width, int* free_pages,
                          const int* free_count, int pages, int page_tokens, int* refs, int* table_out,
                          int* free_count_out, zt_stream_t stream) {
    if (requests < 0 || width < 1 || pages < 0 || pages > 1 << 20 || !page_tokens_ok(page_tokens) ||
        (long)requests * width >= (1l << 31) - kTrimThreads || requests >= 1 << 24)
        return kInvalid;
    if ((requests && (!kv_lens || !keep || !table || !table_out)) || (pages && !free_pages) || !free_count || !free_count_out)
        return kInvalid;
    const void* ints[] = {kv_lens, keep, table, free_pages, free_count, refs, table_out, free_count_out};
    for (const void* p : ints)
        if ((uintptr_t)p & 3) return kInvalid;
    const long row = 4l * requests, rows = row * width, list = 4l * pages;
    const Bytes in[] = {{kv_lens, row}, {keep, row}, {free_count, 4}, {table, table_out == table ? 0 : rows}};
    const Bytes out[] = {{free_pages, list}, {refs, refs ? list : 0}, {table_out, rows}, {free_count_out, 4}};
    if (!apart(in, out)) return kInvalid;
    static std::atomic<uint64_t> raised{0};
    const int lds = (pages + 31) / 32 * 4;
    if (lds > 48 << 10) {  // (beside the kernel's own)
        const hipError_t rc = raise_lds((const void*)trim_kernel, (1 << 20) / 8, raised);
        if (rc != hipSuccess) return (int)rc;
    }
    const TrimArgs g{kv_lens, keep, table, requests, width, __builtin_ctz(page_tokens), pages, free_pages, refs, table_out, free_count_out, free_count};
    trim_kernel<<<table_out == table ? 1 : requests + 1, kTrimThreads, lds, stream>>>(g);
    return (int)hipGetLastError();
}

ZT_EXPORT int zt_kv8_fork(const zt_kv8_fork_call* a, zt_stream_t stream) {
    if (!a || a->n < 0 || a->rows < 0 || a->width < 1 || a->pages < 0 || !page_tokens_ok(a->page_tokens) || a->reserved ||
        (long)a->rows * a->width >= (1l << 31) - 256 || a->rows >= 1 << 24 || a->n >= 1 << 24)
        return kInvalid;
    if ((a->n && (!a->source || !a->target || !a->copy_from || !a->copy_to)) ||
        (a->rows && (!a->kv_lens || !a->table || !a->kv_lens_out || !a->table_out)) ||
        (a->pages && (!a->free_pages || !a->refs)) || !a->free_count || !a->free_count_out)
        return kInvalid;
    const void* ints[] = {a->source, a->target, a->kv_lens, a->table, a->free_pages, a->free_count, a->refs, a->kv_lens_out,
                          a->table_out, a->free_count_out, a->copy_from, a->copy_to};
    for (const void* p : ints)
        if ((uintptr_t)p & 3) return kInvalid;
    const long row = 4l * a->rows, list = 4l * a->pages, forks = 4l * a->n;
    const Bytes in[] = {{a->source, forks}, {a->target, forks}, {a->kv_lens, row}, {a->table, row * a->width}, {a->free_pages, list}, {a->free_count, 4}};
    const Bytes out[] = {{a->refs, list}, {a->kv_lens_out, row}, {a->table_out, row * a->width}, {a->free_count_out, 4}, {a->copy_from, forks}, {a->copy_to, forks}};
    if (!apart(in, out)) return kInvalid;
    fork_kernel<<<a->rows + 1, kThreads, (std::min(a->rows, kMet) + 31) / 32 * 4, stream>>>({*a, __builtin_ctz(a->page_tokens)});
    return (int)hipGetLastError();
}
