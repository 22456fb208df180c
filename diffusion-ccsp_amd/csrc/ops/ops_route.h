// ops_route.h -- the plan of a routed layer: assignments sorted by expert, and by token where tokens come as a list.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
//
// An assignment a joins token n(a) to expert e(a); it is active if both ids are in range.  Wanted: the active assignments in the order of
// (e(a), a), the inverse, the experts' first places -- and for list tokens the active assignments in the order of (n(a), a).  Both are stable
// counting sorts with keys in [0, E] and [0, N], the last key for what is dropped: place = (items with a smaller key) + (items before it
// with its own key).  Counts are sums of whole numbers and the rank inside a tile comes from the items' order, so the result does not
// depend on how the blocks run.
//
// A wave ranks 64 consecutive items at once: one ballot per key bit leaves the mask of the lanes that hold the same key, the bits
// below the own lane are the rank, and a counter per (wave, key) in LDS carries from one step to the next; at the end the counters are the wave's
// counts.  (No LDS atomics: sorted ids, or one popular expert, would send all 64 lanes to one counter.)
//
// Latency bounds all of it: a plan of 40000 assignments is 1 MB.  So a thread loads the ids of all of its items at once and keeps the keys in registers
// for the count and the rank.  Forms, by the number of assignments: everything in one block per sort and ONE launch; or two launches, count per tile and
// place, where a placing block adds up the tiles before its own by itself; with many tiles a scan between them does that once.  Keys of more than
// 4096 values (tokens) are sorted by 12-bit digits, low digit first.

struct RouteIds {
    const void* expert;
    const void* token;      // null: token of a = a / k
    int id64, A, k, E, N;
};

__device__ __forceinline__ int load_id(const void* p, int id64, long i) {
    if (!id64) return static_cast<const int*>(p)[i];
    const long v = static_cast<const long*>(p)[i];
    return v < 0 || v > 0x7fffffffL ? -1 : (int)v;
}

// the key of assignment a under either sort; E / N if dropped
__device__ __forceinline__ int token_of(const RouteIds& r, int a) { return r.token ? load_id(r.token, r.id64, a) : a / r.k; }
__device__ __forceinline__ int route_key(const RouteIds& r, int by_token, int a) {
    const int e = load_id(r.expert, r.id64, a), t = token_of(r, a);
    const bool in = e >= 0 && e < r.E && t >= 0 && t < r.N;
    return by_token ? (in ? t : r.N) : (in ? e : r.E);
}

// The keys (and tokens) of a thread's items, -1 for no item.  Every load is made, past the end the last item's: under a condition each would be
// waited for before the next is asked for.
template <int PER>
__device__ __forceinline__ void load_keys(const RouteIds& r, int by_token, const int (&item)[PER], int (&key)[PER], int (&tok)[PER]) {
    int e[PER];
    if (r.id64) {
        long le[PER], lt[PER];
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            const int a = item[s] < 0 ? 0 : item[s];
            le[s] = static_cast<const long*>(r.expert)[a];
            lt[s] = r.token ? static_cast<const long*>(r.token)[a] : 0;
        }
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            e[s] = le[s] < 0 || le[s] > 0x7fffffffL ? -1 : (int)le[s];
            tok[s] = lt[s] < 0 || lt[s] > 0x7fffffffL ? -1 : (int)lt[s];
        }
    } else {
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            const int a = item[s] < 0 ? 0 : item[s];
            e[s] = static_cast<const int*>(r.expert)[a];
            tok[s] = r.token ? static_cast<const int*>(r.token)[a] : 0;
        }
    }
#pragma unroll
    for (int s = 0; s < PER; ++s) {
        if (!r.token) tok[s] = item[s] / r.k;
        const bool in = e[s] >= 0 && e[s] < r.E && tok[s] >= 0 && tok[s] < r.N;
        key[s] = item[s] < 0 ? -1 : (by_token ? (in ? tok[s] : r.N) : (in ? e[s] : r.E));
    }
}
// a wave's or block's items i0, i0 + step, ..
template <int PER>
__device__ __forceinline__ void load_items(const RouteIds& r, const int* in, long i0, int step, long end, int (&item)[PER]) {
#pragma unroll
    for (int s = 0; s < PER; ++s) {
        const long i = i0 + (long)step * s;
        item[s] = in ? in[i < end ? i : end - 1] : (int)i;
    }
#pragma unroll
    for (int s = 0; s < PER; ++s) if (i0 + (long)step * s >= end) item[s] = -1;
}

// one pass of one sort
struct RoutePass {
    const int* in;          // items in their present order; null: 0, 1, 2, ...
    int* out;               // items in their new order (the expert sort leaves its result in RouteOut)
    int* hist;              // [tiles][bins]; behind them, where a scan runs, totals [bins]
    int by_token, shift, bins, bits;
    int last;               // the pass that leaves the sorted order
};
struct RouteOut {
    int* offsets;           // [E + 1]
    int* rows;              // [A] assignment -> row, -1 if dropped
    int* assign;            // [A] row -> assignment a; ~a in the rows behind the last active one
    int* row_token;         // [A] row -> token, -1 behind the last active one
    int* place;             // [A] the inverse of assign: assignment -> row p; ~p if dropped
    int* token_ptr;         // [N + 1] (list tokens)
    int* token_assign;      // [A]
};

constexpr int ROUTE_TILE = 2048;                                 // items of a block: 4 waves x 8 steps x 64
constexpr int ROUTE_BITS = 12, ROUTE_BINS = 1 << ROUTE_BITS;     // 4 waves x 4096 counters = 64 KB of LDS
constexpr int ROUTE_PER = ROUTE_TILE / 256;                      // items of a thread
constexpr int ROUTE_SCAN = 64;                                   // more reads of tile counts per thread of a placing block: a scan of its own
constexpr int ROUTE_SMALL = 8192, ROUTE_SMALL_TOKENS = 16384;    // limits of the one-launch form
constexpr int ROUTE_SMALL_BITS = 10;

__device__ __forceinline__ int pass_digit(const RoutePass& p, int key) { return (key >> p.shift) & ((1 << p.bits) - 1); }

// rank of the lane's item among the lanes of the wave that hold the same digit (ascending lane), and the number of those lanes
__device__ __forceinline__ int match_rank(int d, int bits, bool in, int* n) {
    unsigned long long m = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long v = __ballot((d >> b) & 1);
        m &= (d >> b) & 1 ? v : ~v;
    }
    const int lane = threadIdx.x & 63;
    *n = __popcll(m);
    return __popcll(m & ((1ull << lane) - 1));
}

// PER steps of a wave: rank of every item among the wave's items of its digit; cnt (zeroed, the wave's own) becomes the wave's counts
template <int PER>
__device__ __forceinline__ void wave_ranks(const RoutePass& p, const int (&key)[PER], int (&rank)[PER], int* cnt, int steps) {
#pragma unroll
    for (int s = 0; s < PER; ++s) {
        if (s >= steps) break;
        const bool in = key[s] >= 0;
        const int d = in ? pass_digit(p, key[s]) : 0;
        int n;
        const int r = match_rank(d, p.bits, in, &n);
        // (atomic accesses: other lanes of the wave write a counter between a lane's reads of it)
        const int base = in ? __hip_atomic_load(&cnt[d], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : 0;
        __builtin_amdgcn_wave_barrier();                         // every lane has read before the first of a digit writes
        if (in && r == 0) __hip_atomic_store(&cnt[d], base + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __builtin_amdgcn_wave_barrier();
        rank[s] = base + r;
    }
}

// lower bound of key t in the sorted order
__device__ __forceinline__ int route_bound(const RouteIds& r, const int* order, int t) {
    int lo = 0, hi = r.A;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (route_key(r, 1, order[mid]) < t) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// ---- several launches a pass ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_route_count(RouteIds r, RoutePass p0, RoutePass p1) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    extern __shared__ int cnt[];
    for (int d = threadIdx.x; d < p.bins; d += 256) cnt[d] = 0;
    const long i0 = (long)blockIdx.x * ROUTE_TILE + threadIdx.x;
    int item[ROUTE_PER], key[ROUTE_PER], tok[ROUTE_PER];
    load_items(r, p.in, i0, 256, r.A, item);
    load_keys(r, p.by_token, item, key, tok);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < ROUTE_PER; ++s) {
        const int d = key[s] >= 0 ? pass_digit(p, key[s]) : 0;
        int n;
        if (match_rank(d, p.bits, key[s] >= 0, &n) == 0 && key[s] >= 0) atomicAdd(&cnt[d], n);      // one lane per digit
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.bins; d += 256) p.hist[(size_t)blockIdx.x * p.bins + d] = cnt[d];
}

// a thread per digit: exclusive sum over the tiles, total behind
__global__ __launch_bounds__(64) void k_route_scan(RoutePass p0, RoutePass p1, int tiles) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    const int d = blockIdx.x * 64 + threadIdx.x, bins = p.bins;
    if (d >= bins) return;
    int run = 0;
    for (int t = 0; t < tiles; t += 16) {
        int c[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) c[u] = t + u < tiles ? p.hist[(size_t)(t + u) * bins + d] : 0;
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (t + u < tiles) { p.hist[(size_t)(t + u) * bins + d] = run; run += c[u]; }
    }
    p.hist[(size_t)tiles * bins + d] = run;
}

// exclusive sum over n values f(0) .. f(n - 1) by a block of NT threads, handed to g(i, sum); sums: one int per wave of LDS
template <int NT, typename F, typename G>
__device__ __forceinline__ void block_exclusive(int n, int* sums, F f, G g) {
    const int per = (n + NT - 1) / NT, lo = threadIdx.x * per, hi = lo + per < n ? lo + per : n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int own = 0;
    for (int i = lo; i < hi; ++i) own += f(i);
    int v = own;
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o); v += lane >= o ? u : 0; }
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    int run = v - own;
    for (int w = 0; w < wave; ++w) run += sums[w];
    for (int i = lo; i < hi; ++i) { const int c = f(i); g(i, run); run += c; }
    __syncthreads();
}

__global__ __launch_bounds__(256) void k_route_place(RouteIds r, RoutePass p0, RoutePass p1, RouteOut o, int tiles, int scanned) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, bins = p.bins;
    extern __shared__ int cnt[];                                 // [4][bins], then [bins]
    __shared__ int sums[4];
    int* const start = cnt + 4 * bins;
    for (int d = threadIdx.x; d < 4 * bins; d += 256) cnt[d] = 0;
    const long i0 = (long)blockIdx.x * ROUTE_TILE + wave * (ROUTE_TILE / 4) + lane;
    int* const own = cnt + wave * bins;
    int item[ROUTE_PER], key[ROUTE_PER], tok[ROUTE_PER], rank[ROUTE_PER];
    load_items(r, p.in, i0, 64, r.A, item);
    load_keys(r, p.by_token, item, key, tok);
    __syncthreads();
    wave_ranks(p, key, rank, own, ROUTE_PER);
    __syncthreads();
    if (scanned) {                                               // start = the digit's total, counts = places inside the digit
        for (int d0 = threadIdx.x; d0 < bins; d0 += 1024) {
            int run[4], total[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int d = d0 + 256 * u;
                run[u] = d < bins ? p.hist[(size_t)blockIdx.x * bins + d] : 0;
                total[u] = d < bins ? p.hist[(size_t)tiles * bins + d] : 0;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int d = d0 + 256 * u;
                if (d >= bins) break;
                start[d] = total[u];
                int at = run[u];
#pragma unroll
                for (int w = 0; w < 4; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = at; at += c; }
            }
        }
    } else {
        for (int d = threadIdx.x; d < bins; d += 256) {
            int run = 0, total = 0;
            for (int t = 0; t < tiles; t += 8) {
                int c[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) c[u] = t + u < tiles ? p.hist[(size_t)(t + u) * bins + d] : 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) { total += c[u]; run += t + u < (int)blockIdx.x ? c[u] : 0; }
            }
            start[d] = total;
#pragma unroll
            for (int w = 0; w < 4; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = run; run += c; }
        }
    }
    __syncthreads();
    block_exclusive<256>(bins, sums, [&](int d) { return start[d]; }, [&](int d, int first) { start[d] = first; });
    int* first = !p.last ? nullptr : (p.by_token ? (p.shift == 0 ? o.token_ptr : nullptr) : o.offsets);      // (one-pass sorts: the digit is the key)
    if (first && blockIdx.x == 0) for (int d = threadIdx.x; d < bins; d += 256) first[d] = start[d];         // (keys 0 .. E: the dropped ones start where the active rows end)
#pragma unroll
    for (int s = 0; s < ROUTE_PER; ++s) {
        if (key[s] < 0) continue;
        const int a = item[s], d = pass_digit(p, key[s]), pos = start[d] + own[d] + rank[s];
        if (p.by_token || !p.last) p.out[pos] = a;
        else {
            const bool act = key[s] < r.E;
            o.assign[pos] = act ? a : ~a;
            o.rows[a] = act ? pos : -1;
            o.place[a] = act ? pos : ~pos;
            o.row_token[pos] = act ? tok[s] : -1;
        }
    }
}

__global__ __launch_bounds__(256) void k_route_ptr(RouteIds r, const int* order, int* token_ptr) {
    const long t = (long)blockIdx.x * 256 + threadIdx.x;
    if (t <= r.N) token_ptr[t] = route_bound(r, order, (int)t);
}

__global__ __launch_bounds__(256) void k_route_zero(int* a, long na, int* b, long nb) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < na) a[i] = 0;
    else if (i - na < nb) b[i - na] = 0;
}

// ---- one launch: block 0 sorts by expert, block 1 (list tokens) by token -------------------------------------------------
template <int PER>                                               // items of a thread
__global__ __launch_bounds__(512) void k_route_small(RouteIds r, RouteOut o, int* tmp, int expert_bits, int token_bits) {
    extern __shared__ int cnt[];                                 // [8][bins]
    __shared__ int sums[8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, by_token = blockIdx.x;
    const int key_bits = by_token ? token_bits : expert_bits;
    const int passes = by_token ? (key_bits + ROUTE_SMALL_BITS - 1) / ROUTE_SMALL_BITS : 1;
    const int steps = (r.A + 511) / 512, i0 = wave * steps * 64 + lane;      // a wave's run of items
    const int* in = nullptr;
    for (int ps = 0; ps < passes; ++ps) {
        RoutePass p;
        p.shift = ps * ROUTE_SMALL_BITS;
        p.bits = by_token ? (key_bits - p.shift < ROUTE_SMALL_BITS ? key_bits - p.shift : ROUTE_SMALL_BITS) : key_bits;
        int* const out = ps == passes - 1 ? o.token_assign : tmp;            // (two passes at most: ROUTE_SMALL_TOKENS)
        const int bins = by_token ? 1 << p.bits : r.E + 1;
        int* const own = cnt + wave * bins;
        for (int d = threadIdx.x; d < 8 * bins; d += 512) cnt[d] = 0;
        int item[PER], key[PER], tok[PER], rank[PER];
        const long end = (wave + 1) * steps * 64 < r.A ? (wave + 1) * steps * 64 : r.A;
        load_items(r, in, i0, 64, end, item);
        load_keys(r, by_token, item, key, tok);
        __syncthreads();
        wave_ranks(p, key, rank, own, steps);
        __syncthreads();
        block_exclusive<512>(bins, sums, [&](int d) { int c = 0; for (int w = 0; w < 8; ++w) c += cnt[w * bins + d]; return c; },
            [&](int d, int run) {
                if (!by_token) o.offsets[d] = run;
                for (int w = 0; w < 8; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = run; run += c; }
            });
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            if (key[s] < 0) continue;
            const int a = item[s], d = pass_digit(p, key[s]), pos = own[d] + rank[s];
            if (by_token) out[pos] = a;
            else {
                const bool act = d < r.E;
                o.assign[pos] = act ? a : ~a;
                o.rows[a] = act ? pos : -1;
                o.place[a] = act ? pos : ~pos;
                o.row_token[pos] = act ? tok[s] : -1;
            }
        }
        __syncthreads();                                         // (the block's own writes are the next pass's input)
        in = out;
    }
    if (by_token)
        for (int t = threadIdx.x; t <= r.N; t += 512) o.token_ptr[t] = route_bound(r, o.token_assign, t);
}

// bits that hold `keys` values; one at least, so that every sort has a pass (no tokens: one key, and everything is dropped)
inline int bits_for(long keys) { int b = 1; while ((1l << b) < keys) ++b; return b; }

// ints of workspace: histograms of one pass of each sort, two orders between passes of the token sort
inline size_t route_workspace_ints(long A, int E, long N, bool list) {
    const long tiles = cdiv(A, ROUTE_TILE);
    size_t w = (size_t)(E + 1) * (tiles + 1);
    if (list) {
        const int bits = bits_for(N + 1);
        w += (size_t)(bits > ROUTE_BITS ? ROUTE_BINS : N + 1) * (tiles + 1) + 2 * (size_t)A;
    }
    return w;
}

int route(const RouteIds& r, const RouteOut& o, int* ws, hipStream_t s) {
    const bool list = o.token_ptr != nullptr;
    const int ebits = bits_for((long)r.E + 1), tbits = list ? bits_for((long)r.N + 1) : 0;
    if (r.A == 0) {                                              // every first place is 0
        hipLaunchKernelGGL(k_route_zero, dim3((unsigned)cdiv((long)r.E + 1 + (list ? (long)r.N + 1 : 0), 256)), dim3(256), 0, s, o.offsets, r.E + 1, o.token_ptr, list ? r.N + 1 : 0);
        LAUNCHED();
        return 0;
    }
    if (r.A <= ROUTE_SMALL && (!list || r.N <= ROUTE_SMALL_TOKENS)) {
        const int token_bins = 1 << (tbits < ROUTE_SMALL_BITS ? tbits : ROUTE_SMALL_BITS), bins = list && token_bins > r.E + 1 ? token_bins : r.E + 1;
        const dim3 grid(list ? 2 : 1), block(512);
        const size_t lds = 8 * bins * sizeof(int);
        if (r.A <= 1024) hipLaunchKernelGGL(k_route_small<2>, grid, block, lds, s, r, o, ws, ebits, tbits);      // (one token's 8: 4.6 us against 6.8)
        else hipLaunchKernelGGL(k_route_small<ROUTE_SMALL / 512>, grid, block, lds, s, r, o, ws, ebits, tbits);
        LAUNCHED();
        return 0;
    }
    const int tiles = (int)cdiv(r.A, ROUTE_TILE);
    const RoutePass pe = {nullptr, nullptr, ws, 0, 0, r.E + 1, ebits, 1};
    RoutePass pt = {};
    const int tpasses = list ? (int)cdiv(tbits, ROUTE_BITS) : 0;
    int *tmp0 = ws + (size_t)(r.E + 1) * (tiles + 1), *tmp1 = tmp0 + r.A, *thist = tmp1 + r.A;
    const int* tin = nullptr;
    for (int ps = 0; ps < (tpasses > 1 ? tpasses : 1); ++ps) {
        int jobs = ps == 0 ? 1 : 0;
        if (list) {
            pt.in = tin; pt.hist = thist; pt.by_token = 1; pt.shift = ps * ROUTE_BITS;
            pt.bits = tbits - pt.shift < ROUTE_BITS ? tbits - pt.shift : ROUTE_BITS;
            pt.bins = tpasses == 1 ? r.N + 1 : 1 << pt.bits;
            pt.last = ps == tpasses - 1;
            pt.out = pt.last ? o.token_assign : (ps & 1 ? tmp1 : tmp0);
            tin = pt.out;
            ++jobs;
        }
        const RoutePass& a = ps == 0 ? pe : pt;                  // (the expert sort is one pass: it runs beside the tokens' first)
        const int bins = jobs == 2 && pt.bins > pe.bins ? pt.bins : a.bins;
        const int scan = tiles * cdiv(bins, 256) > ROUTE_SCAN;
        hipLaunchKernelGGL(k_route_count, dim3(tiles, jobs), dim3(256), bins * sizeof(int), s, r, a, pt);
        if (scan) hipLaunchKernelGGL(k_route_scan, dim3((unsigned)cdiv(bins, 64), jobs), dim3(64), 0, s, a, pt, tiles);
        hipLaunchKernelGGL(k_route_place, dim3(tiles, jobs), dim3(256), 5 * bins * sizeof(int), s, r, a, pt, o, tiles, scan);
    }
    if (tpasses > 1) hipLaunchKernelGGL(k_route_ptr, dim3((unsigned)cdiv((long)r.N + 1, 256)), dim3(256), 0, s, r, o.token_assign, o.token_ptr);
    LAUNCHED();
    return 0;
}
