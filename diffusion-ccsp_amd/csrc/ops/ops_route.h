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
// below the own lane are the rank, and a counter per (wave, key) in LDS carries from one step to the next.
//
// Two forms, by the number of assignments (both sides at the benchmark's ROUTE_SMALL limit are in the launch rule below): everything in
// one block per sort and ONE launch, or three launches (count per tile, scan per key, place).  Keys of more than 4096 values (tokens) are
// sorted by 12-bit digits, low digit first.

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

// one pass of one sort
struct RoutePass {
    const int* in;          // items in their present order; null: 0, 1, 2, ...
    int* out;               // items in their new order
    int* hist;              // [bins][tiles], then totals [bins]
    int by_token, shift, bins, bits;
    int last;               // the pass that leaves the sorted order
};
struct RouteOut {
    int* offsets;           // [E + 1]
    int* rows;              // [A] assignment -> row, -1 if dropped
    int* assign;            // [A] row -> assignment a; ~a in the rows behind the last active one
    int* row_token;         // [A] row -> token, -1 behind the last active one
    int* token_ptr;         // [N + 1] (list tokens)
    int* token_assign;      // [A]
};

constexpr int ROUTE_TILE = 2048;                                 // items of a block: 4 waves x 8 steps x 64
constexpr int ROUTE_BITS = 12, ROUTE_BINS = 1 << ROUTE_BITS;     // 4 waves x 4096 counters = 64 KB of LDS
constexpr int ROUTE_SMALL = 8192, ROUTE_SMALL_TOKENS = 16384;    // limits of the one-launch form
constexpr int ROUTE_SMALL_BITS = 10;

__device__ __forceinline__ int pass_digit(const RouteIds& r, const RoutePass& p, int a) { return (route_key(r, p.by_token, a) >> p.shift) & ((1 << p.bits) - 1); }

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

// what the last pass of a sort leaves for item a at place pos
__device__ __forceinline__ void route_place(const RouteIds& r, const RoutePass& p, const RouteOut& o, int a, int pos) {
    p.out[pos] = a;
    if (!p.last || p.by_token) return;
    const bool in = route_key(r, 0, a) < r.E;
    o.assign[pos] = in ? a : ~a;
    o.rows[a] = in ? pos : -1;
    o.row_token[pos] = in ? token_of(r, a) : -1;
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

// ---- three launches a pass -----------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_route_count(RouteIds r, RoutePass p0, RoutePass p1, int tiles) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    extern __shared__ int cnt[];
    for (int d = threadIdx.x; d < p.bins; d += 256) cnt[d] = 0;
    __syncthreads();
    const long i0 = (long)blockIdx.x * ROUTE_TILE;
    for (int s = 0; s < ROUTE_TILE; s += 256) {
        const long i = i0 + s + threadIdx.x;
        if (i < r.A) atomicAdd(&cnt[pass_digit(r, p, p.in ? p.in[i] : (int)i)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.bins; d += 256) p.hist[(size_t)d * tiles + blockIdx.x] = cnt[d];
}

// a wave per digit: exclusive sum over the tiles, total behind
__global__ __launch_bounds__(256) void k_route_scan(RoutePass p0, RoutePass p1, int tiles) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    const int d = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (d >= p.bins) return;
    int* h = p.hist + (size_t)d * tiles;
    int run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 64) {
        const int own = t0 + lane < tiles ? h[t0 + lane] : 0;
        int v = own;
        for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o); v += lane >= o ? u : 0; }
        if (t0 + lane < tiles) h[t0 + lane] = run + v - own;
        run += __shfl(v, 63);
    }
    if (lane == 0) p.hist[(size_t)p.bins * tiles + d] = run;
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

__global__ __launch_bounds__(256) void k_route_place(RouteIds r, RoutePass p0, RoutePass p1, RouteOut o, int tiles) {
    const RoutePass p = blockIdx.y ? p1 : p0;
    extern __shared__ int cnt[];                                 // [4][bins]
    __shared__ int sums[4];
    const int wave = threadIdx.x >> 6, bins = p.bins;
    for (int d = threadIdx.x; d < 4 * bins; d += 256) cnt[d] = 0;
    __syncthreads();
    const long i0 = (long)blockIdx.x * ROUTE_TILE + wave * (ROUTE_TILE / 4) + (threadIdx.x & 63);
    int* const cown = cnt + wave * bins;
    volatile int* const own = cown;                              // (other lanes of the wave write it between a lane's reads)
    for (int s = 0; s < ROUTE_TILE / 4; s += 64)
        if (i0 + s < r.A) atomicAdd(&cown[pass_digit(r, p, p.in ? p.in[i0 + s] : (int)(i0 + s))], 1);
    __syncthreads();
    const int* total = p.hist + (size_t)bins * tiles;
    int* first = p.last ? (p.by_token ? (p.shift == 0 ? o.token_ptr : nullptr) : o.offsets) : nullptr;   // (one-pass sorts: the digit is the key)
    block_exclusive<256>(bins, sums, [&](int d) { return total[d]; },
        [&](int d, int start) {
            if (first && blockIdx.x == 0) first[d] = start;      // (keys 0 .. E: the dropped ones start where the active rows end)
            int run = start + p.hist[(size_t)d * tiles + blockIdx.x];
            for (int w = 0; w < 4; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = run; run += c; }
        });
    for (int s = 0; s < ROUTE_TILE / 4; s += 64) {
        const bool in = i0 + s < r.A;
        const int a = in ? (p.in ? p.in[i0 + s] : (int)(i0 + s)) : 0;
        const int d = in ? pass_digit(r, p, a) : 0;
        int n;
        const int rank = match_rank(d, p.bits, in, &n);
        const int base = in ? own[d] : 0;
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) own[d] = base + n;
        __builtin_amdgcn_wave_barrier();
        if (in) route_place(r, p, o, a, base + rank);
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
__global__ __launch_bounds__(512) void k_route_small(RouteIds r, RouteOut o, int* tmp0, int* tmp1, int expert_bits, int token_bits) {
    extern __shared__ int cnt[];                                 // [8][bins]
    __shared__ int sums[8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, by_token = blockIdx.x;
    const int key_bits = by_token ? token_bits : expert_bits;
    const int passes = by_token ? (key_bits + ROUTE_SMALL_BITS - 1) / ROUTE_SMALL_BITS : 1;
    const int per = ((r.A + 511) / 512) * 64, i0 = wave * per + lane, i1 = wave * per + per < r.A ? wave * per + per : r.A;
    const int* in = nullptr;
    for (int ps = 0; ps < passes; ++ps) {
        RoutePass p;
        p.in = in; p.by_token = by_token; p.shift = ps * ROUTE_SMALL_BITS;
        p.bits = by_token ? (key_bits - p.shift < ROUTE_SMALL_BITS ? key_bits - p.shift : ROUTE_SMALL_BITS) : key_bits;
        p.bins = by_token ? 1 << p.bits : r.E + 1;
        p.last = ps == passes - 1;
        p.out = by_token ? (p.last ? o.token_assign : (ps & 1 ? tmp1 : tmp0)) : nullptr;
        const int bins = p.bins;
        int* const cown = cnt + wave * bins;
        volatile int* const own = cown;
        for (int d = threadIdx.x; d < 8 * bins; d += 512) cnt[d] = 0;
        __syncthreads();
        for (int i = i0; i < i1; i += 64) atomicAdd(&cown[pass_digit(r, p, in ? in[i] : i)], 1);
        __syncthreads();
        block_exclusive<512>(bins, sums, [&](int d) { int c = 0; for (int w = 0; w < 8; ++w) c += cnt[w * bins + d]; return c; },
            [&](int d, int run) {
                if (!by_token) o.offsets[d] = run;
                for (int w = 0; w < 8; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = run; run += c; }
            });
        for (int i = i0; i < i0 - lane + per; i += 64) {          // (every lane of the wave in every step: the ballots are the wave's)
            const bool live = i < i1;
            const int a = live ? (in ? in[i] : i) : 0;
            const int d = live ? pass_digit(r, p, a) : 0;
            int n;
            const int rank = match_rank(d, p.bits, live, &n);
            const int base = live ? own[d] : 0;
            __builtin_amdgcn_wave_barrier();
            if (live && rank == 0) own[d] = base + n;
            __builtin_amdgcn_wave_barrier();
            if (live) {
                if (by_token) p.out[base + rank] = a;
                else {
                    const bool act = d < r.E;
                    o.assign[base + rank] = act ? a : ~a;
                    o.rows[a] = act ? base + rank : -1;
                    o.row_token[base + rank] = act ? token_of(r, a) : -1;
                }
            }
        }
        __syncthreads();                                         // (the block's own writes to p.out are the next pass's input)
        in = p.out;
    }
    if (by_token)
        for (int t = threadIdx.x; t <= r.N; t += 512) o.token_ptr[t] = route_bound(r, o.token_assign, t);
}

inline int bits_for(long keys) { int b = 0; while ((1l << b) < keys) ++b; return b; }        // digits that hold `keys` values

// ints of workspace: histograms of the passes of both sorts (one at a time) and two orders between passes
inline size_t route_workspace_ints(long A, int E, long N, bool list) {
    const long tiles = cdiv(A, ROUTE_TILE);
    size_t w = (size_t)(E + 1) * (tiles + 1);
    if (list) {
        const int bits = bits_for(N + 1);
        const long bins = bits > ROUTE_BITS ? ROUTE_BINS : N + 1;
        w += (size_t)bins * (tiles + 1) + 2 * (size_t)A + (size_t)A;   // (+ the expert sort's own order)
    } else w += (size_t)A;
    return w;
}

int route(const RouteIds& r, const RouteOut& o, int* ws, hipStream_t s) {
    const bool list = o.token_ptr != nullptr;
    const int ebits = bits_for((long)r.E + 1), tbits = list ? bits_for((long)r.N + 1) : 0;
    if (r.A == 0) {
        // (nothing to sort: every first place is 0)
        hipLaunchKernelGGL(k_route_zero, dim3((unsigned)cdiv((long)r.E + 1 + (list ? (long)r.N + 1 : 0), 256)), dim3(256), 0, s, o.offsets, r.E + 1, o.token_ptr, list ? r.N + 1 : 0);
        LAUNCHED();
        return 0;
    }
    if (r.A <= ROUTE_SMALL && (!list || r.N <= ROUTE_SMALL_TOKENS)) {
        const int bins = list && (1 << ROUTE_SMALL_BITS) > r.E + 1 ? 1 << ROUTE_SMALL_BITS : r.E + 1;
        hipLaunchKernelGGL(k_route_small, dim3(list ? 2 : 1), dim3(512), 8 * bins * sizeof(int), s, r, o, ws, ws + r.A, ebits, tbits);
        LAUNCHED();
        return 0;
    }
    const int tiles = (int)cdiv(r.A, ROUTE_TILE);
    RoutePass pe = {nullptr, ws, ws + r.A, 0, 0, r.E + 1, ebits, 1}, pt = {};
    int* w = ws + r.A + (size_t)(r.E + 1) * (tiles + 1);
    const int tpasses = list ? (int)cdiv(tbits, ROUTE_BITS) : 0;
    int *tmp0 = w, *tmp1 = w + r.A, *thist = w + 2 * (size_t)r.A;
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
        hipLaunchKernelGGL(k_route_count, dim3(tiles, jobs), dim3(256), bins * sizeof(int), s, r, a, pt, tiles);
        hipLaunchKernelGGL(k_route_scan, dim3((unsigned)cdiv(bins, 4), jobs), dim3(256), 0, s, a, pt, tiles);
        hipLaunchKernelGGL(k_route_place, dim3(tiles, jobs), dim3(256), 4 * bins * sizeof(int), s, r, a, pt, o, tiles);
    }
    if (tpasses > 1) hipLaunchKernelGGL(k_route_ptr, dim3((unsigned)cdiv((long)r.N + 1, 256)), dim3(256), 0, s, r, o.token_assign, o.token_ptr);
    LAUNCHED();
    return 0;
}
