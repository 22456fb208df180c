// ops_rows.h -- rows to their experts' order and back.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
//
//   gather    dst[p] = src[token(p)], 0 behind the last active row            (sort_rows; the unweighted gradient of combine_rows)
//   combine   dst[n] = sum over the token's assignments a, ascending, of w[a] src[row(a)]   (combine_rows; the gradient of sort_rows, w = 1)
//   back      d_src[p] = w[a] dy[n], d_w[a] = <dy[n], src[p]>                 (the gradient of combine_rows)
//
// All three move rows and compute next to nothing: bytes bound them.  A row is read in accesses of 16 bytes (rows that are shorter: the largest power of
// two that they hold) by TPR threads, wherever it starts; the last access ends with the row and may overlap the one before it, whose values it
// then writes a second time.  Rows of one block are independent, sums are held in 32 bits and in the order of the assignments, so a result does not depend on the launch.
//
// gather and back go over the assignments either in the order of their rows, or in the order of their tokens: then the rows that share a token follow each other
// and its row comes out of a cache instead of once per expert over the fabric, while the rows written are scattered.  Worth it for rows of ROWS_BY_TOKEN bytes
// and more (4096 tokens x 4, 4096 in bf16: gather 39 -> 28 us, back 62 -> 57); shorter ones would scatter pieces of lines.
constexpr int ROWS_BY_TOKEN = 512;
// Results that the last-level cache (256 MB) cannot hold anyway are written past it, which leaves it to the tokens' rows where those are in it: 32768 tokens x 8, 2048 in
// bf16 (1 GB from 134 MB), written into the cache against past it: gather in a loop 317 us against 197, behind combine's result 320 against 202, behind back's 305 against 229;
// but where another GB was written or read before it there is nothing to keep: 323 against 330, 308 against 316, and a training step over such rows has 293.  In
// loops: 65536 x 2, 1024 (268 MB) 79 against 60; but 4096 x 4, 4096 (134 MB) 27.5 against 28.8.  (back: 449 against 430 and 129 against 124.)
constexpr long ROWS_PAST_CACHE = 192l << 20;
// combine reads each of its rows once; past the cache they leave it to what the next kernels read, unless they are few enough to be read from it again by the
// gradient.  A pass of gather, combine, back, combine in 16 bits, kept in the cache against past it: 4099 tokens x 3, 1024 (25 MB) 37 us against 40; 8192 x 4, 1024 (67 MB)
// 71 against 74; 16384 x 4, 1024 (134 MB) 155 against 144; 32768 x 4, 1024 (268 MB) 317 against 279.  Between 75 and 120 MB it goes by what else the pass holds:
// 8192 x 5 (84 MB) 85 against 92, 8192 x 6 (101 MB) 98 against 104, but 12288 x 4 (101 MB) 113 against 104, 8192 x 7 (117 MB) 127 against 119; in 32 bits 10000 x 2, 1024
// (82 MB) 104 against 100; 40528 rows of 2304 tokens, 512 (83 MB) 89 against 97, but 146 against 135 where combine's rows are not what gather wrote, as behind a product.
constexpr long ROWS_READ_ONCE = 72l << 20;

struct RowOrder {
    const int* row_token;   // [A]
    const int* assign;      // [A]
    const int* place;       // [A], null: in the order of the rows
    const int* token_assign;// [A] assignments in the order of their tokens (null: 0, 1, 2, ..)
};
// row, token and assignment of the i-th; token and assignment < 0 behind the last active row (~a)
__device__ __forceinline__ void row_at(const RowOrder& o, long i, int* p, int* tok, int* a) {
    if (!o.place) { *p = (int)i; *tok = o.row_token[i]; *a = o.assign[i]; return; }
    const int as = o.token_assign ? o.token_assign[i] : (int)i, pl = o.place[as];
    *p = pl < 0 ? ~pl : pl;
    *tok = o.row_token[*p];
    *a = pl < 0 ? ~as : as;
}

template <bool ONCE, typename V> __device__ __forceinline__ V load_once(const V* p) { if constexpr (ONCE) return __builtin_nontemporal_load(p); else return *p; }

// first element of access c of a row of n in accesses of V
template <int V> __device__ __forceinline__ long access_at(int c, int n) { const int at = c * V; return at + V <= n ? at : n - V; }

// in units of 2 bytes.  RU rows per thread: their loads are in flight together.  NT: the stores pass the last-level cache by
template <int V, bool NT>
__global__ __launch_bounds__(256) void k_rows_gather(RowOrder o, long n_rows, int width, int tpr_log2, const unsigned short* __restrict__ src, long src_stride, unsigned short* __restrict__ dst, long dst_stride) {
    typedef typename LooseOf<unsigned short, V>::type C;
    constexpr int RU = 4;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long i0 = (block_id() * rpb + (threadIdx.x >> tpr_log2)) * RU;
    int row[RU], tok[RU], as;
#pragma unroll
    for (int u = 0; u < RU; ++u) row_at(o, i0 + u < n_rows ? i0 + u : n_rows - 1, &row[u], &tok[u], &as);
    if (!src) {                                                  // (no tokens: nothing to read, whatever the plan says)
#pragma unroll
        for (int u = 0; u < RU; ++u) tok[u] = -1;
    }
    for (int c = threadIdx.x & (tpr - 1); c * V < width; c += tpr) {
        const long at = access_at<V>(c, width);
        C v[RU];
#pragma unroll
        for (int u = 0; u < RU; ++u) v[u] = tok[u] >= 0 ? *reinterpret_cast<const C*>(src + tok[u] * src_stride + at) : C(0);
#pragma unroll
        for (int u = 0; u < RU; ++u)
            if (i0 + u < n_rows) {
                C* const to = reinterpret_cast<C*>(dst + row[u] * dst_stride + at);
                if (NT) __builtin_nontemporal_store(v[u], to); else *to = v[u];
            }
    }
}

// weights: none, 32 bits or the rows' type
template <typename T> __device__ __forceinline__ float weight_at(const void* w, int wf32, int a) {
    return !w ? 1.0f : (wf32 ? static_cast<const float*>(w)[a] : (float)static_cast<const T*>(w)[a]);
}

// token_ptr null: the assignments of token n are n k .. n k + k - 1.  U rows of a token in flight.  NT: they are read past the last-level cache
template <typename T, int V, int U, bool NT>
__global__ __launch_bounds__(256) void k_rows_combine(long n_tokens, int width, int tpr_log2, int k, const int* __restrict__ token_ptr, const int* __restrict__ token_assign,
                                                      const int* __restrict__ rows, const void* __restrict__ w, int wf32, const T* __restrict__ src, long src_stride,
                                                      T* __restrict__ dst, long dst_stride) {
    typedef typename LooseOf<T, V>::type VT;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long n = block_id() * rpb + (threadIdx.x >> tpr_log2);
    if (n >= n_tokens) return;
    const long j0 = token_ptr ? token_ptr[n] : n * k, j1 = token_ptr ? token_ptr[n + 1] : j0 + k;
    for (int c = threadIdx.x & (tpr - 1); c * V < width; c += tpr) {
        const long at = access_at<V>(c, width);
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        for (long j = j0; j < j1; j += U) {                      // U rows in flight
            // (every load is made, past the token's end the last one's: under a condition each would be waited for before the next)
            VT v[U];
            float wt[U];
            int row[U], as[U];
#pragma unroll
            for (int u = 0; u < U; ++u) { const long i = j + u < j1 ? j + u : j1 - 1; as[u] = token_ptr ? token_assign[i] : (int)i; }
#pragma unroll
            for (int u = 0; u < U; ++u) { row[u] = rows[as[u]]; wt[u] = weight_at<T>(w, wf32, as[u]); }
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = load_once<NT>(reinterpret_cast<const VT*>(src + (row[u] < 0 ? 0 : row[u]) * src_stride + at));
#pragma unroll
            for (int u = 0; u < U; ++u) if (j + u >= j1) row[u] = -1;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (row[u] >= 0) {                               // (a dropped assignment adds nothing, not 0 x something)
                    const T* e = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += wt[u] * (float)e[i];
                }
        }
        VT o;
        T* e = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = (T)acc[i];
        *reinterpret_cast<VT*>(dst + n * dst_stride + at) = o;
    }
}

// d_src and / or d_w may be null.  tpr <= 64: a row's sum stays inside a wave
template <typename T, int V, bool NT>
__global__ __launch_bounds__(256) void k_rows_back(RowOrder o, long n_rows, int width, int tpr_log2, const void* __restrict__ w, int wf32, const T* __restrict__ dy, long dy_stride,
                                                   const T* __restrict__ src, long src_stride, T* __restrict__ d_src, long ds_stride, void* __restrict__ d_w) {
    typedef typename LooseOf<T, V>::type VT;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long i = block_id() * rpb + (threadIdx.x >> tpr_log2);
    const bool in = i < n_rows;
    int p, a, tok;
    row_at(o, in ? i : n_rows - 1, &p, &tok, &a);
    if (!dy) tok = -1;                                           // (no tokens)
    const float wt = a >= 0 ? weight_at<T>(w, wf32, a) : 0.0f;
    float dot = 0.0f;
    for (int c = threadIdx.x & (tpr - 1); c * V < width; c += tpr) {
        if (!in) break;
        const long at = access_at<V>(c, width);
        const int seen = c * V - (int)at;                        // elements that the access before has added to the sum
        VT g, s, d;
        if (tok >= 0) {
            g = *reinterpret_cast<const VT*>(dy + tok * dy_stride + at);
            if (d_w) s = load_once<NT>(reinterpret_cast<const VT*>(src + p * src_stride + at));
        }
        const T *ge = reinterpret_cast<const T*>(&g), *se = reinterpret_cast<const T*>(&s);
        T* de = reinterpret_cast<T*>(&d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            de[j] = tok >= 0 ? (T)(wt * (float)ge[j]) : (T)0.0f;
            if (d_w && tok >= 0 && j >= seen) dot += (float)ge[j] * (float)se[j];
        }
        if (d_src) {
            VT* const to = reinterpret_cast<VT*>(d_src + p * ds_stride + at);
            if (NT) __builtin_nontemporal_store(d, to); else *to = d;
        }
    }
    if (!d_w) return;
    for (int x = tpr >> 1; x > 0; x >>= 1) dot += __shfl_xor(dot, x);
    if (in && (threadIdx.x & (tpr - 1)) == 0) {
        const int id = a >= 0 ? a : ~a;                          // (a dropped assignment's row lies behind the last active one: its weight's gradient is 0)
        if (wf32) static_cast<float*>(d_w)[id] = dot; else static_cast<T*>(d_w)[id] = (T)dot;
    }
}

// threads per row for `chunks` accesses: a power of two, at most `most`
inline int tpr_log2_for(long chunks, int most_log2) { int l = 0; while (l < most_log2 && (1l << l) < chunks) ++l; return l; }

// f(elements per access) for a row of n > 0 elements of `bytes` bytes: 16 bytes, or what a shorter row holds
template <int BYTES, typename F>
void dispatch_vec(long n, F&& f) {
    if constexpr (BYTES == 2) if (n >= 8) return f(std::integral_constant<int, 8>{});
    if (n >= 4) return f(std::integral_constant<int, 4>{});
    if (n >= 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

// widths and strides in units of 2 bytes
int rows_gather(RowOrder o, long n_rows, int width, const void* src, long src_stride, void* dst, long dst_stride, hipStream_t s) {
    if (n_rows == 0 || width == 0) return 0;
    if (2l * width < ROWS_BY_TOKEN) o.place = nullptr;
    dispatch_vec<2>(width, [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        const int l = tpr_log2_for(cdiv(width, V), 8);
        auto go = [&](auto k) {
            hipLaunchKernelGGL(k, grid_of(cdiv(n_rows, 4 * (256 >> l))), dim3(256), 0, s, o, n_rows, width, l, (const unsigned short*)src, src_stride, (unsigned short*)dst, dst_stride);
        };
        if (V == 8 && 2 * n_rows * width >= ROWS_PAST_CACHE) go(k_rows_gather<V, V == 8>); else go(k_rows_gather<V, false>);
    });
    LAUNCHED();
    return 0;
}

template <typename T>
int rows_combine(long n_tokens, long n_rows, int width, int k, const int* token_ptr, const int* token_assign, const int* rows, const void* w, int wf32, const T* src, long src_stride, T* dst, long dst_stride, hipStream_t s) {
    if (n_tokens == 0 || width == 0) return 0;
    dispatch_vec<sizeof(T)>(width, [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        const int l = tpr_log2_for(cdiv(width, V), 8);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid_of(cdiv(n_tokens, 256 >> l)), dim3(256), 0, s, n_tokens, width, l, k, token_ptr, token_assign, rows, w, wf32, src, src_stride, dst, dst_stride);
        };
        // (rows past a token's last are the last again: no more of them than it has)
        auto by_rows = [&](auto nt) {
            constexpr bool NT = decltype(nt)::value;
            if (token_ptr || k > 4) go(k_rows_combine<T, V, 8, NT>);
            else if (k > 2) go(k_rows_combine<T, V, 4, NT>);
            else go(k_rows_combine<T, V, 2, NT>);
        };
        constexpr bool whole = V * sizeof(T) == 16;
        if (whole && n_rows * width * (long)sizeof(T) >= ROWS_READ_ONCE) by_rows(std::integral_constant<bool, whole>{}); else by_rows(std::false_type{});
    });
    LAUNCHED();
    return 0;
}

template <typename T>
int rows_back(RowOrder o, long n_rows, int width, const void* w, int wf32, const T* dy, long dy_stride, const T* src, long src_stride, T* d_src, long ds_stride, void* d_w, hipStream_t s) {
    if (n_rows == 0) return 0;
    if ((long)width * (long)sizeof(T) < ROWS_BY_TOKEN) o.place = nullptr;
    dispatch_vec<sizeof(T)>(width, [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        const int l = tpr_log2_for(cdiv(width, V), 6);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid_of(cdiv(n_rows, 256 >> l)), dim3(256), 0, s, o, n_rows, width, l, w, wf32, dy, dy_stride, src, src_stride, d_src, ds_stride, d_w);
        };
        if (V * sizeof(T) == 16 && n_rows * width * (long)sizeof(T) >= ROWS_PAST_CACHE) go(k_rows_back<T, V, V * sizeof(T) == 16>); else go(k_rows_back<T, V, false>);
    });
    LAUNCHED();
    return 0;
}
