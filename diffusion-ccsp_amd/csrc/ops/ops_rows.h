// ops_rows.h -- rows to their experts' order and back.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
//
//   gather    dst[p] = src[token(p)], 0 behind the last active row            (sort_rows; the unweighted gradient of combine_rows)
//   combine   dst[n] = sum over the token's assignments a, ascending, of w[a] src[row(a)]   (combine_rows; the gradient of sort_rows, w = 1)
//   back      d_src[p] = w[a] dy[n], d_w[a] = <dy[n], src[p]>                 (the gradient of combine_rows)
//
// All three move rows and compute next to nothing: bytes bound them.  A row is read in accesses of VB bytes (16 where width, strides and
// addresses allow, else the largest power of two that does) by TPR threads, rows of one block are independent, sums are held in 32 bits and in the
// order of the assignments, so a result does not depend on the launch.


template <int VB> struct Chunk;
template <> struct Chunk<16> { typedef u32x4 t; };
template <> struct Chunk<8> { typedef uint2 t; };
template <> struct Chunk<4> { typedef unsigned int t; };
template <> struct Chunk<2> { typedef unsigned short t; };
template <typename C> __device__ __forceinline__ C chunk_zero() { C z; __builtin_memset(&z, 0, sizeof(C)); return z; }

// RU rows per thread: their loads are in flight together
template <int VB, int RU>
__global__ __launch_bounds__(256) void k_rows_gather(long n_rows, int chunks, int tpr_log2, const char* __restrict__ src, long src_stride, const int* __restrict__ row_token,
                                                     char* __restrict__ dst, long dst_stride) {
    typedef typename Chunk<VB>::t C;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long p0 = block_id() * rpb * RU + (threadIdx.x >> tpr_log2);
    int tok[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) tok[u] = p0 + u * rpb < n_rows ? row_token[p0 + u * rpb] : -1;
    for (int c = threadIdx.x & (tpr - 1); c < chunks; c += tpr) {
        C v[RU];
#pragma unroll
        for (int u = 0; u < RU; ++u) v[u] = tok[u] >= 0 ? *reinterpret_cast<const C*>(src + tok[u] * src_stride + (long)c * VB) : chunk_zero<C>();
#pragma unroll
        for (int u = 0; u < RU; ++u)
            if (p0 + u * rpb < n_rows) *reinterpret_cast<C*>(dst + (p0 + u * rpb) * dst_stride + (long)c * VB) = v[u];
    }
}

// weights: none, 32 bits or the rows' type
template <typename T> __device__ __forceinline__ float weight_at(const void* w, int wf32, int a) {
    return !w ? 1.0f : (wf32 ? static_cast<const float*>(w)[a] : (float)static_cast<const T*>(w)[a]);
}

// token_ptr null: the assignments of token n are n k .. n k + k - 1
template <typename T, int V>
__global__ __launch_bounds__(256) void k_rows_combine(long n_tokens, int chunks, int tpr_log2, int k, const int* __restrict__ token_ptr, const int* __restrict__ token_assign,
                                                      const int* __restrict__ rows, const void* __restrict__ w, int wf32, const T* __restrict__ src, long src_stride,
                                                      T* __restrict__ dst, long dst_stride) {
    typedef typename VecOf<T, V>::type VT;
    constexpr int U = 8;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long n = block_id() * rpb + (threadIdx.x >> tpr_log2);
    if (n >= n_tokens) return;
    const long j0 = token_ptr ? token_ptr[n] : n * k, j1 = token_ptr ? token_ptr[n + 1] : j0 + k;
    for (int c = threadIdx.x & (tpr - 1); c < chunks; c += tpr) {
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        for (long j = j0; j < j1; j += U) {                      // U rows in flight
            VT v[U];
            float wt[U];
            int row[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                row[u] = -1; wt[u] = 0.0f;
                if (j + u < j1) {
                    const int a = token_ptr ? token_assign[j + u] : (int)(j + u);
                    row[u] = rows[a];
                    wt[u] = weight_at<T>(w, wf32, a);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (row[u] >= 0) v[u] = *reinterpret_cast<const VT*>(src + row[u] * src_stride + (long)c * V);
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
        *reinterpret_cast<VT*>(dst + n * dst_stride + (long)c * V) = o;
    }
}

// d_src and / or d_w may be null.  tpr <= 64: a row's sum stays inside a wave
template <typename T, int V>
__global__ __launch_bounds__(256) void k_rows_back(long n_rows, int chunks, int tpr_log2, const int* __restrict__ assign, const int* __restrict__ row_token, const void* __restrict__ w,
                                                   int wf32, const T* __restrict__ dy, long dy_stride, const T* __restrict__ src, long src_stride, T* __restrict__ d_src,
                                                   long ds_stride, void* __restrict__ d_w) {
    typedef typename VecOf<T, V>::type VT;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const long p = block_id() * rpb + (threadIdx.x >> tpr_log2);
    const bool in = p < n_rows;
    const int a = in ? assign[p] : -1, tok = in ? row_token[p] : -1;
    const float wt = a >= 0 ? weight_at<T>(w, wf32, a) : 0.0f;
    float dot = 0.0f;
    for (int c = threadIdx.x & (tpr - 1); c < chunks; c += tpr) {
        if (!in) break;
        VT g, s, o;
        if (tok >= 0) {
            g = *reinterpret_cast<const VT*>(dy + tok * dy_stride + (long)c * V);
            if (d_w) s = *reinterpret_cast<const VT*>(src + p * src_stride + (long)c * V);
        }
        const T *ge = reinterpret_cast<const T*>(&g), *se = reinterpret_cast<const T*>(&s);
        T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            oe[i] = tok >= 0 ? (T)(wt * (float)ge[i]) : (T)0.0f;
            if (d_w && tok >= 0) dot += (float)ge[i] * (float)se[i];
        }
        if (d_src) *reinterpret_cast<VT*>(d_src + p * ds_stride + (long)c * V) = o;
    }
    if (!d_w) return;
    for (int o = tpr >> 1; o > 0; o >>= 1) dot += __shfl_xor(dot, o);
    if (in && (threadIdx.x & (tpr - 1)) == 0) {
        const int id = a >= 0 ? a : ~a;                          // (a dropped assignment's row lies behind the last active one: its weight's gradient is 0)
        if (wf32) static_cast<float*>(d_w)[id] = dot; else static_cast<T*>(d_w)[id] = (T)dot;
    }
}

// threads per row for `chunks` accesses: a power of two, at most `most`
inline int tpr_log2_for(long chunks, int most_log2) { int l = 0; while (l < most_log2 && (1l << l) < chunks) ++l; return l; }

int rows_gather(long n_rows, long row_bytes, const void* src, long src_stride, const int* row_token, void* dst, long dst_stride, hipStream_t s) {
    if (n_rows == 0 || row_bytes == 0) return 0;
    const int vb = common_align({(uint64_t)row_bytes, (uint64_t)(uintptr_t)src, (uint64_t)(uintptr_t)dst, (uint64_t)src_stride, (uint64_t)dst_stride});
    const long chunks = row_bytes / vb;
    const int l = tpr_log2_for(chunks, 8);
    const long per = 4 * (256 >> l);
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid_of(cdiv(n_rows, per)), dim3(256), 0, s, n_rows, (int)chunks, l, (const char*)src, src_stride, row_token, (char*)dst, dst_stride); };
    if (vb == 16) go(k_rows_gather<16, 4>);
    else if (vb == 8) go(k_rows_gather<8, 4>);
    else if (vb == 4) go(k_rows_gather<4, 4>);
    else go(k_rows_gather<2, 4>);
    LAUNCHED();
    return 0;
}

// elements per access that width, strides (in elements) and addresses allow
template <typename T>
int rows_vec(long width, std::initializer_list<const void*> ptrs, std::initializer_list<long> strides) {
    uint64_t m = (uint64_t)width * sizeof(T);
    for (const void* p : ptrs) m |= (uint64_t)(uintptr_t)p;
    for (long st : strides) m |= (uint64_t)st * sizeof(T);
    return common_align({m}) / (int)sizeof(T);
}
template <typename T, typename F>
void dispatch_vec(int v, F&& f) {
    if constexpr (sizeof(T) == 2) if (v == 8) return f(std::integral_constant<int, 8>{});
    if (v >= 4) return f(std::integral_constant<int, 4>{});
    if (v == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

template <typename T>
int rows_combine(long n_tokens, int width, int k, const int* token_ptr, const int* token_assign, const int* rows, const void* w, int wf32, const T* src, long src_stride, T* dst, long dst_stride, hipStream_t s) {
    if (n_tokens == 0 || width == 0) return 0;
    dispatch_vec<T>(rows_vec<T>(width, {src, dst}, {src_stride, dst_stride}), [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        const int chunks = width / V, l = tpr_log2_for(chunks, 8);
        hipLaunchKernelGGL((k_rows_combine<T, V>), grid_of(cdiv(n_tokens, 256 >> l)), dim3(256), 0, s, n_tokens, chunks, l, k, token_ptr, token_assign, rows, w, wf32, src, src_stride, dst, dst_stride);
    });
    LAUNCHED();
    return 0;
}

template <typename T>
int rows_back(long n_rows, int width, const int* assign, const int* row_token, const void* w, int wf32, const T* dy, long dy_stride, const T* src, long src_stride, T* d_src, long ds_stride,
              void* d_w, hipStream_t s) {
    if (n_rows == 0) return 0;
    dispatch_vec<T>(rows_vec<T>(width, {dy, src, d_src}, {dy_stride, src_stride, ds_stride}), [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        const int chunks = width / V, l = tpr_log2_for(chunks, 6);
        hipLaunchKernelGGL((k_rows_back<T, V>), grid_of(cdiv(n_rows, 256 >> l)), dim3(256), 0, s, n_rows, chunks, l, assign, row_token, w, wf32, dy, dy_stride, src, src_stride, d_src, ds_stride, d_w);
    });
    LAUNCHED();
    return 0;
}
