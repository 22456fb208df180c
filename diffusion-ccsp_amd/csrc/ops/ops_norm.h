// ops_norm.h -- the global norm of a list of tensors, and clipping by it.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
//
// norm = sqrt(sum over all elements of g^2); out = g min(1, max_norm / (norm + 1e-6)).  Squares and sums are held in 64 bits: a square of a
// 32-bit gradient leaves 32 bits' range at 1.8e19 and 1e-23, and a block's partial sum then needs no scaling.  (Two 64-bit operations
// an element are a few per cent of the time that the element's bytes take.)  Every block sums a fixed chunk of one tensor into its own place, one block adds the places in
// order: no atomics, the same value in every run.
//
// The tensor table travels in the kernel arguments, NORM_TENSORS a launch: no copy to the device, nothing that a captured graph
// would have to find again at replay but the addresses themselves.
constexpr int NORM_TENSORS = 112;
// Elements of a block.  Few elements are cut finer, so that there are blocks for every CU and short chains (300 odd tensors of 400000 elements in all: clip 8.0 -> 5.1 us a launch);
// many are not, because each block ends with a sum over its threads.
constexpr long NORM_FINE = 4096, NORM_COARSE = 16384, NORM_MANY = 1l << 26;
inline long norm_chunk_for(int count, const int64_t* n) {
    long total = 0;
    for (int i = 0; i < count; ++i) total += n[i];
    return total < NORM_MANY ? NORM_FINE : NORM_COARSE;
}

struct NormTable {
    const void* in[NORM_TENSORS];
    void* out[NORM_TENSORS];
    long n[NORM_TENSORS];
    int first[NORM_TENSORS + 1];                                 // first block of a tensor
    unsigned char type[NORM_TENSORS];
    int count, chunk;
};

// the tensor of block b: the number of first blocks <= b, less one (tensors without elements share their first block with the next)
__device__ __forceinline__ int norm_tensor(const NormTable& t, int b) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i = 0; i < NORM_TENSORS; i += 64) n += __popcll(__ballot(i + lane < t.count && t.first[i + lane < t.count ? i + lane : 0] <= b));
    return __builtin_amdgcn_readfirstlane(n - 1);
}

template <typename T>
__device__ __forceinline__ double norm_chunk(const T* p, long n) {
    constexpr int V = 16 / sizeof(T);
    typedef typename VecOf<T, V>::type VT;
    double s = 0.0;
    const long head_all = (16 - ((uintptr_t)p & 15) & 15) / sizeof(T), head = head_all < n ? head_all : n;
    if ((long)threadIdx.x < head) { const double v = (float)p[threadIdx.x]; s += v * v; }
    const VT* q = reinterpret_cast<const VT*>(p + head);
    const long nv = (n - head) / V;
    long i = threadIdx.x;
    for (; i + 768 < nv; i += 1024) {                            // four accesses in flight
        VT x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = q[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) { const double v = (float)x[u][j]; s += v * v; }
    }
    for (; i < nv; i += 256) {
        const VT x = q[i];
#pragma unroll
        for (int j = 0; j < V; ++j) { const double v = (float)x[j]; s += v * v; }
    }
    for (long t = head + nv * V + threadIdx.x; t < n; t += 256) { const double v = (float)p[t]; s += v * v; }
    return s;
}

__device__ __forceinline__ double block_sum(double s, double* part, int waves) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    double r = 0.0;
    for (int w = 0; w < waves; ++w) r += part[w];
    return r;
}

__global__ __launch_bounds__(256) void k_norm_part(NormTable t, double* part) {
    __shared__ double sums[4];
    const int i = norm_tensor(t, blockIdx.x);
    const long at = (long)(blockIdx.x - t.first[i]) * t.chunk;
    const long n = t.n[i] - at < t.chunk ? t.n[i] - at : t.chunk;
    double s;
    if (t.type[i] == CCSP_OPS_F32) s = norm_chunk(static_cast<const float*>(t.in[i]) + at, n);
    else if (t.type[i] == CCSP_OPS_BF16) s = norm_chunk(static_cast<const bf16*>(t.in[i]) + at, n);
    else s = norm_chunk(static_cast<const fp16*>(t.in[i]) + at, n);
    s = block_sum(s, sums, 4);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// norm[0] = the norm, scale[0] = the factor.  A norm that is not finite gives what the formula gives: factor 0 for infinity, NaN for NaN.
__global__ __launch_bounds__(1024) void k_norm_finish(const double* part, long n, double max_norm, float* norm, float* scale) {
    __shared__ double sums[16];
    double s = 0.0;
    for (long i = threadIdx.x; i < n; i += 16384) {              // sixteen loads in flight
        double v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) v[u] = i + 1024 * u < n ? part[i + 1024 * u] : 0.0;
#pragma unroll
        for (int u = 0; u < 16; ++u) s += v[u];
    }
    s = sqrt(block_sum(s, sums, 16));
    if (threadIdx.x == 0) {
        norm[0] = (float)s;
        const double c = max_norm / (s + 1e-6);
        if (scale) scale[0] = c >= 1.0 ? 1.0f : (float)c;        // (NaN compares false and stays)
    }
}

// (accesses start where p is a multiple of 16; o may lie otherwise)
template <typename T>
__device__ __forceinline__ void clip_chunk(const T* p, T* o, long n, float c) {
    constexpr int V = 16 / sizeof(T);
    typedef typename VecOf<T, V>::type VT;
    typedef typename LooseOf<T, V>::type OT;
    const long head_all = (16 - ((uintptr_t)p & 15) & 15) / sizeof(T), head = head_all < n ? head_all : n;
    if ((long)threadIdx.x < head) o[threadIdx.x] = (T)((float)p[threadIdx.x] * c);
    const VT* q = reinterpret_cast<const VT*>(p + head);
    OT* r = reinterpret_cast<OT*>(o + head);
    const long nv = (n - head) / V;
    long i = threadIdx.x;
    for (; i + 768 < nv; i += 1024) {                            // four accesses in flight
        VT x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = q[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[u][j] = (T)((float)x[u][j] * c);
            r[i + 256 * u] = x[u];
        }
    }
    for (; i < nv; i += 256) {
        VT x = q[i];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (T)((float)x[j] * c);
        r[i] = x;
    }
    for (long t = head + nv * V + threadIdx.x; t < n; t += 256) o[t] = (T)((float)p[t] * c);
}

__global__ __launch_bounds__(256) void k_norm_clip(NormTable t, int blocks, const float* scale) {
    const float c = scale[0];
    const int b = blocks - 1 - blockIdx.x;                       // a table from its end: with one table, what the norm read last is still in the last-level cache
    const int i = norm_tensor(t, b);
    if (c == 1.0f && t.in[i] == t.out[i]) return;                // g x 1 in place
    const long at = (long)(b - t.first[i]) * t.chunk;
    const long n = t.n[i] - at < t.chunk ? t.n[i] - at : t.chunk;
    if (t.type[i] == CCSP_OPS_F32) clip_chunk(static_cast<const float*>(t.in[i]) + at, static_cast<float*>(t.out[i]) + at, n, c);
    else if (t.type[i] == CCSP_OPS_BF16) clip_chunk(static_cast<const bf16*>(t.in[i]) + at, static_cast<bf16*>(t.out[i]) + at, n, c);
    else clip_chunk(static_cast<const fp16*>(t.in[i]) + at, static_cast<fp16*>(t.out[i]) + at, n, c);
}

// hands tables of at most NORM_TENSORS tensors that have elements to f(table, blocks, blocks before it), first to last.  (With several tables clip starts on the first, which
// the norm read longest ago.)
template <typename F>
int norm_tables(int count, const void* const* in, void* const* out, const int64_t* n, const int32_t* type, F&& f) {
    const long chunk = norm_chunk_for(count, n);
    long before = 0;
    for (int i = 0; i < count;) {
        NormTable t;
        int blocks = 0;
        t.count = 0;
        t.chunk = (int)chunk;
        for (; i < count && t.count < NORM_TENSORS; ++i) {
            if (n[i] == 0) continue;
            const long b = cdiv(n[i], chunk);
            if (b > 0x800000L) return fail("tensor %d has too many elements", i);
            if (t.count && blocks + b > 0x800000L) break;      // (a grid holds 2^32 threads)
            t.in[t.count] = in[i]; t.out[t.count] = out ? out[i] : nullptr; t.n[t.count] = n[i]; t.type[t.count] = (unsigned char)type[i];
            t.first[t.count++] = blocks;
            blocks += (int)b;
        }
        if (t.count == 0) break;
        if (f(t, blocks, before)) return 1;
        before += blocks;
    }
    return 0;
}
