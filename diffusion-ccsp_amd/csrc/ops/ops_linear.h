// ops_linear.h -- the experts' products: y = act(x W[e]^T + b[e]) over the rows of every expert, and the three products of its gradient.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
//
// All three are C(m, n) = sum over k of A(m, k) B(n, k) per expert:
//   forward          m = row, n = output, k = input      A = x (k contiguous)      B = W[e] (k contiguous)
//   input gradient   m = row, n = input,  k = output     A = dz (k contiguous)     B = W[e] (n contiguous)
//   weight gradient  m = output, n = input, k = row      A = dz (m contiguous)     B = x (n contiguous)
// Row groups are ragged and known on the device only: a block takes tile t, finds its expert from the first rows (find_tile) and leaves
// if there are fewer tiles.  The rows behind the last group are a group of their own whose tiles are written as zeros.

enum { PROD_FORWARD = 0, PROD_INPUT = 1, PROD_WEIGHT = 2 };

struct ProdArgs {
    const void* a; long lda;                                     // strides in elements
    const void* b; long ldb, b_expert;
    const void* bias;                                            // [E, N] or null
    void* c; long ldc, c_expert;
    void* z;                                                     // pre-activation (forward, or null)
    const int* offsets;
    int E, R, M, N, K;                                           // M, N, K of one expert's product; the one that is a row count is -1
    int silu;
};

// group g in [0, E] (E: the rows behind the last one), first row and end of tile t's rows; false if there is no tile t.  Every lane of the
// wave takes part; the result is the same in all.
__device__ __forceinline__ bool find_tile(const int* __restrict__ off, int E, int R, int tm_log2, int t, int* g, int* r0, int* r1) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int g0 = 0; g0 <= E; g0 += 64) {
        const int i = g0 + lane;
        const int lo = i <= E ? off[i] : 0, hi = i < E ? off[i + 1] : (i == E ? R : 0);
        const int own = (hi - lo + (1 << tm_log2) - 1) >> tm_log2;
        int v = own;
        for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o); v += lane >= o ? u : 0; }
        const unsigned long long past = __ballot(before + v > t);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int start = __shfl(lo, l), end = __shfl(hi, l), first = before + __shfl(v - own, l);
            *g = __builtin_amdgcn_readfirstlane(g0 + l);
            *r0 = __builtin_amdgcn_readfirstlane(start + ((t - first) << tm_log2));
            *r1 = __builtin_amdgcn_readfirstlane(end);
            return true;
        }
        before += __shfl(v, 63);
    }
    return false;
}
// most tiles of 2^l rows that R rows in E groups and a tail can have
inline long most_tiles(long R, long E, int l) { const long g = R < E + 1 ? R : E + 1; return (R >> l) + g; }

__device__ __forceinline__ float silu_value(float z) { return z / (1.0f + expf(-z)); }
__device__ __forceinline__ float silu_slope(float z) { const float s = 1.0f / (1.0f + expf(-z)); return s * (1.0f + z * (1.0f - s)); }

template <typename T> struct Vec8 { typedef T t __attribute__((ext_vector_type(8))); };
__device__ __forceinline__ f32x4 mfma16(Vec8<bf16>::t a, Vec8<bf16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Vec8<fp16>::t a, Vec8<fp16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// eight (16-bit) or four (32-bit) elements of a row of the operand, along its contiguous side; WIDE: strides, addresses and extents let a 16-byte access
// do, and a piece is in or out as a whole
template <typename T, bool WIDE>
__device__ __forceinline__ u32x4 load_piece(const T* p, int left) {
    constexpr int V = 16 / sizeof(T);
    if (WIDE) return left > 0 ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
    union { T e[V]; u32x4 v; } x;
    x.v = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < left) x.e[i] = p[i];
    return x.v;
}

// ------------------------------------------------------------------------------------------------------------------------
// 16-bit types.  Tile 128 x 128 x 64, 4 waves as 2 x 2, each 64 x 64 as 4 x 4 tiles of v_mfma 16x16x32; the operands are handed over in exchanged roles
// (n on the rows of the result), so that a lane holds four consecutive n of one m and stores them as one access.
// LDS holds an operand in pieces of 16 bytes.  k contiguous: [128 rows][8 pieces], piece c of row r at c ^ (r & 7): the 16 lanes of a fragment
// read touch every bank alike.  k across rows: [64 k][128], read by ds_read_tr16_b64, which hands lane i of 16 the column i of a 4 x 16 block; the
// block's 32 bytes sit at (column / 16) ^ (k & 3 | (k >> 3 & 1) << 2), so that the 16 row segments of an access spread over the banks.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int PT = 128, PK = 64;

template <bool KC> __device__ __forceinline__ int lds_piece(int row, int c) {      // element index of piece c of row `row` (KC: row = m or n; else row = k)
    if (KC) return row * PK + ((c ^ (row & 7)) << 3);
    const int f = (row & 3) | ((row >> 3 & 1) << 2);
    return row * PT + ((((c >> 1) ^ f) << 1 | (c & 1)) << 3);
}

template <typename T, bool KC>
__device__ __forceinline__ typename Vec8<T>::t lds_frag(const T* s, int r0, int ks) {
    typedef typename Vec8<T>::t V8;
    const int lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
    if constexpr (KC) {
        return *reinterpret_cast<const V8*>(s + lds_piece<true>(r0 + i, ks * 4 + q));
    } else {
        typedef __attribute__((address_space(3))) s16x4* P;
        union { s16x4 h[2]; V8 v; } x;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 32 * ks + 8 * q + 4 * h + (i >> 2), f = (k & 3) | ((k >> 3 & 1) << 2);
            x.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(s + k * PT + (((r0 >> 4) ^ f) << 4) + 4 * (i & 3)));
        }
        return x.v;
    }
}

template <typename T, int PROD, bool WIDE>
__global__ __launch_bounds__(256) void k_prod16(ProdArgs p, int tiles_n) {
    constexpr bool AKC = PROD != PROD_WEIGHT, BKC = PROD == PROD_FORWARD;
    __shared__ __attribute__((aligned(16))) T sA[PT * PK], sB[PT * PK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const int bid = blockIdx.x;
    int e, r0 = 0, r1 = 0, m0, n0, M, K;
    if (PROD == PROD_WEIGHT) {
        const int tiles_m = (p.M + PT - 1) / PT;
        e = bid / (tiles_m * tiles_n);
        const int t = bid - e * tiles_m * tiles_n;
        m0 = t / tiles_n * PT; n0 = t % tiles_n * PT; M = p.M;
        r0 = p.offsets[e]; K = p.offsets[e + 1] - r0;
    } else {
        if (!find_tile(p.offsets, p.E, p.R, 7, bid / tiles_n, &e, &r0, &r1)) return;
        m0 = 0; n0 = bid % tiles_n * PT; M = r1 - r0 < PT ? r1 - r0 : PT; K = e < p.E ? p.K : 0;
    }
    const int N = p.N;
    const T* A = static_cast<const T*>(p.a) + (PROD == PROD_WEIGHT ? (long)r0 * p.lda + m0 : (long)r0 * p.lda);
    const T* B = static_cast<const T*>(p.b) + (PROD == PROD_WEIGHT ? (long)r0 * p.ldb + n0 : e * p.b_expert + (BKC ? (long)n0 * p.ldb : (long)n0));
    const int left_m = M - m0, left_n = N - n0;
    u32x4 ra[4], rb[4];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = tid + 256 * i;
            if (AKC) { const int r = x >> 3, c = x & 7; ra[i] = load_piece<T, WIDE>(A + (long)r * p.lda + k0 + 8 * c, r < left_m ? K - k0 - 8 * c : 0); }
            else { const int k = x >> 4, c = x & 15; ra[i] = load_piece<T, WIDE>(A + (long)(k0 + k) * p.lda + 8 * c, k0 + k < K ? left_m - 8 * c : 0); }
            if (BKC) { const int r = x >> 3, c = x & 7; rb[i] = load_piece<T, WIDE>(B + (long)r * p.ldb + k0 + 8 * c, r < left_n ? K - k0 - 8 * c : 0); }
            else { const int k = x >> 4, c = x & 15; rb[i] = load_piece<T, WIDE>(B + (long)(k0 + k) * p.ldb + 8 * c, k0 + k < K ? left_n - 8 * c : 0); }
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (K > 0) load(0);
    for (int k0 = 0; k0 < K; k0 += PK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = tid + 256 * i;
            *reinterpret_cast<u32x4*>(sA + (AKC ? lds_piece<true>(x >> 3, x & 7) : lds_piece<false>(x >> 4, x & 15))) = ra[i];
            *reinterpret_cast<u32x4*>(sB + (BKC ? lds_piece<true>(x >> 3, x & 7) : lds_piece<false>(x >> 4, x & 15))) = rb[i];
        }
        __syncthreads();
        if (k0 + PK < K) load(k0 + PK);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            typename Vec8<T>::t fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { fa[i] = lds_frag<T, AKC>(sA, wm + 16 * i, ks); fb[i] = lds_frag<T, BKC>(sB, wn + 16 * i, ks); }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma16(fb[j], fa[i], acc[i][j]);
        }
    }
    T* C = static_cast<T*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    T* Z = PROD == PROD_FORWARD && p.z ? static_cast<T*>(p.z) + (long)r0 * p.ldc : nullptr;
    const T* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const T*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = n0 + wn + 16 * j + 4 * (lane >> 4);
        float bv[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) bv[r] = bias && n + r < N ? (float)bias[n + r] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = wm + 16 * i + (lane & 15);
            if (m >= left_m || n >= N) continue;
            typename VecOf<T, 4>::type y, z;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = acc[i][j][r] + bv[r];
                z[r] = (T)v;
                y[r] = silu ? (T)silu_value(v) : (T)v;
            }
            const long at = (long)m * p.ldc + n;
            if (WIDE) {                                          // (N is a multiple of 8 and n of 4)
                *reinterpret_cast<typename VecOf<T, 4>::type*>(C + at) = y;
                if (Z) *reinterpret_cast<typename VecOf<T, 4>::type*>(Z + at) = z;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < N) { C[at + r] = y[r]; if (Z) Z[at + r] = z[r]; }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// 32 bits: v_mfma_f32_32x32x2_f32, products and sums in 32 bits throughout.  Tile 128 x 128 x 32, 4 waves as 2 x 2, each 64 x 64 as 2 x 2.
// LDS: k contiguous [128][33], else [32][132]: one word per lane and fragment, no two lanes on one bank.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int FK = 32, FLD_KC = FK + 1, FLD_NC = PT + 4;
template <bool KC> __device__ __forceinline__ int f32_at(int r, int k) { return KC ? r * FLD_KC + k : k * FLD_NC + r; }

template <int PROD, bool WIDE>
__global__ __launch_bounds__(256) void k_prod32(ProdArgs p, int tiles_n) {
    constexpr bool AKC = PROD != PROD_WEIGHT, BKC = PROD == PROD_FORWARD;
    __shared__ __attribute__((aligned(16))) float sA[PT * FLD_KC], sB[PT * FLD_KC];
    static_assert(FK * FLD_NC <= PT * FLD_KC, "both layouts fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const int bid = blockIdx.x;
    int e, r0 = 0, r1 = 0, m0, n0, M, K;
    if (PROD == PROD_WEIGHT) {
        const int tiles_m = (p.M + PT - 1) / PT;
        e = bid / (tiles_m * tiles_n);
        const int t = bid - e * tiles_m * tiles_n;
        m0 = t / tiles_n * PT; n0 = t % tiles_n * PT; M = p.M;
        r0 = p.offsets[e]; K = p.offsets[e + 1] - r0;
    } else {
        if (!find_tile(p.offsets, p.E, p.R, 7, bid / tiles_n, &e, &r0, &r1)) return;
        m0 = 0; n0 = bid % tiles_n * PT; M = r1 - r0 < PT ? r1 - r0 : PT; K = e < p.E ? p.K : 0;
    }
    const int N = p.N;
    const float* A = static_cast<const float*>(p.a) + (PROD == PROD_WEIGHT ? (long)r0 * p.lda + m0 : (long)r0 * p.lda);
    const float* B = static_cast<const float*>(p.b) + (PROD == PROD_WEIGHT ? (long)r0 * p.ldb + n0 : e * p.b_expert + (BKC ? (long)n0 * p.ldb : (long)n0));
    const int left_m = M - m0, left_n = N - n0;
    u32x4 ra[4], rb[4];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = tid + 256 * i;
            if (AKC) { const int r = x >> 3, c = x & 7; ra[i] = load_piece<float, WIDE>(A + (long)r * p.lda + k0 + 4 * c, r < left_m ? K - k0 - 4 * c : 0); }
            else { const int k = x >> 5, c = x & 31; ra[i] = load_piece<float, WIDE>(A + (long)(k0 + k) * p.lda + 4 * c, k0 + k < K ? left_m - 4 * c : 0); }
            if (BKC) { const int r = x >> 3, c = x & 7; rb[i] = load_piece<float, WIDE>(B + (long)r * p.ldb + k0 + 4 * c, r < left_n ? K - k0 - 4 * c : 0); }
            else { const int k = x >> 5, c = x & 31; rb[i] = load_piece<float, WIDE>(B + (long)(k0 + k) * p.ldb + 4 * c, k0 + k < K ? left_n - 4 * c : 0); }
        }
    };
    auto put = [&](float* s, bool kc, int x, u32x4 v) {
        if (kc) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[(x >> 3) * FLD_KC + 4 * (x & 7) + j] = __uint_as_float(v[j]);
        } else *reinterpret_cast<u32x4*>(s + (x >> 5) * FLD_NC + 4 * (x & 31)) = v;
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (K > 0) load(0);
    for (int k0 = 0; k0 < K; k0 += FK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) { put(sA, AKC, tid + 256 * i, ra[i]); put(sB, BKC, tid + 256 * i, rb[i]); }
        __syncthreads();
        if (k0 + FK < K) load(k0 + FK);
#pragma unroll
        for (int k = 0; k < FK; k += 2) {
            float fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = sA[f32_at<AKC>(wm + 32 * i + (lane & 31), k + (lane >> 5))];
                fb[i] = sB[f32_at<BKC>(wn + 32 * i + (lane & 31), k + (lane >> 5))];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }
    float* C = static_cast<float*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    float* Z = PROD == PROD_FORWARD && p.z ? static_cast<float*>(p.z) + (long)r0 * p.ldc : nullptr;
    const float* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const float*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = n0 + wn + 32 * j + 8 * g + 4 * (lane >> 5);
            float bv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[r] = bias && n + r < N ? bias[n + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = wm + 32 * i + (lane & 31);
                if (m >= left_m || n >= N) continue;
                f32x4 y, z;
#pragma unroll
                for (int r = 0; r < 4; ++r) { z[r] = acc[i][j][4 * g + r] + bv[r]; y[r] = silu ? silu_value(z[r]) : z[r]; }
                const long at = (long)m * p.ldc + n;
                if (WIDE) {
                    *reinterpret_cast<f32x4*>(C + at) = y;
                    if (Z) *reinterpret_cast<f32x4*>(Z + at) = z;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < N) { C[at + r] = y[r]; if (Z) Z[at + r] = z[r]; }
                }
            }
        }
}

// ---- around the products -------------------------------------------------------------------------------------------------
// dz = dy silu'(z) over the active rows (z as it was stored: its rounding moves the slope by less than dz's own rounding does)
template <typename T, int V>
__global__ __launch_bounds__(256) void k_silu_back(const int* __restrict__ active, int chunks, const T* __restrict__ dy, long dy_stride, const T* __restrict__ z, T* __restrict__ dz) {
    typedef typename VecOf<T, V>::type VT;
    const long n = (long)active[0] * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / chunks, c = i - r * chunks;
        const VT g = *reinterpret_cast<const VT*>(dy + r * dy_stride + c * V), zz = *reinterpret_cast<const VT*>(z + i * V);
        const T *ge = reinterpret_cast<const T*>(&g), *ze = reinterpret_cast<const T*>(&zz);
        VT o;
        T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int j = 0; j < V; ++j) oe[j] = (T)((float)ge[j] * silu_slope((float)ze[j]));
        *reinterpret_cast<VT*>(dz + i * V) = o;
    }
}

// db[e] = sum of dz over the expert's rows: 64 columns a block, four interleaved sums of rows joined in order
template <typename T>
__global__ __launch_bounds__(256) void k_bias_back(const int* __restrict__ offsets, int O, const T* __restrict__ dz, long stride, T* __restrict__ db) {
    __shared__ float part[4][64];
    const int e = blockIdx.y, n = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
    const int r1 = offsets[e + 1];
    float s = 0.0f;
    if (n < O) for (int r = offsets[e] + w; r < r1; r += 4) s += (float)dz[r * stride + n];
    part[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && n < O) db[(long)e * O + n] = (T)(((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x]);
}

template <typename T, int PROD>
int launch_prod(const ProdArgs& p, hipStream_t s) {
    const int tn = (int)cdiv(p.N, PT);
    const long blocks = PROD == PROD_WEIGHT ? (long)p.E * cdiv(p.M, PT) * tn : most_tiles(p.R, p.E, 7) * tn;
    if (blocks > 0x00ffffffL) return fail("expert_linear: %ld tiles are more than a launch holds", blocks);
    if (blocks == 0) return 0;
    constexpr int V = 16 / sizeof(T);
    // 16-byte accesses: every address and stride a multiple of 16 bytes, and no piece that is partly out
    const bool wide = common_align({(uint64_t)(uintptr_t)p.a, (uint64_t)(uintptr_t)p.b, (uint64_t)(uintptr_t)p.c, (uint64_t)(uintptr_t)p.z, (uint64_t)p.lda * sizeof(T), (uint64_t)p.ldb * sizeof(T),
                                    (uint64_t)p.ldc * sizeof(T)}) == 16 && p.N % V == 0 && (PROD == PROD_WEIGHT ? p.M % V == 0 : p.K % V == 0);
    if constexpr (sizeof(T) == 4) {
        if (wide) hipLaunchKernelGGL((k_prod32<PROD, true>), dim3((unsigned)blocks), dim3(256), 0, s, p, tn);
        else hipLaunchKernelGGL((k_prod32<PROD, false>), dim3((unsigned)blocks), dim3(256), 0, s, p, tn);
    } else {
        if (wide) hipLaunchKernelGGL((k_prod16<T, PROD, true>), dim3((unsigned)blocks), dim3(256), 0, s, p, tn);
        else hipLaunchKernelGGL((k_prod16<T, PROD, false>), dim3((unsigned)blocks), dim3(256), 0, s, p, tn);
    }
    LAUNCHED();
    return 0;
}
