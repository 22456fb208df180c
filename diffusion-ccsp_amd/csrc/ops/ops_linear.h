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
    void* sum;                                                   // [E, M]: sum over k of A (weight gradient: the bias gradient, or null)
    const int* offsets;
    int E, R, M, N, K;                                           // M, N, K of one expert's product; the one that is a row count is -1
    int silu;
    float* parts;                                                // weight gradient of experts with more than 2^seg_log2 rows: [slot][M N + M] partial sums
    int seg_log2;                                                // 31: no expert's rows are cut
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
__device__ __forceinline__ int count_tiles(const int* __restrict__ off, int E, int R, int tm_log2) {
    const int lane = threadIdx.x & 63, up = (1 << tm_log2) - 1;
    int n = 0;
    for (int i = lane; i <= E; i += 64) n += ((i < E ? off[i + 1] : R) - off[i] + up) >> tm_log2;
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    return __builtin_amdgcn_readfirstlane(n);
}
// most tiles of 2^l rows that R rows in E groups and a tail can have
inline long most_tiles(long R, long E, int l) { const long g = R < E + 1 ? R : E + 1; return (R >> l) + g; }

__device__ __forceinline__ float silu_value(float z) { return z / (1.0f + expf(-z)); }
__device__ __forceinline__ float silu_slope(float z) { const float s = 1.0f / (1.0f + expf(-z)); return s * (1.0f + z * (1.0f - s)); }

template <typename T> struct Vec8 { typedef T t __attribute__((ext_vector_type(8))); };
__device__ __forceinline__ f32x4 mfma16(Vec8<bf16>::t a, Vec8<bf16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Vec8<fp16>::t a, Vec8<fp16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// 16 bytes of a row of the operand along its contiguous side, `left` elements of it in range
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* p, int left) {
    constexpr int V = 16 / sizeof(T);
    union { T e[V]; u32x4 v; } x;
    x.v = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < left) x.e[i] = p[i];
    return x.v;
}

// ------------------------------------------------------------------------------------------------------------------------
// 16-bit types, rows of any alignment.  Tile 128 x 128 x 64, 4 waves as 2 x 2, each 64 x 64 as 4 x 4 tiles of v_mfma 16x16x32; the operands are handed over in exchanged roles
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

template <typename T, int PROD>
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
            if (AKC) { const int r = x >> 3, c = x & 7; ra[i] = load_piece<T>(A + (long)r * p.lda + k0 + 8 * c, r < left_m ? K - k0 - 8 * c : 0); }
            else { const int k = x >> 4, c = x & 15; ra[i] = load_piece<T>(A + (long)(k0 + k) * p.lda + 8 * c, k0 + k < K ? left_m - 8 * c : 0); }
            if (BKC) { const int r = x >> 3, c = x & 7; rb[i] = load_piece<T>(B + (long)r * p.ldb + k0 + 8 * c, r < left_n ? K - k0 - 8 * c : 0); }
            else { const int k = x >> 4, c = x & 15; rb[i] = load_piece<T>(B + (long)(k0 + k) * p.ldb + 8 * c, k0 + k < K ? left_n - 8 * c : 0); }
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bool sums = PROD == PROD_WEIGHT && p.sum && n0 + wn == 0;
    f32x4 sum[4] = {};
    typename Vec8<T>::t ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (T)1.0f;
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
            if (sums) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = mfma16(ones, fa[i], sum[i]);
            }
        }
    }
    T* C = static_cast<T*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    T* Z = PROD == PROD_FORWARD && p.z ? static_cast<T*>(p.z) + (long)r0 * p.ldc : nullptr;
    const T* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const T*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
    if (sums && lane < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (wm + 16 * i + lane < left_m) static_cast<T*>(p.sum)[(long)e * p.M + m0 + wm + 16 * i + lane] = (T)sum[i][0];
    }
    if (PROD == PROD_WEIGHT && !p.c) return;                     // (the sums alone)
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
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < N) { C[at + r] = y[r]; if (Z) Z[at + r] = z[r]; }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// 16-byte rows: the operands go from memory to LDS without passing a register (buffer_load ... lds), a stage ahead of the products.
// A lane's 16 bytes land at a fixed place of its wave's 1 KB, so the swizzle of a layout is made by choosing which bytes a lane asks for; what is out
// of range (rows past the group, columns past the matrix, k past its end) is asked for past the buffer's end and arrives as zeros.  The buffer's base
// advances with k, so that no offset inside it passes 31 bits however long a group is.
//
// A stage is 128 bytes of k: 64 values of 16 bits or 32 of 32 bits.  k contiguous: [R rows][8 pieces], piece c of row r at c ^ (r & 7), for every type.  k across
// rows, 16 bits: [64 k][R], 32-byte blocks at block ^ (k & 3 | (k >> 3 & 1) << 2) for the transposing read; 32 bits: [32 k][R], 128-byte blocks at block ^
// (k >> 2 & 1), because the two halves of a wave read k and k + 4.
//
// 32 bits use v_mfma_f32_32x32x2_f32 (products and sums in 32 bits throughout); its two k are taken 4 apart, so that a lane's k of four instructions are
// one 16-byte read where k is contiguous.
//
// TM x TN by WM x WN waves, two LDS stages.  A wave's TM / WM x TN / WN part decides how many LDS bytes a product costs: in 16 bits the LDS port is as
// busy as the matrix pipe at 64 x 64 and three quarters of it at 128 x 64.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lds_dma16(u32x4 rsrc, unsigned int offset, unsigned int lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
constexpr unsigned int DMA_OUT = 0x80000000u;                    // an offset past every buffer

// place of piece c in k row k (k across rows)
template <typename T> __device__ __forceinline__ int across_piece(int k, int c) {
    if (sizeof(T) == 4) return c ^ (k >> 2 & 1) << 3;
    const int f = (k & 3) | ((k >> 3 & 1) << 2);
    return ((c >> 1) ^ f) << 1 | (c & 1);
}

// one operand of a block: R rows (m or n) by K, staged 128 bytes of k at a time
template <typename T, bool KC, int R, int WAVES>
struct Stager {
    static constexpr int SK = 128 / sizeof(T);                   // k of a stage
    static constexpr int N = R * 128 / 1024 / WAVES;             // accesses of a wave per stage
    static_assert(N * 1024 * WAVES == R * 128, "the waves share a stage evenly");
    unsigned long base; long step;                               // bytes
    unsigned int off[N];
    int row_bytes, kk;                                           // KC: the lane's first k; else: bytes of a k row
    __device__ __forceinline__ void init(const void* p, long ld, int left) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        base = (unsigned long)p;
        row_bytes = (int)(ld * sizeof(T));
        step = KC ? 128 : SK * ld * (long)sizeof(T);
        constexpr int V = 16 / sizeof(T);
        kk = ((lane & 7) ^ (lane >> 3 & 7)) * V;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = wave * N + i;                         // the 1 KB piece of the stage
            if (KC) {
                const int r = at * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
                off[i] = r < left ? (unsigned int)(r * row_bytes + c * 16) : DMA_OUT;
            } else {
                constexpr int CH = R / V;                        // pieces of 16 bytes in a k row
                const int x = at * 64 + lane, k = x / CH, c = across_piece<T>(k, x % CH);      // (the swizzle is its own inverse)
                off[i] = V * c < left ? (unsigned int)(k * row_bytes + c * 16) : DMA_OUT;
            }
        }
    }
    // `left` > 0 of k from here on
    __device__ __forceinline__ void load(unsigned int lds, int left) {
        u32x4 r;
        r[0] = __builtin_amdgcn_readfirstlane((unsigned int)base);
        r[1] = __builtin_amdgcn_readfirstlane((unsigned int)(base >> 32) & 0xffffu);
        r[2] = KC ? 0x7fffffffu : (unsigned int)__builtin_amdgcn_readfirstlane((left < SK ? left : SK) * row_bytes);
        r[3] = 0x00020000u;
        const unsigned int to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * N * 1024);
        if (KC && left < SK) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds_dma16(r, kk < left ? off[i] : DMA_OUT, to + i * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) lds_dma16(r, off[i], to + i * 1024);
        }
        base += step;
    }
};

// 16 bits: the eight k of a lane (8 (lane >> 4) ..) of row r0 + (lane & 15), k step ks of 32
template <typename T, bool KC, int R>
__device__ __forceinline__ typename Vec8<T>::t stage_frag(const T* s, int r0, int ks) {
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
            x.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(s + k * R + (((r0 >> 4) ^ f) << 4) + 4 * (i & 3)));
        }
        return x.v;
    }
}
// 32 bits: k 8 ks + 4 (lane >> 5) .. + 3 of row r0 + (lane & 31)
template <bool KC, int R>
__device__ __forceinline__ f32x4 stage_frag32(const float* s, int r0, int ks) {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = r0 + (lane & 31);
    if constexpr (KC) {
        return *reinterpret_cast<const f32x4*>(s + r * 32 + (((2 * ks + h) ^ (r & 7)) << 2));
    } else {
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = s[(8 * ks + 4 * h + j) * R + (r ^ h << 5)];        // (k >> 2 & 1 is h)
        return v;
    }
}

// tile (m, n) of block b < tiles_m tiles_n: blocks b, b + 8, .. share an XCD and its L2, so each XCD takes a run of tiles, and the run goes through bands of
// 8 row tiles.  tiles_m is the number that there is, not the number that there might be: with empty tiles in it one XCD would get them all.
__device__ __forceinline__ void tile_order(int b, int tiles_m, int tiles_n, int* m, int* n) {
    const int blocks = tiles_m * tiles_n, per = blocks >> 3, rest = blocks & 7, x = b & 7;
    const int t = x * per + (x < rest ? x : rest) + (b >> 3);
    const int band = 8 * tiles_n, g = t / band, first = g * 8, h = tiles_m - first < 8 ? tiles_m - first : 8, in = t - g * band;
    *m = first + in % h;
    *n = in / h;
}

// Partial sums of segment i of an expert whose rows start at `first` and are more than 2^l: no two segments of experts that are cut share a slot.  (Their
// starts are more than 2^l apart, so first segments differ in first >> l; segment i > 0 has (first >> l) + i, which is at most (end >> l), and the
// next expert's second segment at least one more.)
__host__ __device__ __forceinline__ int seg_slot(int first, int i, int l) { return 2 * ((first >> l) + i) + (i > 0); }

template <int V> struct Log2 { static constexpr int v = 1 + Log2<V / 2>::v; };
template <> struct Log2<1> { static constexpr int v = 0; };

template <typename T, int PROD, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_prod_direct(ProdArgs p, int tiles_m, int tiles_n) {
    constexpr bool AKC = PROD != PROD_WEIGHT, BKC = PROD == PROD_FORWARD, F32 = sizeof(T) == 4;
    constexpr int G = F32 ? 32 : 16, FA = TM / WM / G, FB = TN / WN / G, RG = F32 ? 16 : 4;      // fragment side, fragments, result registers
    constexpr int SK = 128 / sizeof(T), STAGE = (TM + TN) * SK;
    typedef typename VecOf<float, RG>::type Acc;
    extern __shared__ __attribute__((aligned(16))) unsigned short lds[];
    const T* const sm = reinterpret_cast<const T*>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    int e, r0 = 0, r1 = 0, m0 = 0, M, K, tm, tn;
    float* part = nullptr;                                       // this block's partial sums, if its expert's rows are cut
    if (PROD == PROD_WEIGHT) {
        const int per = tiles_m * tiles_n, t = blockIdx.x / per; // (XCDs share the tiles of one segment: experts differ in length)
        tile_order(blockIdx.x - t * per, tiles_m, tiles_n, &tm, &tn);
        if (p.seg_log2 == 31) { e = t; r0 = p.offsets[e]; K = p.offsets[e + 1] - r0; }
        else {
            if (!find_tile(p.offsets, p.E, p.offsets[p.E], p.seg_log2, t, &e, &r0, &r1)) return;
            const int first = p.offsets[e], i = (r0 - first) >> p.seg_log2;
            K = r1 - r0 < 1 << p.seg_log2 ? r1 - r0 : 1 << p.seg_log2;
            if (r1 - first > 1 << p.seg_log2) part = p.parts + (long)seg_slot(first, i, p.seg_log2) * ((long)p.M * p.N + p.M);
        }
        m0 = tm * TM;
        M = p.M;
    } else {
        const int tiles = count_tiles(p.offsets, p.E, p.R, Log2<TM>::v);
        if (blockIdx.x >= tiles * tiles_n) return;
        tile_order(blockIdx.x, tiles, tiles_n, &tm, &tn);
        find_tile(p.offsets, p.E, p.R, Log2<TM>::v, tm, &e, &r0, &r1);
        M = r1 - r0 < TM ? r1 - r0 : TM; K = e < p.E ? p.K : 0;
    }
    const int n0 = tn * TN, N = p.N, left_m = M - m0;
    const T* A = static_cast<const T*>(p.a) + (PROD == PROD_WEIGHT ? (long)r0 * p.lda + m0 : (long)r0 * p.lda);
    const T* B = static_cast<const T*>(p.b) + (PROD == PROD_WEIGHT ? (long)r0 * p.ldb + n0 : e * p.b_expert + (BKC ? (long)n0 * p.ldb : (long)n0));
    Acc acc[FA][FB] = {};
    // the bias gradient (sum over k of A) is made on the way by the waves that hold the first columns of n: in 16 bits a product with a column of ones,
    // in 32 bits one addition beside each 64-cycle matrix instruction
    const bool sums = PROD == PROD_WEIGHT && p.sum && n0 + wn == 0;
    f32x4 sum16[FA] = {};
    float sum32[FA] = {};
    if (K > 0) {
        Stager<T, AKC, TM, WM * WN> ga;
        Stager<T, BKC, TN, WM * WN> gb;
        ga.init(A, p.lda, left_m);
        gb.init(B, p.ldb, N - n0);
        const unsigned int l0 = (unsigned int)(unsigned long)(__attribute__((address_space(3))) unsigned short*)lds;
        ga.load(l0, K);
        gb.load(l0 + TM * 128, K);
        auto loop = [&](auto with_sums) {
            constexpr bool S = decltype(with_sums)::value;
            int buf = 0;
            for (int k0 = 0; k0 < K; k0 += SK, buf ^= 1) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // this wave's part of the stage is there;
                __syncthreads();                                 // everyone's, and nobody reads the other stage any more
                if (k0 + SK < K) {
                    const unsigned int l1 = l0 + (buf ^ 1) * STAGE * (int)sizeof(T);
                    ga.load(l1, K - k0 - SK);
                    gb.load(l1 + TM * 128, K - k0 - SK);
                }
                const T *sA = sm + buf * STAGE, *sB = sA + TM * SK;
                if constexpr (F32) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        f32x4 fa[FA], fb[FB];
#pragma unroll
                        for (int j = 0; j < FB; ++j) fb[j] = stage_frag32<BKC, TN>(sB, wn + G * j, ks);
#pragma unroll
                        for (int i = 0; i < FA; ++i) fa[i] = stage_frag32<AKC, TM>(sA, wm + G * i, ks);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int i = 0; i < FA; ++i) {
#pragma unroll
                                for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j][k], fa[i][k], acc[i][j], 0, 0, 0);
                                if (S) sum32[i] += fa[i][k];
                            }
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        typename Vec8<T>::t fa[FA], fb[FB], ones;
#pragma unroll
                        for (int i = 0; i < 8; ++i) ones[i] = (T)1.0f;
#pragma unroll
                        for (int j = 0; j < FB; ++j) fb[j] = stage_frag<T, BKC, TN>(sB, wn + G * j, ks);
#pragma unroll
                        for (int i = 0; i < FA; ++i) fa[i] = stage_frag<T, AKC, TM>(sA, wm + G * i, ks);
#pragma unroll
                        for (int i = 0; i < FA; ++i) {
#pragma unroll
                            for (int j = 0; j < FB; ++j) acc[i][j] = mfma16(fb[j], fa[i], acc[i][j]);
                            if (S) sum16[i] = mfma16(ones, fa[i], sum16[i]);
                        }
                    }
                }
            }
        };
        if (PROD == PROD_WEIGHT && sums) loop(std::true_type{}); else loop(std::false_type{});
    }
    typedef typename VecOf<T, 4>::type V4;
    T* C = static_cast<T*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    T* Z = PROD == PROD_FORWARD && p.z ? static_cast<T*>(p.z) + (long)r0 * p.ldc : nullptr;
    const T* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const T*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
    if (sums) {
#pragma unroll
        for (int i = 0; i < FA; ++i) {
            const float v = F32 ? sum32[i] + __shfl_xor(sum32[i], 32) : sum16[i][0];
            const int m = wm + G * i + lane;
            if (lane < G && m < left_m) {
                if (part) part[(long)p.M * p.N + m0 + m] = v; else static_cast<T*>(p.sum)[(long)e * p.M + m0 + m] = (T)v;
            }
        }
    }
    if (PROD == PROD_WEIGHT && !p.c) return;                     // (the sums alone)
#pragma unroll
    for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int g = 0; g < RG / 4; ++g) {
            const int n = n0 + wn + G * j + (F32 ? 8 * g + 4 * (lane >> 5) : 4 * (lane >> 4));
            if (n >= N) continue;                                // (N is a multiple of 4: four columns are in or out together)
            float bv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (bias) {
#pragma unroll
                for (int r = 0; r < 4; ++r) bv[r] = (float)bias[n + r];
            }
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const int m = wm + G * i + (lane & (G - 1));
                if (m >= left_m) continue;
                if (PROD == PROD_WEIGHT && part) {
                    *reinterpret_cast<f32x4*>(part + (long)(m0 + m) * N + n) = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                    continue;
                }
                V4 y, z;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = acc[i][j][4 * g + r] + bv[r];
                    z[r] = (T)v;
                    y[r] = silu ? (T)silu_value(v) : (T)v;
                }
                *reinterpret_cast<V4*>(C + (long)m * p.ldc + n) = y;
                if (Z) *reinterpret_cast<V4*>(Z + (long)m * p.ldc + n) = z;
            }
        }
}

// ------------------------------------------------------------------------------------------------------------------------
// 32 bits, rows of any alignment.  Tile 64 x 64 x 32, 4 waves as 2 x 2.  LDS: k contiguous [64][33], else [32][68]: one word per lane and fragment, no two lanes on one bank.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int TS = 64, FK = 32, FLD_KC = FK + 1;
template <bool KC> __device__ __forceinline__ int f32_at(int r, int k) { return KC ? r * FLD_KC + k : k * (TS + 4) + r; }

template <int PROD>
__global__ __launch_bounds__(256) void k_prod32(ProdArgs p, int tiles_n) {
    constexpr bool AKC = PROD != PROD_WEIGHT, BKC = PROD == PROD_FORWARD;
    __shared__ __attribute__((aligned(16))) float sA[FK * (TS + 4)], sB[FK * (TS + 4)];
    constexpr int F = TS / 64, NP = TS / 32, CH = TS / 4;          // fragments of a wave's side, pieces of a thread, pieces of a k row
    static_assert(TS * FLD_KC <= FK * (TS + 4), "both layouts fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * (TS / 2), wn = (wave & 1) * (TS / 2);
    const int bid = blockIdx.x;
    int e, r0 = 0, r1 = 0, m0, n0, M, K;
    if (PROD == PROD_WEIGHT) {
        const int tiles_m = (p.M + TS - 1) / TS;
        e = bid / (tiles_m * tiles_n);
        const int t = bid - e * tiles_m * tiles_n;
        m0 = t / tiles_n * TS; n0 = t % tiles_n * TS; M = p.M;
        r0 = p.offsets[e]; K = p.offsets[e + 1] - r0;
    } else {
        if (!find_tile(p.offsets, p.E, p.R, 6, bid / tiles_n, &e, &r0, &r1)) return;
        m0 = 0; n0 = bid % tiles_n * TS; M = r1 - r0 < TS ? r1 - r0 : TS; K = e < p.E ? p.K : 0;
    }
    const int N = p.N;
    const float* A = static_cast<const float*>(p.a) + (PROD == PROD_WEIGHT ? (long)r0 * p.lda + m0 : (long)r0 * p.lda);
    const float* B = static_cast<const float*>(p.b) + (PROD == PROD_WEIGHT ? (long)r0 * p.ldb + n0 : e * p.b_expert + (BKC ? (long)n0 * p.ldb : (long)n0));
    const int left_m = M - m0, left_n = N - n0;
    u32x4 ra[NP], rb[NP];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int x = tid + 256 * i;
            if (AKC) { const int r = x >> 3, c = x & 7; ra[i] = load_piece<float>(A + (long)r * p.lda + k0 + 4 * c, r < left_m ? K - k0 - 4 * c : 0); }
            else { const int k = x / CH, c = x % CH; ra[i] = load_piece<float>(A + (long)(k0 + k) * p.lda + 4 * c, k0 + k < K ? left_m - 4 * c : 0); }
            if (BKC) { const int r = x >> 3, c = x & 7; rb[i] = load_piece<float>(B + (long)r * p.ldb + k0 + 4 * c, r < left_n ? K - k0 - 4 * c : 0); }
            else { const int k = x / CH, c = x % CH; rb[i] = load_piece<float>(B + (long)(k0 + k) * p.ldb + 4 * c, k0 + k < K ? left_n - 4 * c : 0); }
        }
    };
    auto put = [&](float* s, bool kc, int x, u32x4 v) {
        if (kc) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[(x >> 3) * FLD_KC + 4 * (x & 7) + j] = __uint_as_float(v[j]);
        } else *reinterpret_cast<u32x4*>(s + x / CH * (TS + 4) + 4 * (x % CH)) = v;
    };
    f32x16 acc[F][F], sum[F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            sum[i][r] = 0.0f;
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j][r] = 0.0f;
        }
    const bool sums = PROD == PROD_WEIGHT && p.sum && n0 + wn == 0;
    if (K > 0) load(0);
    for (int k0 = 0; k0 < K; k0 += FK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NP; ++i) { put(sA, AKC, tid + 256 * i, ra[i]); put(sB, BKC, tid + 256 * i, rb[i]); }
        __syncthreads();
        if (k0 + FK < K) load(k0 + FK);
#pragma unroll
        for (int k = 0; k < FK; k += 2) {
            float fa[F], fb[F];
#pragma unroll
            for (int i = 0; i < F; ++i) {
                fa[i] = sA[f32_at<AKC>(wm + 32 * i + (lane & 31), k + (lane >> 5))];
                fb[i] = sB[f32_at<BKC>(wn + 32 * i + (lane & 31), k + (lane >> 5))];
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j], fa[i], acc[i][j], 0, 0, 0);
            if (sums) {
#pragma unroll
                for (int i = 0; i < F; ++i) sum[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(1.0f, fa[i], sum[i], 0, 0, 0);
            }
        }
    }
    float* C = static_cast<float*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    float* Z = PROD == PROD_FORWARD && p.z ? static_cast<float*>(p.z) + (long)r0 * p.ldc : nullptr;
    const float* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const float*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
    if (sums && lane < 32) {
#pragma unroll
        for (int i = 0; i < F; ++i)
            if (wm + 32 * i + lane < left_m) static_cast<float*>(p.sum)[(long)e * p.M + m0 + wm + 32 * i + lane] = sum[i][0];
    }
    if (PROD == PROD_WEIGHT && !p.c) return;                     // (the sums alone)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = n0 + wn + 32 * j + 8 * g + 4 * (lane >> 5);
            float bv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[r] = bias && n + r < N ? bias[n + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < F; ++i) {
                const int m = wm + 32 * i + (lane & 31);
                if (m >= left_m || n >= N) continue;
                f32x4 y, z;
#pragma unroll
                for (int r = 0; r < 4; ++r) { z[r] = acc[i][j][4 * g + r] + bv[r]; y[r] = silu ? silu_value(z[r]) : z[r]; }
                const long at = (long)m * p.ldc + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < N) { C[at + r] = y[r]; if (Z) Z[at + r] = z[r]; }
            }
        }
}

// The weight gradient of experts whose rows were cut, their segments' partial sums added in order; zeros for experts without rows (they have no
// segment); the rest is there already.  x: 1024 values of M N and M, y: expert
template <typename T>
__global__ __launch_bounds__(256) void k_join_parts(ProdArgs p) {
    const int e = blockIdx.y, first = p.offsets[e], n = p.offsets[e + 1] - first, l = p.seg_log2;
    if (n > 0 && n <= 1 << l) return;
    const long mn = (long)p.M * p.N, all = mn + (p.sum ? p.M : 0);
    const int segs = (n + (1 << l) - 1) >> l;
    typedef typename VecOf<T, 4>::type V4;
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < all; i += (long)gridDim.x * 1024) {       // (M N and M are multiples of 4)
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < segs; ++k) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p.parts + (long)seg_slot(first, k, l) * (mn + p.M) + i);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += a[r];
        }
        V4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (T)v[r];
        if (i < mn) { if (p.c) *reinterpret_cast<V4*>(static_cast<T*>(p.c) + e * p.c_expert + i) = o; }
        else {
#pragma unroll
            for (int r = 0; r < 4; ++r) static_cast<T*>(p.sum)[(long)e * p.M + i - mn + r] = o[r];
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

template <typename T, int PROD, int TM, int TN, int WM, int WN>
int launch_direct(const ProdArgs& p, hipStream_t s) {
    const long tn = cdiv(p.N, TN), tm = PROD == PROD_WEIGHT ? cdiv(p.M, TM) : most_tiles(p.R, p.E, Log2<TM>::v);
    const bool cut = PROD == PROD_WEIGHT && p.seg_log2 != 31;
    const long blocks = (PROD == PROD_WEIGHT ? (cut ? most_tiles(p.R, p.E, p.seg_log2) : p.E) : 1) * tm * tn;
    if (blocks > 0x003fffffL) return fail("expert_linear: %ld tiles are more than a launch holds", blocks);
    if (blocks) hipLaunchKernelGGL((k_prod_direct<T, PROD, TM, TN, WM, WN>), dim3((unsigned)blocks), dim3(64 * WM * WN), 2 * (TM + TN) * 128, s, p, (int)tm, (int)tn);
    if (cut) {
        const long per = cdiv((long)p.M * p.N + p.M, 1024);
        hipLaunchKernelGGL(k_join_parts<T>, dim3((unsigned)(per < 1024 ? per : 1024), p.E), dim3(256), 0, s, p);
    }
    LAUNCHED();
    return 0;
}

template <typename K>
int launch_any(K kernel, const ProdArgs& p, bool weight, int ts_log2, hipStream_t s) {
    const long tn = cdiv(p.N, 1 << ts_log2), blocks = weight ? (long)p.E * cdiv(p.M, 1 << ts_log2) * tn : most_tiles(p.R, p.E, ts_log2) * tn;
    if (blocks > 0x00ffffffL) return fail("expert_linear: %ld tiles are more than a launch holds", blocks);
    if (blocks == 0) return 0;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, s, p, (int)tn);
    LAUNCHED();
    return 0;
}

// The tile of a product: 256 x 256 where there are enough of them to go round the CUs a few times (E: groups, for the weight gradient with tiles of its own)
template <typename T>
bool prod_big(bool weight, long R, long E, long M, long N) { return sizeof(T) == 2 && (weight ? E * cdiv(M, 256) : most_tiles(R, E, 8)) * cdiv(N, 256) >= 1024; }

// Rows of a segment of the weight gradient (log2; 31: uncut).  An expert's tile is one block's chain over all of its rows, so a few long experts would
// leave most CUs idle: rows are cut until there are about four blocks a CU.  A segment's partial sums cost 8 bytes a value to write and add, which
// its products have to be worth.
template <typename T>
int seg_log2_for(long R, long E, long M, long N) {
    if (prod_big<T>(true, R, E, M, N)) return 31;
    constexpr int TS = sizeof(T) == 4 ? 64 : 128, least = sizeof(T) == 4 ? 9 : 10;
    const long want = R * cdiv(M, TS) * cdiv(N, TS) / 1024;
    int l = least;
    while (l < 30 && (2l << l) <= want) ++l;
    return (1l << l) >= R ? 31 : l;
}

template <typename T, int PROD>
bool prod_direct(const ProdArgs& p) {
    constexpr int V = 16 / sizeof(T);
    // every address and stride a multiple of 16 bytes, no piece that is partly out, an offset inside a stage below 2^31
    return common_align({(uint64_t)(uintptr_t)p.a, (uint64_t)(uintptr_t)p.b, (uint64_t)(uintptr_t)p.c, (uint64_t)(uintptr_t)p.z, (uint64_t)p.lda * sizeof(T), (uint64_t)p.ldb * sizeof(T),
                         (uint64_t)p.ldc * sizeof(T)}) == 16 &&
           p.N % V == 0 && (PROD == PROD_WEIGHT ? p.M % V == 0 : p.K % V == 0) && p.lda < (1 << 21) && p.ldb < (1 << 21);
}

template <typename T, int PROD>
int launch_prod(const ProdArgs& p, hipStream_t s) {
    constexpr bool W = PROD == PROD_WEIGHT;
    if constexpr (sizeof(T) == 4) {
        if (prod_direct<T, PROD>(p)) return launch_direct<T, PROD, 64, 64, 2, 2>(p, s);
        return launch_any(k_prod32<PROD>, p, W, 6, s);
    } else {
        if (prod_direct<T, PROD>(p)) return prod_big<T>(W, p.R, p.E, p.M, p.N) ? launch_direct<T, PROD, 256, 256, 2, 4>(p, s) : launch_direct<T, PROD, 128, 128, 2, 2>(p, s);
        return launch_any(k_prod16<T, PROD>, p, W, 7, s);
    }
}
