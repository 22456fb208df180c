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
    int pieces;                                                  // elements of a result's row that one access may take: 8, 4 or 1
    int past;                                                    // the results pass the last-level cache by (in whole pieces)
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

// sigmoid: in 32 bits by expf and a true division; for results of 16 bits by the hardware's exponential and reciprocal, whose 2^-22 is a thousandth of the
// result's own rounding and whose few instructions an epilogue notices (8192 rows, 32 experts of 2048 -> 1408: the forward product 115 -> 77 us)
template <typename T> __device__ __forceinline__ float sigmoid_of(float z) {
    if (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
template <typename T> __device__ __forceinline__ float silu_value(float z) { return sizeof(T) == 4 ? z / (1.0f + expf(-z)) : z * sigmoid_of<T>(z); }
template <typename T> __device__ __forceinline__ float silu_slope(float z) { const float s = sigmoid_of<T>(z); return s * (1.0f + z * (1.0f - s)); }

// A pre-activation as it is kept for the gradient: one that is finite in 32 bits stays finite in the type, or the slope of silu, 0 or 1 that far out, would be NaN (0 x inf).
// (An infinite one stays what it is: the formula's NaN.)
template <typename T> __device__ __forceinline__ T kept_value(float v) {
    if constexpr (sizeof(T) == 4) return v;
    constexpr float most = std::is_same<T, fp16>::value ? 65504.0f : 0x1.fep127f;
    return (T)(v - v == 0.0f ? __builtin_amdgcn_fmed3f(v, -most, most) : v);
}

template <typename T> struct Vec8 { typedef T t __attribute__((ext_vector_type(8))); };
__device__ __forceinline__ f32x4 mfma16(Vec8<bf16>::t a, Vec8<bf16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Vec8<fp16>::t a, Vec8<fp16>::t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// ------------------------------------------------------------------------------------------------------------------------
// The operands go from memory to LDS without passing a register (buffer_load ... lds), NST - 1 stages ahead of the products.  Their rows are whole 16-byte
// pieces at multiples of 16 bytes; rows that are not are copied and padded first (k_pad_rows).
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
// TM x TN by WM x WN waves.  A wave's TM / WM x TN / WN part decides how many LDS bytes a product costs: at 128 x 64 (256 x 256 by 2 x 4) in 16 bits the
// LDS is busy 23 % of the time and the matrix pipe 60.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lds_dma16(u32x4 rsrc, unsigned int offset, unsigned int lds) {
    // (five wait states between a vector instruction's scalar result, as the descriptor may be one, and the load: the compiler does not see the load)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory", "m0");
}
constexpr unsigned int DMA_OUT = 0x80000000u;                    // an offset past every buffer

// 16 bits, k across rows: which 32-byte block a block of k row k goes to (R / 16 blocks a row)
template <int R> __device__ __forceinline__ int block_swizzle(int k) { return ((k & 3) | ((k >> 3 & 1) << 2)) & (R / 16 - 1); }
// place of piece c in k row k (k across rows)
template <typename T, int R> __device__ __forceinline__ int across_piece(int k, int c) {
    if (sizeof(T) == 4) return c ^ (k >> 2 & 1) << 3;
    return ((c >> 1) ^ block_swizzle<R>(k)) << 1 | (c & 1);
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
                const int x = at * 64 + lane, k = x / CH, c = across_piece<T, R>(k, x % CH);      // (the swizzle is its own inverse)
                off[i] = V * c < left ? (unsigned int)(k * row_bytes + c * 16) : DMA_OUT;
            }
        }
    }
    __device__ __forceinline__ u32x4 rsrc(int k) const {         // k of the stage are there
        u32x4 r;
        r[0] = __builtin_amdgcn_readfirstlane((unsigned int)base);
        r[1] = __builtin_amdgcn_readfirstlane((unsigned int)(base >> 32) & 0xffffu);
        r[2] = KC ? 0x7fffffffu : (unsigned int)__builtin_amdgcn_readfirstlane(k * row_bytes);
        r[3] = 0x00020000u;
        return r;
    }
    __device__ __forceinline__ unsigned int place(unsigned int lds) const { return __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * N * 1024); }
    // the next stage to LDS address `lds`: `left` > 0 of k from here on
    __device__ __forceinline__ void load(unsigned int lds, int left) {
        const u32x4 r = rsrc(left < SK ? left : SK);
        const unsigned int to = place(lds);
        if (KC && left < SK) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds_dma16(r, kk < left ? off[i] : DMA_OUT, to + i * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) lds_dma16(r, off[i], to + i * 1024);
        }
        base += step;
    }
    // the same piece by piece without a branch, i = 0 .. N - 1 in turn; left may be <= 0
    __device__ __forceinline__ void load_piece(unsigned int lds, int left, int i) {
        const int k = left < SK ? left : SK;
        lds_dma16(rsrc(left > 0 ? k : 0), !KC || kk < left ? off[i] : DMA_OUT, place(lds) + i * 1024);
        if (i == N - 1) base += step;
    }
};

// 16 bits: the eight k of a lane (8 (lane >> 4) ..) of row r0 + (lane & 15), k step ks of 32
template <typename T, bool KC, int R>
__device__ __forceinline__ typename Vec8<T>::t stage_frag(const T* s, int r0, int ks) {
    typedef typename Vec8<T>::t V8;
    const int lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
    if constexpr (KC) {
        const int r = r0 + i;
        return *reinterpret_cast<const V8*>(s + r * 64 + (((ks * 4 + q) ^ (r & 7)) << 3));
    } else {
        typedef __attribute__((address_space(3))) s16x4* P;
        union { s16x4 h[2]; V8 v; } x;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 32 * ks + 8 * q + 4 * h + (i >> 2);
            x.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(s + k * R + (((r0 >> 4) ^ block_swizzle<R>(k)) << 4) + 4 * (i & 3)));
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
// a slot: the product, the sums, rounded up to 16 bytes
__host__ __device__ __forceinline__ long part_floats(long M, long N) { return (M * N + M + 3) & ~3l; }

// asks the scheduler for LDS reads and matrix instructions in turn, R reads spread over M
template <int R, int M, int I = 0>
__device__ __forceinline__ void spread_reads() {
    if constexpr (I < R) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);       // one LDS read
        constexpr int n = (I + 1) * M / R - I * M / R;
        if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x008, n, 0);
        spread_reads<R, M, I + 1>();
    }
}

template <int V> struct Log2 { static constexpr int v = 1 + Log2<V / 2>::v; };
template <> struct Log2<1> { static constexpr int v = 0; };

template <typename T, int PROD, int TM, int TN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_product(ProdArgs p, int tiles_m, int tiles_n) {
    constexpr bool AKC = PROD != PROD_WEIGHT, BKC = PROD == PROD_FORWARD, F32 = sizeof(T) == 4;
    constexpr int G = F32 ? 32 : 16, FA = TM / WM / G, FB = TN / WN / G, RG = F32 ? 16 : 4;      // fragment side, fragments, result registers
    constexpr int SK = 128 / sizeof(T), STAGE = (TM + TN) * SK;
    constexpr int KS = F32 ? 4 : 2;                              // k steps of a stage
    constexpr bool SPREAD = TM * TN == 65536 && PROD != PROD_WEIGHT;
    typedef typename VecOf<float, RG>::type Acc;
    typedef typename std::conditional<F32, f32x4, typename Vec8<T>::t>::type Frag;
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
            if (r1 - first > 1 << p.seg_log2) part = p.parts + seg_slot(first, i, p.seg_log2) * part_floats(p.M, p.N);
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
    // The bias gradient (sum over k of A) is made on the way, by the blocks of the first columns.  32 bits: one addition beside each matrix instruction, by the
    // waves that hold the first columns, over the k that a lane holds.  16 bits: the waves share a stage's k rows, a lane adds up four columns of
    // its rows from LDS; as a product with ones it cost these blocks an eighth of their time and a second set of fragments.
    const bool sums = PROD == PROD_WEIGHT && p.sum && n0 + (F32 ? wn : 0) == 0;
    constexpr int LPR = TM / 4, RPI = 64 / LPR, WAVES = WM * WN;             // lanes of a k row, k rows of an access
    float col[4] = {};
    float sum[FA] = {};
    // 32 bits: a chain of K additions into one register would lose sqrt(K) roundings' worth; every FLUSH stages it goes into a second one
    constexpr int FLUSH = 4;
    Acc total[F32 ? FA : 1][F32 ? FB : 1] = {};
    float total_sum[F32 ? FA : 1] = {};
    if (K > 0) {
        Stager<T, AKC, TM, WM * WN> ga;
        Stager<T, BKC, TN, WM * WN> gb;
        ga.init(A, p.lda, left_m);
        gb.init(B, p.ldb, N - n0);
        const unsigned int l0 = (unsigned int)(unsigned long)(__attribute__((address_space(3))) unsigned short*)lds;
        constexpr int BYTES = STAGE * (int)sizeof(T), L = ga.N + gb.N;       // of a stage; a wave's loads for it
        static_assert((NST - 1) * L < 64, "the wait's counter");
        const int stages = (K + SK - 1) / SK;
        auto fetch = [&](int st, int buf) {
            ga.load(l0 + buf * BYTES, K - st * SK);
            gb.load(l0 + buf * BYTES + TM * 128, K - st * SK);
        };
        auto piece = [&](int st, int buf, int i) {               // 0 .. L - 1 in turn
            if (i < ga.N) ga.load_piece(l0 + buf * BYTES, K - st * SK, i);
            else gb.load_piece(l0 + buf * BYTES + TM * 128, K - st * SK, i - ga.N);
        };
#pragma unroll
        for (int i = 0; i < NST; ++i) {
            if constexpr (SPREAD) {
#pragma unroll
                for (int l = 0; l < L; ++l) piece(i, i, l);
            } else if (i < stages) fetch(i, i);
        }
        // A wave multiplies one k step while the next one's fragments come out of LDS; at a stage's last step those are the next stage's, so that is where it
        // has to be there.  Its loads come back in order: NST - 2 later stages may still be on their way.  The barrier makes it everyone's part of
        // the stage, and says that nobody reads this stage any more (its reads have come back): the loads for the stage NST further go into its place.
        // In one burst these fill the queue that the LDS reads wait in too.  The rows' products in the largest tile have them among their matrix instructions, without a
        // condition (behind the last stage they ask for nothing and write zeros): 16384 rows, 1 expert 4096 -> 4096: forward 440 -> 390 us, input gradient 420 -> 391.
        // The weight gradient gains nothing from it (405: its reads are twice as many), and smaller tiles have few stages, of which the empty ones are a part (32 experts of
        // 256 rows, 2048 x 1408: 88 -> 94).
        Frag fa[2][FA], fb[2][FB];
        constexpr int ACROSS = F32 ? 4 : 2, READS = FA * (AKC ? 1 : ACROSS) + FB * (BKC ? 1 : ACROSS);       // LDS reads of a k step
        auto read_b = [&](int set, const T* sB, int ks, int j) {
            if constexpr (F32) fb[set][j] = stage_frag32<BKC, TN>(sB, wn + G * j, ks);
            else fb[set][j] = stage_frag<T, BKC, TN>(sB, wn + G * j, ks);
        };
        auto read_a = [&](int set, const T* sA, int ks, int i) {
            if constexpr (F32) fa[set][i] = stage_frag32<AKC, TM>(sA, wm + G * i, ks);
            else fa[set][i] = stage_frag<T, AKC, TM>(sA, wm + G * i, ks);
        };
        auto read = [&](int set, int buf, int ks) {
            const T *sA = sm + buf * STAGE, *sB = sA + TM * SK;
#pragma unroll
            for (int j = 0; j < FB; ++j) read_b(set, sB, ks, j);
#pragma unroll
            for (int i = 0; i < FA; ++i) read_a(set, sA, ks, i);
        };
        auto loop = [&](auto with_sums) {
            constexpr bool S = decltype(with_sums)::value;
            auto multiply_row = [&](int set, int i, int k) {
#pragma unroll
                for (int j = 0; j < FB; ++j) {
                    if constexpr (F32) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[set][j][k], fa[set][i][k], acc[i][j], 0, 0, 0);
                    else acc[i][j] = mfma16(fb[set][j], fa[set][i], acc[i][j]);
                }
                if constexpr (F32) { if (S) sum[i] += fa[set][i][k]; }
            };
            auto multiply = [&](int set) {
#pragma unroll
                for (int k = 0; k < (F32 ? 4 : 1); ++k)
#pragma unroll
                    for (int i = 0; i < FA; ++i) multiply_row(set, i, k);
            };
            if (SPREAD || NST <= stages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * L) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            read(0, 0, 0);
            int buf = 0;
            for (int st = 0; st < stages; ++st) {
                if constexpr (!F32 && PROD == PROD_WEIGHT) if (sums) {
#pragma unroll
                    for (int i = 0; i < SK / WAVES / RPI; ++i) {
                        const int k = wave * (SK / WAVES) + i * RPI + lane / LPR, l = lane % LPR;
                        const typename VecOf<T, 4>::type v = *reinterpret_cast<const typename VecOf<T, 4>::type*>(sm + buf * STAGE + k * TM + (((l >> 2) ^ block_swizzle<TM>(k)) << 4) + 4 * (l & 3));
#pragma unroll
                        for (int r = 0; r < 4; ++r) col[r] += (float)v[r];
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS - 1; ++ks) {
                    read((ks + 1) & 1, buf, ks + 1);
                    multiply(ks & 1);
                    spread_reads<READS, FA * FB * (F32 ? 4 : 1)>();
                }
                if (SPREAD || st + NST - 1 < stages) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * L) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const int freed = buf;
                if (!SPREAD && st + NST < stages) fetch(st + NST, freed);
                buf = buf + 1 == NST ? 0 : buf + 1;              // (behind the last stage: whatever lies there, unused)
                if constexpr (SPREAD) {
                    const T *sA = sm + buf * STAGE, *sB = sA + TM * SK;
#pragma unroll
                    for (int g = 0; g < FA; ++g) {
#pragma unroll
                        for (int f = g * (FA + FB) / FA; f < (g + 1) * (FA + FB) / FA; ++f) if (f < FB) read_b(0, sB, 0, f); else read_a(0, sA, 0, f - FB);
#pragma unroll
                        for (int l = g * L / FA; l < (g + 1) * L / FA; ++l) piece(st + NST, freed, l);
                        __builtin_amdgcn_s_setprio(1);           // (a wave with products before one that asks for data)
                        multiply_row((KS - 1) & 1, g, 0);
                        __builtin_amdgcn_s_setprio(0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    asm volatile("" ::: "memory");               // (or the compiler reads them in the next round after all)
                } else {
                    read(0, buf, 0);
                    asm volatile("" ::: "memory");
                    multiply((KS - 1) & 1);
                    spread_reads<READS, FA * FB * (F32 ? 4 : 1)>();
                }
                if constexpr (F32) {
                    if ((st + 1) % FLUSH == 0) {
                        asm volatile("" ::: "memory");          // (a branch, not 48 selects every stage)
#pragma unroll
                        for (int i = 0; i < FA; ++i) {
#pragma unroll
                            for (int j = 0; j < FB; ++j) { total[i][j] += acc[i][j]; acc[i][j] = Acc{}; }
                            if (S) { total_sum[i] += sum[i]; sum[i] = 0.0f; }
                        }
                    }
                }
            }
            if constexpr (SPREAD) {                              // (the loads for stages that are not there write zeros: the LDS is free behind them)
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
        };
        if (F32 && PROD == PROD_WEIGHT && sums) loop(std::true_type{}); else loop(std::false_type{});
    }
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < FA; ++i) {
#pragma unroll
            for (int j = 0; j < FB; ++j) acc[i][j] += total[i][j];
            sum[i] += total_sum[i];
        }
    }
    typedef typename VecOf<T, 4>::type V4;
    T* C = static_cast<T*>(p.c) + (PROD == PROD_WEIGHT ? e * p.c_expert + (long)m0 * p.ldc : (long)r0 * p.ldc);
    T* Z = PROD == PROD_FORWARD && p.z ? static_cast<T*>(p.z) + (long)r0 * p.ldc : nullptr;
    const T* bias = PROD == PROD_FORWARD && p.bias && e < p.E ? static_cast<const T*>(p.bias) + (long)e * N : nullptr;
    const bool silu = PROD == PROD_FORWARD && p.silu && e < p.E;
    if (PROD == PROD_WEIGHT && sums) {
        auto put = [&](int m, float v) {
            if (m >= left_m) return;
            if (part) part[(long)p.M * p.N + m0 + m] = v; else static_cast<T*>(p.sum)[(long)e * p.M + m0 + m] = (T)v;
        };
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const float v = sum[i] + __shfl_xor(sum[i], 32);       // (two lanes hold a row's k between them)
                if (lane < G) put(wm + G * i + lane, v);
            }
        } else {
            // [WAVES][TM] sums in LDS, added in order (the whole block is here: `sums` is the block's; LDS is free since the last barrier)
            float* const cs = reinterpret_cast<float*>(lds);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                for (int o = LPR; o < 64; o <<= 1) col[r] += __shfl_xor(col[r], o);
                if (lane < LPR) cs[wave * TM + 4 * lane + r] = col[r];
            }
            __syncthreads();
            if (threadIdx.x < TM) {
                float v = 0.0f;
                for (int w = 0; w < WAVES; ++w) v += cs[w * TM + threadIdx.x];
                put(threadIdx.x, v);
            }
            __syncthreads();                                     // (the results go through the same LDS)
        }
    }
    if (PROD == PROD_WEIGHT && !p.c) return;                     // (the sums alone)
    if constexpr (!F32) {
        // Whole 16-byte pieces: the wave's part goes through its share of LDS (free since the last barrier), so that a store writes eight rows' runs of
        // 16 (TN / WN) / 8 bytes instead of sixteen rows' 32: 65536 rows, 16 experts 2048 -> 4096: 1220 -> 1080 us.  Where the last-level cache cannot
        // hold operands and result together, results are written past it and leave it to the operands, which other tiles and the next products read again: 8192 rows, 32 experts
        // 2048 -> 1408 with gradients (184 MB of weights) 286 -> 258 us, of which only the weight gradient past it 277; the weight gradient of 64 experts 2048 -> 1408 of
        // 2048 rows 117 -> 98 us.  Where all fits, a result is read from the cache next; a combine_rows that reads one from behind the cache is no slower for it (8192 rows,
        // 32 experts 2048 -> 1408, product and combine: 77 us either way; 4096 rows, 64 experts 2048 -> 1024: 61 and 62).
        if (p.pieces == 8 && !part) {
            constexpr int PM = TM / WM, PN = TN / WN, CH = PN / 8;         // the wave's part, 16-byte pieces of its row
            T* const own = reinterpret_cast<T*>(lds) + wave * PM * PN;
            static_assert(WM * WN * PM * PN * 2 <= NST * (TM + TN) * 128, "the parts fit");
            f32x4 bv[FB];
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                const int n = n0 + wn + G * j + 4 * (lane >> 4);
                bv[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (bias && n < N) {
                    const V4 b = *reinterpret_cast<const V4*>(bias + n);
#pragma unroll
                    for (int r = 0; r < 4; ++r) bv[j][r] = (float)b[r];
                }
            }
            auto out = [&](T* to, bool act, auto keep, auto past) {
#pragma unroll
                for (int i = 0; i < FA; ++i)
#pragma unroll
                    for (int j = 0; j < FB; ++j) {
                        const int m = G * i + (lane & 15), c = 2 * j + (lane >> 5);
                        V4 y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float v = acc[i][j][r] + bv[j][r];
                            if constexpr (decltype(keep)::value) y[r] = kept_value<T>(v); else y[r] = act ? (T)silu_value<T>(v) : (T)v;
                        }
                        *reinterpret_cast<V4*>(own + m * PN + ((c ^ (m & (CH - 1))) << 3) + 4 * (lane >> 4 & 1)) = y;
                    }
                asm volatile("" ::: "memory");                   // (a wave's LDS accesses keep their order; other lanes wrote what a lane reads)
#pragma unroll
                for (int it = 0; it < PM * CH / 64; ++it) {
                    const int m = it * (64 / CH) + lane / CH, c = lane % CH, n = n0 + wn + 8 * c;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(own + m * PN + ((c ^ (m & (CH - 1))) << 3));
                    if (wm + m >= left_m || n >= N) continue;
                    u32x4* const at = reinterpret_cast<u32x4*>(to + (long)(wm + m) * p.ldc + n);
                    if constexpr (decltype(past)::value) __builtin_nontemporal_store(v, at); else *at = v;
                }
                asm volatile("" ::: "memory");
            };
            if (p.past) {
                out(C, silu, std::false_type{}, std::true_type{});
                if (Z) out(Z, false, std::true_type{}, std::true_type{});
            } else {
                out(C, silu, std::false_type{}, std::false_type{});
                if (Z) out(Z, false, std::true_type{}, std::false_type{});
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int g = 0; g < RG / 4; ++g) {
            const int n = n0 + wn + G * j + (F32 ? 8 * g + 4 * (lane >> 5) : 4 * (lane >> 4));
            if (n >= N) continue;
            const int left_n = N - n < 4 ? N - n : 4;
            float bv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (bias) {
#pragma unroll
                for (int r = 0; r < 4; ++r) bv[r] = r < left_n ? (float)bias[n + r] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const int m = wm + G * i + (lane & (G - 1));
                if (m >= left_m) continue;
                if (PROD == PROD_WEIGHT && part) {
                    float* const to = part + (long)(m0 + m) * N + n;
                    if (p.pieces >= 4) *reinterpret_cast<f32x4*>(to) = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                    else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) if (r < left_n) to[r] = acc[i][j][4 * g + r];
                    }
                    continue;
                }
                V4 y, z;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = acc[i][j][4 * g + r] + bv[r];
                    z[r] = kept_value<T>(v);
                    y[r] = silu ? (T)silu_value<T>(v) : (T)v;
                }
                const long at = (long)m * p.ldc + n;
                if (p.pieces >= 4) {
                    *reinterpret_cast<V4*>(C + at) = y;
                    if (Z) *reinterpret_cast<V4*>(Z + at) = z;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r < left_n) { C[at + r] = y[r]; if (Z) Z[at + r] = z[r]; }
                }
            }
        }
}

// The weight gradient of experts whose rows were cut, their segments' partial sums added in order; zeros for experts without rows (they have no
// segment); the rest is there already.  V values (of M N, then of M) a thread, y: expert
template <typename T, int V>
__global__ __launch_bounds__(256) void k_join_parts(ProdArgs p) {
    const int e = blockIdx.y, first = p.offsets[e], n = p.offsets[e + 1] - first, l = p.seg_log2;
    if (n > 0 && n <= 1 << l) return;
    const long mn = (long)p.M * p.N, all = mn + (p.sum ? p.M : 0), slot = part_floats(p.M, p.N);
    const int segs = (n + (1 << l) - 1) >> l;
    typedef typename VecOf<T, V>::type VT;
    typedef typename VecOf<float, V>::type VF;
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * V; i < all; i += (long)gridDim.x * 256 * V) {
        float v[V] = {};
        for (int k = 0; k < segs; ++k) {
            const VF a = *reinterpret_cast<const VF*>(p.parts + seg_slot(first, k, l) * slot + i);
            const float* ae = reinterpret_cast<const float*>(&a);
#pragma unroll
            for (int r = 0; r < V; ++r) v[r] += ae[r];
        }
        VT o;
        T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int r = 0; r < V; ++r) oe[r] = (T)v[r];
        if (i < mn) { if (p.c) *reinterpret_cast<VT*>(static_cast<T*>(p.c) + e * p.c_expert + i) = o; }
        else {
#pragma unroll
            for (int r = 0; r < V; ++r) static_cast<T*>(p.sum)[(long)e * p.M + i - mn + r] = oe[r];
        }
    }
}

// rows of any width, stride and address as rows of whole 16-byte pieces, zeros behind the width; y: operand (both in one launch)
struct PadJob { const void* src; long rows; int width; long stride; void* dst; int pieces; };
template <typename T>
__global__ __launch_bounds__(256) void k_pad_rows(PadJob j0, PadJob j1) {
    const PadJob p = blockIdx.y ? j1 : j0;
    constexpr int V = 16 / sizeof(T);
    const long n = p.rows * p.pieces;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / p.pieces;
        const int c = (int)(i - r * p.pieces) * V;
        const T* const src = static_cast<const T*>(p.src) + r * p.stride;
        union { T e[V]; unsigned long h[2]; u32x4 v; } x;
        if (p.width >= V) {                                      // the last piece ends with the row and is moved down
            const int at = c + V <= p.width ? c : p.width - V, by = (c - at) * 8 * (int)sizeof(T);
            const typename LooseOf<T, V>::type v = *reinterpret_cast<const typename LooseOf<T, V>::type*>(src + at);
            __builtin_memcpy(&x, &v, 16);
            if (by >= 64) { x.h[0] = x.h[1] >> (by - 64); x.h[1] = 0; }
            else if (by > 0) { x.h[0] = x.h[0] >> by | x.h[1] << (64 - by); x.h[1] >>= by; }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x.e[j] = j < p.width ? src[j] : (T)0.0f;
        }
        *reinterpret_cast<u32x4*>(static_cast<T*>(p.dst) + i * V) = x.v;
    }
}

// ---- around the products -------------------------------------------------------------------------------------------------
// dz = dy silu'(z) over the active rows, rounded to the type that the matrix pipe takes it in.  z is as it was stored: in 16 bits its rounding moves the slope by up to
// |silu''| u |z| <= u |z| / 2, which for most z below -0.6 is more than dz's own rounding (near the slope's zero at -1.28 by any factor).  The alternative is z in 32 bits, 2 bytes a value
// more to write and read.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_silu_back(const int* __restrict__ active, int width, const T* __restrict__ dy, long dy_stride, const T* __restrict__ z, T* __restrict__ dz) {
    typedef typename LooseOf<T, V>::type VT;
    const int chunks = (width + V - 1) / V;
    const long n = (long)active[0] * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / chunks, c = access_at<V>((int)(i - r * chunks), width);
        const VT g = *reinterpret_cast<const VT*>(dy + r * dy_stride + c), zz = *reinterpret_cast<const VT*>(z + r * width + c);
        const T *ge = reinterpret_cast<const T*>(&g), *ze = reinterpret_cast<const T*>(&zz);
        VT o;
        T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int j = 0; j < V; ++j) oe[j] = (T)((float)ge[j] * silu_slope<T>((float)ze[j]));
        *reinterpret_cast<VT*>(dz + r * width + c) = o;
    }
}

template <typename T, int PROD, int TM, int TN, int WM, int WN, int NST>
int launch_tiles(const ProdArgs& p, hipStream_t s) {
    const long tn = cdiv(p.N, TN), tm = PROD == PROD_WEIGHT ? cdiv(p.M, TM) : most_tiles(p.R, p.E, Log2<TM>::v);
    const bool cut = PROD == PROD_WEIGHT && p.seg_log2 != 31;
    const long blocks = (PROD == PROD_WEIGHT ? (cut ? most_tiles(p.R, p.E, p.seg_log2) : p.E) : 1) * tm * tn;
    if (blocks * 64 * WM * WN > 0xffffffffL) return fail("expert_linear: %ld tiles are more than a launch holds", blocks);
    if (blocks) hipLaunchKernelGGL((k_product<T, PROD, TM, TN, WM, WN, NST>), dim3((unsigned)blocks), dim3(64 * WM * WN), NST * (TM + TN) * 128, s, p, (int)tm, (int)tn);
    if (cut) {
        const bool four = p.pieces >= 4 && p.M % 4 == 0;
        const long per = cdiv((long)p.M * p.N + p.M, four ? 1024 : 256);
        const dim3 grid((unsigned)(per < 1024 ? per : 1024), p.E);
        if (four) hipLaunchKernelGGL((k_join_parts<T, 4>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((k_join_parts<T, 1>), grid, dim3(256), 0, s, p);
    }
    LAUNCHED();
    return 0;
}

// Tiles of a product by how many there are: 256 x 256 where they fill the CUs, 128 x 128, and 64 x 64 with four stages where even those are too few to
// keep enough bytes on their way (one token's experts, short prompts).  Measured in bf16, 128 against 256:
//   rows x outputs: 8192 rows, 1 expert, 4096 -> 4096 (528 tiles of 256): 279 us against 215; 20264 rows, 13 experts, 2048 -> 2048 (736): 187 against 166; 8192 rows,
//   8 experts, 4096 -> 4096 (656): 310 against 283; 16384 rows, 16 experts, 2048 -> 2048 (640): 148 both, and below: at 1024 rows an expert an eighth of
//   the 256-row tiles is empty; 8192 rows, 32 experts, 2048 -> 1408 (390): 64 against 93
//   weight gradient: 8192 rows, 1 expert, 4096 x 4096 (256 tiles): 281 against 248; 32768 rows, 8 experts, 2048 x 1024 (256): 129 against 110; 16384 rows, 12 experts,
//   2048 x 2048 (768): 139 against 132; but 20264 rows, 13 experts (832): 174 against 188, three rounds of the CUs and a quarter; 32 experts of 256 rows, 2048 x 1408: 81 against
//   82, uneven ones 110 against 128: few rows an expert write more than they multiply, and a CU's two small blocks do one while the other does the other
inline long prod_tiles(bool weight, long R, long E, long M, long N, int l) { return (weight ? E * cdiv(M, 1l << l) : most_tiles(R, E, l)) * cdiv(N, 1l << l); }
enum { TILE_64 = 6, TILE_128 = 7, TILE_256 = 8 };
template <typename T>
int prod_tile(bool weight, long R, long E, long M, long N) {
    if (sizeof(T) == 4) return TILE_64;
    const long big = prod_tiles(weight, R, E, M, N, 8);
    if (weight ? big >= 256 && R >= 1024 * E : big >= 1024 || (big >= 512 && R >= 1024 * E)) return TILE_256;
    return prod_tiles(weight, R, E, M, N, 7) >= 512 ? TILE_128 : TILE_64;
}

// Rows of a segment of the weight gradient (log2; 31: uncut).  An expert's tile is one block's chain over all of its rows, so a few long experts would
// leave most CUs idle: rows are cut until there are about four blocks a CU.  A segment's partial sums cost 8 bytes a value to write and add, which
// its products have to be worth: in 32 bits (20264 rows, 13 experts, 512 x 1024, some experts thrice as long as others) 352 -> 200 us; in 16 bits not where one expert alone
// has a tile for every other CU (8192 rows, 32 experts, 1408 x 2048: 113 us cut, 94 uncut).
template <typename T>
int seg_log2_for(long R, long E, long M, long N) {
    const int tile = prod_tile<T>(true, R, E, M, N);
    if (tile == TILE_256) return 31;
    const int least = sizeof(T) == 4 ? 9 : 10;
    const long tiles = cdiv(M, 1l << tile) * cdiv(N, 1l << tile), want = R * tiles / 1024;
    if (sizeof(T) == 2 && tiles >= 128) return 31;
    int l = least;
    while (l < 30 && (2l << l) <= want) ++l;
    return (1l << l) >= R ? 31 : l;
}

template <typename T, int PROD>
int launch_prod(const ProdArgs& p, int tile, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (tile == TILE_256) return launch_tiles<T, PROD, 256, 256, 2, 4, 2>(p, s);
        if (tile == TILE_128) return launch_tiles<T, PROD, 128, 128, 2, 2, 2>(p, s);
        return launch_tiles<T, PROD, 64, 64, 2, 2, 4>(p, s);
    } else {
        return launch_tiles<T, PROD, 64, 64, 2, 2, 2>(p, s);
    }
}

// An operand as the products read it: in place, or copied into the workspace with rows of whole pieces.
template <typename T>
struct Operand {
    const void* p; long rows, width, stride;
    bool fits() const {                                          // (rows that lie on each other are copied too: a buffer's end is a number of rows)
        constexpr long V = 16 / sizeof(T);
        return ((uintptr_t)p & 15) == 0 && width % V == 0 && stride % V == 0 && stride >= width && stride < (1 << 21);
    }
    long padded() const { constexpr long V = 16 / sizeof(T); return (width + V - 1) / V * V; }
    int64_t bytes() const { return fits() ? 0 : (rows * padded() * (long)sizeof(T) + 255) & ~255l; }
    // where the product reads it and its stride; the copy that makes it so, if one is needed; advances the workspace
    PadJob place(const void** at, long* ld, char** ws) const {
        *at = p; *ld = stride;
        if (fits()) return {};
        const PadJob j = {p, rows, (int)width, stride, *ws, (int)(padded() * (long)sizeof(T) / 16)};
        *at = *ws; *ld = padded();
        *ws += bytes();
        return j;
    }
};
template <typename T>
void pad_rows(PadJob a, PadJob b, hipStream_t s) {
    if (a.rows == 0) { a = b; b = {}; }
    const long blocks = cdiv((a.rows * a.pieces > b.rows * b.pieces ? a.rows * a.pieces : b.rows * b.pieces), 256);
    if (blocks) hipLaunchKernelGGL(k_pad_rows<T>, dim3((unsigned)(blocks < 16384 ? blocks : 16384), b.rows ? 2 : 1), dim3(256), 0, s, a, b);
}
template <typename T>
int result_pieces(long N, long ldc, const void* c, const void* z, const void* bias) {
    const int b = common_align({(uint64_t)N * sizeof(T), (uint64_t)ldc * sizeof(T), (uint64_t)(uintptr_t)c, (uint64_t)(uintptr_t)z, (uint64_t)(uintptr_t)bias}) / (int)sizeof(T);
    return b >= 8 ? 8 : (b >= 4 ? 4 : 1);
}

// the operands of a product, as the entry points name them
template <typename T>
void linear_operands(int32_t product, int64_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const void* a, int64_t a_stride, const void* b, int64_t b_stride, Operand<T>* oa,
                            Operand<T>* ob) {
    *oa = {a, (long)n_rows, (long)(product == CCSP_OPS_FORWARD ? inp : out), (long)a_stride};
    if (product == CCSP_OPS_BACK_WEIGHT) *ob = {b, (long)n_rows, (long)inp, (long)b_stride};
    else *ob = {b, (long)(n_experts * out), (long)inp, (long)inp};
}

template <typename T>
int64_t product_workspace(int32_t product, int64_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const void* a, int64_t a_stride, const void* b, int64_t b_stride) {
    Operand<T> oa, ob;
    linear_operands<T>(product, n_experts, n_rows, inp, out, a, a_stride, b, b_stride, &oa, &ob);
    int64_t bytes = oa.bytes() + ob.bytes();
    if (product == CCSP_OPS_BACK_WEIGHT) {
        const int l = seg_log2_for<T>(n_rows, n_experts, out, inp);
        if (l != 31) bytes += 2 * ((n_rows >> l) + 1) * part_floats(out, inp) * 4;
    }
    return bytes;
}

// the product's operands in their places, the rest of its arguments, the launch
template <typename T, int PROD>
int run_product(ProdArgs p, int64_t inp, int64_t out, const void* a, int64_t a_stride, const void* b, int64_t b_stride, void* workspace, int64_t workspace_bytes, hipStream_t s) {
    constexpr int product = PROD == PROD_FORWARD ? CCSP_OPS_FORWARD : (PROD == PROD_INPUT ? CCSP_OPS_BACK_INPUT : CCSP_OPS_BACK_WEIGHT);
    const int64_t need = product_workspace<T>(product, p.E, p.R, inp, out, a, a_stride, b, b_stride);
    CCSP_OPS_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), "linear: workspace of %lld bytes is smaller than %lld or not aligned to 16 bytes",
                   (long long)workspace_bytes, (long long)need);
    char* ws = static_cast<char*>(workspace);
    Operand<T> oa, ob;
    linear_operands<T>(product, p.E, p.R, inp, out, a, a_stride, b, b_stride, &oa, &ob);
    const PadJob ja = oa.place(&p.a, &p.lda, &ws), jb = ob.place(&p.b, &p.ldb, &ws);
    pad_rows<T>(ja, jb, s);
    p.b_expert = (PROD == PROD_WEIGHT ? 0 : out) * p.ldb;
    p.parts = reinterpret_cast<float*>(ws);
    p.pieces = result_pieces<T>(p.N, p.ldc, p.c, p.z, p.bias);
    // elements read and written: rows on both sides, and the weights or their gradient (of a few rows no more experts than rows are read)
    const long experts = PROD == PROD_WEIGHT || p.E < p.R ? p.E : p.R;
    p.past = (p.R * (inp + out) + experts * inp * out) * (long)sizeof(T) >= ROWS_PAST_CACHE;
    // (by the operands, not by p.N: the bias gradient alone is added up in the same order as beside the product)
    return launch_prod<T, PROD>(p, prod_tile<T>(PROD == PROD_WEIGHT, p.R, p.E, out, PROD == PROD_FORWARD ? out : inp), s);
}
