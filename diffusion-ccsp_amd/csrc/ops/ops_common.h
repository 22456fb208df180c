// ops_common.h -- errors, element types and small device helpers of the operator library.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside its namespace): not a standalone header.
thread_local char g_err[512] = "";

int fail(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return 1;
}

#define HIP_TRY(expr)                                                                       \
    do {                                                                                    \
        hipError_t _e = (expr);                                                             \
        if (_e != hipSuccess) return fail("%s failed: %s (%s:%d)", #expr, hipGetErrorString(_e), __FILE__, __LINE__); \
    } while (0)
#define CCSP_OPS_CHECK(cond, ...) do { if (!(cond)) return fail(__VA_ARGS__); } while (0)
// an error that is pending when a call comes in is reported by it, as by any HIP call
#define LAUNCHED() HIP_TRY(hipGetLastError())

typedef __bf16 bf16;
typedef _Float16 fp16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };
// N elements at any element's address: one access of 16 bytes needs no alignment (the target's unaligned access mode, which the compiler counts on for such a type)
template <typename T, int N> struct LooseOf { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
template <typename T> struct LooseOf<T, 1> { typedef T type; };

// one block per item: a grid's x holds 2^32 threads, so large counts spread over y (the last row of blocks may run past the count)
inline dim3 grid_of(long blocks) { return blocks <= (1l << 22) ? dim3((unsigned)blocks) : dim3(1u << 22, (unsigned)((blocks + (1l << 22) - 1) >> 22)); }
__device__ __forceinline__ long block_id() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

inline long cdiv(long n, long b) { return (n + b - 1) / b; }

// element type code -> functor with a value of the type
template <typename F>
int dispatch_type(int t, F&& f) {
    if (t == CCSP_OPS_F32) return f(float{});
    if (t == CCSP_OPS_BF16) return f(bf16{});
    return f(fp16{});
}
inline bool type_ok(int t) { return t == CCSP_OPS_F32 || t == CCSP_OPS_BF16 || t == CCSP_OPS_F16; }
inline int type_bytes(int t) { return t == CCSP_OPS_F32 ? 4 : 2; }

// largest power-of-two access (in bytes, at most 16) that divides every argument
inline int common_align(std::initializer_list<uint64_t> v) {
    uint64_t m = 16;
    for (uint64_t x : v) m |= x;
    return (int)(m & (~m + 1));
}
