// ccsp_trace.h -- phase-trace macros of the profiling builds (-DCCSP_TRACE / -DCCSP_TRACE2); empty in the product build.
// A fragment of the ONE translation unit csrc/ccsp_hip.hip (included there, at this position, inside its namespaces): not a standalone header.

// Profiling builds only (tools/trace_build.py compiles with -DCCSP_TRACE): s_memtime stamps at the phase boundaries of the
// evaluation kernels, one record per sampled workgroup, read back through ccsp_debug_trace.  The product build has none.
#ifdef CCSP_TRACE
__device__ unsigned long long g_trace[3 * 256 * 32];
#define CCSP_TRK(kern, k)                                                                             \
    do {                                                                                              \
        if (threadIdx.x == 0 && (blockIdx.x & 7) == 0 && blockIdx.x < 2048)                           \
            g_trace[((kern) * 256 + (blockIdx.x >> 3)) * 32 + (k)] = __builtin_amdgcn_s_memtime();    \
    } while (0)
// the same on the chip-wide 100 MHz clock (s_memtime counters are per shader engine: not comparable across workgroups)
#define CCSP_TRK_RT(kern, k)                                                                          \
    do {                                                                                              \
        if (threadIdx.x == 0 && (blockIdx.x & 7) == 0 && blockIdx.x < 2048)                           \
            g_trace[((kern) * 256 + (blockIdx.x >> 3)) * 32 + (k)] = __builtin_amdgcn_s_memrealtime(); \
    } while (0)
#else
#define CCSP_TRK(kern, k) do { } while (0)
#define CCSP_TRK_RT(kern, k) do { } while (0)
#endif

// Second profiling build (tools/trace2_build.py, -DCCSP_TRACE2; round 5): the phase boundaries of EVERY workgroup of k_rowgemm_h2 at the product
// kernel's own residency (three workgroups per CU in MODE 0), with the hardware slot the workgroup ran on (HW_ID: shader engine, CU, SIMD of
// wave 0; XCC_ID), so that the phases of the workgroups that SHARE a compute unit can be laid next to each other on that CU's own clock.  A stamp is the
// low half of s_memtime, stored by lane 0 of wave 0 straight to global memory.
#ifdef CCSP_TRACE2
__device__ unsigned int g_trace2[4096 * 40];
// (plain vector stores: each takes a slot of the load / store counter behind the loads in flight, so a hand-counted wait that follows one
// waits for at least what it waits for without it)
#define CCSP_TRK2_DECL unsigned int* const trk2_ptr = g_trace2 + (size_t)(blockIdx.x < 4096 ? blockIdx.x : 4095) * 40;
#define CCSP_TRK2(k)                                                                                                              \
    do {                                                                                                                          \
        const unsigned int lo_ = (unsigned int)__builtin_amdgcn_s_memtime();                                                      \
        if (threadIdx.x == 0) trk2_ptr[k] = lo_;                                                                                  \
    } while (0)
#define CCSP_TRK2_FLUSH()                                                                                                         \
    do {                                                                                                                          \
        unsigned int h0_, h1_;                                                                                                    \
        asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID)" : "=s"(h0_));                                                         \
        asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(h1_));                                                        \
        const unsigned int rt_ = (unsigned int)__builtin_amdgcn_s_memrealtime();                                                  \
        if (threadIdx.x == 0) { trk2_ptr[36] = h0_; trk2_ptr[37] = h1_; trk2_ptr[38] = rt_; }                                     \
    } while (0)
#else
#define CCSP_TRK2_DECL
#define CCSP_TRK2(k) do { } while (0)
#define CCSP_TRK2_FLUSH() do { } while (0)
#endif
