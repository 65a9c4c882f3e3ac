// timeline.h — PROBE BUILDS ONLY (-DOPTEX_TIMELINE, scripts/gemm_timeline_probe.hip): s_memtime stamps inside the GEMM
// kernels.  Every wavefront owns a slab of 64-bit words in tl_buf and appends one shader-clock stamp per call; its first lane
// writes the word with an ordinary vector store (the library build compiles none of this: TL_STAMP expands to nothing).
#pragma once
#ifdef OPTEX_TIMELINE
namespace optex {

// one copy per translation unit (gemm_rs.hip and gemm.hip are compiled apart): the probe sets the copy of the kernel it
// launches through that unit's setter, TL_DEFINE_SETTER(name)
static __device__ unsigned long long* tl_buf;
static __device__ int tl_words;          // words per wavefront slab

typedef unsigned long long* tl_ptr;

// the wavefront's slab, as a uniform (SGPR) pointer
__device__ __forceinline__ tl_ptr tl_begin(unsigned wave_slot) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(tl_buf + (size_t)wave_slot * (size_t)tl_words);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return reinterpret_cast<tl_ptr>(((uintptr_t)hi << 32) | (uintptr_t)lo);
}
// (a cursor that has been through a spill comes back in vector registers: pin it to an SGPR pair again)
__device__ __forceinline__ tl_ptr tl_uniform(tl_ptr p) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return reinterpret_cast<tl_ptr>(((uintptr_t)hi << 32) | (uintptr_t)lo);
}
__device__ __forceinline__ void tl_word(tl_ptr& p, unsigned long long v) {
    const tl_ptr q = tl_uniform(p);
    if (__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) == 0) __builtin_nontemporal_store(v, q);
    p += 1;
}
__device__ __forceinline__ void tl_stamp(tl_ptr& p) { tl_word(p, __builtin_amdgcn_s_memtime()); }
// the constant 100 MHz clock: what a stretch of shader cycles is in time (the effective clock)
__device__ __forceinline__ void tl_stamp_real(tl_ptr& p) { tl_word(p, __builtin_amdgcn_s_memrealtime()); }
__device__ __forceinline__ void tl_end() {}

}  // namespace optex
#define TL_STAMP(p) optex::tl_stamp(p)
#define TL_DEFINE_SETTER(name)                                                                    \
    namespace optex {                                                                             \
    void name(unsigned long long* buf, int words) {                                               \
        (void)hipMemcpyToSymbol(HIP_SYMBOL(tl_buf), &buf, sizeof(buf));                           \
        (void)hipMemcpyToSymbol(HIP_SYMBOL(tl_words), &words, sizeof(words));                     \
    }                                                                                             \
    }
#else
#define TL_DEFINE_SETTER(name)
#define TL_STAMP(p)
#endif
