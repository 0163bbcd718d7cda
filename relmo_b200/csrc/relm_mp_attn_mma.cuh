// Warp-level pieces (m16n8k16 products, matrix loads, asynchronous copies) of the
// cross attention kernels for few query rows and for short sequences.
#pragma once

#include "relm_mp_attn.cuh"

namespace relm_mp {
namespace attn {

template < typename T >
struct Mma;
template <>
struct Mma< __nv_bfloat16 > {
   static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
   {
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
   }
   static __device__ __forceinline__ uint32_t pack(float lo, float hi)
   {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      return *reinterpret_cast< const uint32_t* >(&v);
   }
};
template <>
struct Mma< __half > {
   static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
   {
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
   }
   static __device__ __forceinline__ uint32_t pack(float lo, float hi)
   {
      const __half2 v = __floats2half2_rn(lo, hi);
      return *reinterpret_cast< const uint32_t* >(&v);
   }
};

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr)
{
   asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t addr)
{
   asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                : "r"(addr));
}
// 16 bytes, or zeros when !in (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in)
{
   asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// Byte offset of 16-byte chunk c of row r: chunks of 8 consecutive rows lie in different banks.
template < int DP >
__device__ __forceinline__ uint32_t swizzled(int r, int c)
{
   constexpr int CH = DP / 8;
   return (uint32_t)(r * DP * 2 + ((c ^ (CH >= 8 ? r & 7 : (r >> 1) & 3)) * 16));
}

}  // namespace attn
}  // namespace relm_mp
