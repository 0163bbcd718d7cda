// Shared by the tensor-core cross attention kernels.
#pragma once

#include "relm_mp_attn.cuh"
#include "relm_mp_tc.cuh"

namespace relm_mp {
namespace attn {

// Two floats as one register of two T (low, high), and back.
template < typename T >
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2< __nv_bfloat16 >(float lo, float hi)
{
   const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
   return *reinterpret_cast< const uint32_t* >(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2< __half >(float lo, float hi)
{
   const __half2 v = __floats2half2_rn(lo, hi);
   return *reinterpret_cast< const uint32_t* >(&v);
}
template < typename T >
__device__ __forceinline__ float low2(uint32_t v)
{
   return to_f32((*reinterpret_cast< const T(*)[2] >(&v))[0]);
}
template < typename T >
__device__ __forceinline__ float high2(uint32_t v)
{
   return to_f32((*reinterpret_cast< const T(*)[2] >(&v))[1]);
}

struct TcMaps {
   CUtensorMap q, k, v, go;
};

// Tensor map of [seqs, heads, rows, dim] with boxes of `box_rows` rows by 64 columns;
// columns past dim and rows past the end read 0.
int tc_map(CUtensorMap* map, relm_mp_dtype dtype, const void* base, const int64_t* strides, int dim, int heads, int64_t rows, int64_t seqs,
           int box_rows = kTileRows);

}  // namespace attn
}  // namespace relm_mp
