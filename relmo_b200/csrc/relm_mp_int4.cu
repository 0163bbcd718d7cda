// Products of a few rows with 4-bit weights and group scales:
//
//   y[r, n] = xs[r] * sum_groups s[n, g] * sum_{k in g} x[r, k] * (c[n, k] - z[n, g])
//
// Bound by the weights' bytes (half a byte each), so the inner product runs on
// the matrix instruction with the 16 weight rows as its left operand and up to
// 8 (or 16) x rows as its right one: one instruction per 16 x 16 weights
// whatever the number of rows. The codes become 2-byte floats by setting them
// into the mantissa of 128 (bf16) or 1024 (f16) and subtracting 128 + z (1024
// + z): exact. Each group's sum is float32 and is multiplied by its scale in
// float32, so the only roundings are those of float32 sums.
//
// The right operand keeps x exact: bf16 and f16 as they are, e4m3 as f16, and
// float32 as three bf16 columns (x = hi + mid + lo, 24 bits), which cost
// nothing as the instruction has 8 columns anyway.
//
// Layout (relm_mp_int4_pack): for each 16 rows and 64 columns, lane (g, t) of a
// warp holds one 16-byte word: rows g and g + 8, columns 8 t .. 8 t + 7 of both
// halves of 32. A warp's load is 512 contiguous bytes, the x values of a lane
// are two runs of 8 (the order of k inside a product is free), and a product
// never crosses a group of 32.
#include <cuda_fp8.h>

#include "relm_mp_internal.cuh"

using namespace relm_mp;

namespace {

constexpr int kWarps = 8;
constexpr int kBlockK = 64; // columns of one packed word row

struct Layout {
   int64_t tiles, blocks, groups; // 16-row tiles, 64-column blocks, groups (padded to whole blocks)
   size_t scales, zeros, bytes;
};

Layout layout(int64_t n, int64_t k, int64_t group, bool zeros)
{
   Layout l;
   l.tiles = (n + 15) / 16;
   l.blocks = (k + kBlockK - 1) / kBlockK;
   l.groups = (l.blocks * kBlockK + group - 1) / group;
   l.scales = align_up((size_t)l.tiles * l.blocks * 512);
   l.zeros = l.scales + align_up((size_t)l.tiles * l.groups * 32);
   l.bytes = l.zeros + (zeros ? align_up((size_t)l.tiles * l.groups * 16) : 0);
   return l;
}

// Nibble of word s (column 32 (s / 2) + 8 t + 4 (s % 2) + j) and row half r in a lane's 16 bytes: the pairs
// (j, j + 1) of one row lie 16 bits apart, so one mask yields both halves of a register.
__host__ __device__ constexpr int nibble_of(int r, int j) { return (j & 2) + r + (j & 1) * 4; }

__global__ void __launch_bounds__(256) k_int4_pack(const unsigned char* __restrict__ codes, int64_t n, int64_t k,
                                                   int64_t blocks, int64_t words, uint32_t* __restrict__ out)
{
   const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
   if(w >= words) return;
   const int s = w & 3, lane = (w >> 2) & 31;
   const int64_t tile = (w >> 7) / blocks, blk = (w >> 7) % blocks;
   const int g = lane >> 2, t = lane & 3;
   uint32_t v = 0;
   for(int r = 0; r < 2; ++r)
      for(int j = 0; j < 4; ++j) {
         const int64_t row = tile * 16 + g + 8 * r, col = blk * kBlockK + 32 * (s >> 1) + 8 * t + 4 * (s & 1) + j;
         if(row >= n || col >= k) continue; // padding: x is 0 there, or the output row is not stored
         const uint32_t c = codes[row * (k / 2) + col / 2];
         v |= ((col & 1 ? c >> 4 : c) & 15u) << (4 * nibble_of(r, j));
      }
   out[w] = v;
}

// Per (tile, group): scales (and zero points) of rows (g, g + 8) side by side.
__global__ void __launch_bounds__(256) k_int4_pack_groups(const __half* __restrict__ scales,
                                                          const unsigned char* __restrict__ zeros, int64_t n,
                                                          int64_t src_groups, int64_t groups, int64_t total,
                                                          __half* __restrict__ out_s, unsigned char* __restrict__ out_z)
{
   const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
   if(i >= total) return;
   const int64_t tile = (i >> 4) / groups, grp = (i >> 4) % groups;
   const int e = i & 15;
   const int64_t row = tile * 16 + (e >> 1) + 8 * (e & 1);
   const bool in = row < n && grp < src_groups;
   out_s[i] = in ? scales[row * src_groups + grp] : __float2half_rn(0.f);
   if(out_z) out_z[i] = in ? zeros[row * src_groups + grp] : 0;
}

template < typename M >
struct Magic;
template <>
struct Magic< __nv_bfloat16 > {
   static constexpr uint32_t bits = 0x43004300u; // (128, 128)
   static __device__ __forceinline__ uint32_t base(int z)
   {
      const __nv_bfloat162 v = __float2bfloat162_rn(128.f + (float)z);
      return *reinterpret_cast< const uint32_t* >(&v);
   }
   static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b)
   {
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast< __nv_bfloat162* >(&a), *reinterpret_cast< __nv_bfloat162* >(&b));
      return *reinterpret_cast< const uint32_t* >(&v);
   }
   static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b)
   {
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
   }
};
template <>
struct Magic< __half > {
   static constexpr uint32_t bits = 0x64006400u; // (1024, 1024)
   static __device__ __forceinline__ uint32_t base(int z)
   {
      const __half2 v = __float2half2_rn(1024.f + (float)z);
      return *reinterpret_cast< const uint32_t* >(&v);
   }
   static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b)
   {
      const __half2 v = __hsub2(*reinterpret_cast< __half2* >(&a), *reinterpret_cast< __half2* >(&b));
      return *reinterpret_cast< const uint32_t* >(&v);
   }
   static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b)
   {
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
   }
};

enum Source { kSame = 0, kF32 = 1, kE4m3 = 2 };

// x columns of the right operand per row of x.
template < int SRC >
constexpr int kColumns = SRC == kF32 ? 3 : 1;

__device__ __forceinline__ uint4 load_stream(const uint4* p)
{
   uint4 v;
   asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                : "l"(p));
   return v;
}

// 8 x values of one lane (half a column block) as 4 registers of two. `part`
// chooses the term of a float32's split.
template < typename M, int SRC >
__device__ __forceinline__ void load_x(const void* xrow, int64_t k0, int part, bool vec, uint32_t* b)
{
   if constexpr(SRC == kSame) {
      const M* p = static_cast< const M* >(xrow) + k0;
      if(vec) {
         const uint4 u = __ldg(reinterpret_cast< const uint4* >(p));
         b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w;
      } else {
         const unsigned short* q = reinterpret_cast< const unsigned short* >(p);
#pragma unroll
         for(int i = 0; i < 4; ++i) b[i] = (uint32_t)q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
      }
   } else if constexpr(SRC == kE4m3) {
      const unsigned char* p = static_cast< const unsigned char* >(xrow) + k0;
      uint32_t w[2];
      if(vec) {
         const uint2 u = __ldg(reinterpret_cast< const uint2* >(p));
         w[0] = u.x, w[1] = u.y;
      } else {
#pragma unroll
         for(int i = 0; i < 2; ++i)
            w[i] = (uint32_t)p[4 * i] | (uint32_t)p[4 * i + 1] << 8 | (uint32_t)p[4 * i + 2] << 16 |
                   (uint32_t)p[4 * i + 3] << 24;
      }
#pragma unroll
      for(int i = 0; i < 4; ++i) {
         const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
         b[i] = (uint32_t)h.x | (uint32_t)h.y << 16;
      }
   } else {
      const float* p = static_cast< const float* >(xrow) + k0;
      float f[8];
      if(vec) {
#pragma unroll
         for(int i = 0; i < 2; ++i) {
            const float4 v = __ldg(reinterpret_cast< const float4* >(p) + i);
            f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
         }
      } else {
#pragma unroll
         for(int i = 0; i < 8; ++i) f[i] = p[i];
      }
#pragma unroll
      for(int i = 0; i < 8; ++i) {
         // An infinity or NaN stays in the first term; its rest would be NaN.
         const float hi = __bfloat162float(__float2bfloat16_rn(f[i]));
         const float r1 = fabsf(hi) <= 3.4e38f ? f[i] - hi : 0.f;
         const float mid = __bfloat162float(__float2bfloat16_rn(r1));
         f[i] = part == 0 ? hi : part == 1 ? mid : r1 - mid;
      }
#pragma unroll
      for(int i = 0; i < 4; ++i) {
         const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
         b[i] = *reinterpret_cast< const uint32_t* >(&v);
      }
   }
}

template < typename T >
__device__ __forceinline__ T store_as(float v);
template <>
__device__ __forceinline__ float store_as< float >(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 store_as< __nv_bfloat16 >(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half store_as< __half >(float v) { return __float2half_rn(v); }

struct MatvecArgs {
   const void* x;
   int64_t x_stride;
   const float* x_scale;
   int rows;
   const uint4* codes;
   const __half2* scales;
   const uchar2* zeros; // NULL: 8
   int64_t n, k, groups;
   int blocks, group_shift;
   bool vec;
   void* y;
};

// A block owns 16 * NT weight rows; its warps take the 64-column blocks in turn
// and their sums are joined in shared memory in warp order.
template < typename M, int SRC, int CT, int NT, typename OUT >
__global__ void __launch_bounds__(kWarps * 32) k_int4_matvec(MatvecArgs a)
{
   constexpr int COLS = CT * 8;
   __shared__ float part[kWarps][NT * 16][COLS + 1];
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
   const int64_t tile0 = (int64_t)blockIdx.x * NT;
   float total[NT][CT][4];
#pragma unroll
   for(int n = 0; n < NT; ++n)
#pragma unroll
      for(int c = 0; c < CT; ++c)
#pragma unroll
         for(int i = 0; i < 4; ++i) total[n][c][i] = 0.f;
   const int64_t tiles = (a.n + 15) / 16;
#pragma unroll 4
   for(int blk = warp; blk < a.blocks; blk += kWarps) {
      uint4 w[NT];
#pragma unroll
      for(int n = 0; n < NT; ++n)
         w[n] = tile0 + n < tiles ? load_stream(a.codes + ((tile0 + n) * a.blocks + blk) * 32 + lane) : make_uint4(0, 0, 0, 0);
      uint32_t b[CT][8];
      const int64_t k0 = (int64_t)blk * kBlockK + 8 * t;
      const bool second = (int64_t)blk * kBlockK + 32 < a.k; // k is a multiple of 32
#pragma unroll
      for(int c = 0; c < CT; ++c) {
         const int col = c * 8 + g, row = col / kColumns< SRC >;
         constexpr size_t ES = SRC == kF32 ? 4 : SRC == kE4m3 ? 1 : 2;
         const char* xrow = static_cast< const char* >(a.x) + row * a.x_stride * ES;
#pragma unroll
         for(int h = 0; h < 2; ++h) {
            if(row < a.rows && (h == 0 || second)) {
               load_x< M, SRC >(xrow, k0 + 32 * h, col % kColumns< SRC >, a.vec, b[c] + 4 * h);
            } else {
#pragma unroll
               for(int i = 0; i < 4; ++i) b[c][4 * h + i] = 0;
            }
         }
      }
      // Groups of 64 columns or more cover the block with one scale; groups of 32 change half way.
      const int64_t grp = ((int64_t)blk * kBlockK) >> a.group_shift;
      const int halves = a.group_shift == 5 ? 2 : 1;
#pragma unroll
      for(int n = 0; n < NT; ++n) {
         if(tile0 + n >= tiles) continue;
         const uint32_t* ww = reinterpret_cast< const uint32_t* >(&w[n]);
         float acc[CT][4];
         uint32_t z0 = 0, z1 = 0;
         float s0 = 0.f, s1 = 0.f;
#pragma unroll
         for(int s = 0; s < 4; ++s) {
            if(s == 0 || (s == 2 && halves == 2)) {
               const int64_t at = ((tile0 + n) * a.groups + grp + (s >> 1)) * 8 + g;
               const float2 sc = __half22float2(__ldg(a.scales + at));
               s0 = sc.x, s1 = sc.y;
               uchar2 z = make_uchar2(8, 8);
               if(a.zeros) z = __ldg(a.zeros + at);
               z0 = Magic< M >::base(z.x), z1 = Magic< M >::base(z.y);
#pragma unroll
               for(int c = 0; c < CT; ++c)
#pragma unroll
                  for(int i = 0; i < 4; ++i) acc[c][i] = 0.f;
            }
            uint32_t f[4];
            f[0] = Magic< M >::sub((ww[s] & 0x000f000fu) | Magic< M >::bits, z0);
            f[1] = Magic< M >::sub(((ww[s] >> 4) & 0x000f000fu) | Magic< M >::bits, z1);
            f[2] = Magic< M >::sub(((ww[s] >> 8) & 0x000f000fu) | Magic< M >::bits, z0);
            f[3] = Magic< M >::sub(((ww[s] >> 12) & 0x000f000fu) | Magic< M >::bits, z1);
#pragma unroll
            for(int c = 0; c < CT; ++c) Magic< M >::mma(acc[c], f, &b[c][2 * s]);
            if(s == 3 || (s == 1 && halves == 2)) {
#pragma unroll
               for(int c = 0; c < CT; ++c) {
                  total[n][c][0] += s0 * acc[c][0];
                  total[n][c][1] += s0 * acc[c][1];
                  total[n][c][2] += s1 * acc[c][2];
                  total[n][c][3] += s1 * acc[c][3];
               }
            }
         }
      }
   }
#pragma unroll
   for(int n = 0; n < NT; ++n)
#pragma unroll
      for(int c = 0; c < CT; ++c)
#pragma unroll
         for(int i = 0; i < 4; ++i) part[warp][n * 16 + g + 8 * (i >> 1)][c * 8 + 2 * t + (i & 1)] = total[n][c][i];
   __syncthreads();
   constexpr int PER = kColumns< SRC >;
   for(int i = threadIdx.x; i < a.rows * NT * 16; i += kWarps * 32) {
      const int r = i / (NT * 16), j = i % (NT * 16);
      const int64_t out = tile0 * 16 + j;
      if(out >= a.n) continue;
      float v = 0.f;
#pragma unroll
      for(int w = 0; w < kWarps; ++w)
#pragma unroll
         for(int p = 0; p < PER; ++p) v += part[w][j][r * PER + p];
      if(a.x_scale) v *= a.x_scale[r];
      static_cast< OUT* >(a.y)[(int64_t)r * a.n + out] = store_as< OUT >(v);
   }
}

template < typename M, int SRC, int CT, typename OUT >
void launch(const MatvecArgs& a, cudaStream_t st)
{
   const int64_t tiles = (a.n + 15) / 16;
   k_int4_matvec< M, SRC, CT, 1, OUT ><<< (unsigned)tiles, kWarps * 32, 0, st >>>(a);
}

template < typename M, int SRC, typename OUT >
int matvec(MatvecArgs a, int64_t rows, cudaStream_t st)
{
   // Rows in groups that fill the instruction's columns; the weights of later groups come from L2.
   constexpr int FEW = SRC == kF32 ? 2 : 8, MANY = SRC == kF32 ? 8 : 16;
   const size_t es = SRC == kF32 ? 4 : SRC == kE4m3 ? 1 : 2;
   for(int64_t lo = 0; lo < rows; lo += MANY) {
      MatvecArgs b = a;
      b.rows = (int)(rows - lo < MANY ? rows - lo : MANY);
      b.x = static_cast< const char* >(a.x) + lo * a.x_stride * es;
      b.y = static_cast< OUT* >(a.y) + lo * a.n;
      if(a.x_scale) b.x_scale = a.x_scale + lo;
      if(b.rows <= FEW) launch< M, SRC, 1, OUT >(b, st);
      else launch< M, SRC, MANY * kColumns< SRC > / 8, OUT >(b, st);
      const int rc = check_launch("k_int4_matvec");
      if(rc) return rc;
   }
   return RELM_MP_OK;
}

int check_shape(int64_t n, int64_t k, int64_t group, const char* op)
{
   if(group != 32 && group != 64 && group != 128)
      return fail(RELM_MP_ERR_INVALID_ARGUMENT, std::string(op) + ": group must be 32, 64 or 128.");
   if(n < 1 || k < 1 || k % group || n > (1ll << 31) - 32 || k > (1ll << 30))
      return fail(RELM_MP_ERR_INVALID_ARGUMENT, std::string(op) + ": n must be >= 1 and k a positive multiple of group.");
   return RELM_MP_OK;
}

}  // namespace

size_t relm_mp_int4_packed_bytes(int64_t n, int64_t k, int64_t group, int has_zeros)
{
   if(check_shape(n, k, group, "int4_packed_bytes")) return 0;
   return layout(n, k, group, has_zeros != 0).bytes;
}

int relm_mp_int4_pack(const unsigned char* codes, const void* scales, const unsigned char* zeros, int64_t n, int64_t k,
                      int64_t group, void* packed, size_t packed_bytes, void* stream)
{
   int rc;
   if((rc = check_shape(n, k, group, "int4_pack"))) return rc;
   if(!codes || !scales || !packed) return fail(RELM_MP_ERR_INVALID_ARGUMENT, "int4_pack: pointers must not be NULL.");
   const Layout l = layout(n, k, group, zeros != nullptr);
   if(packed_bytes < l.bytes) return fail(RELM_MP_ERR_WORKSPACE_TOO_SMALL, "int4_pack: packed buffer too small.");
   cudaStream_t st = static_cast< cudaStream_t >(stream);
   char* base = static_cast< char* >(packed);
   const int64_t words = l.tiles * l.blocks * 128, entries = l.tiles * l.groups * 16;
   k_int4_pack<<< (unsigned)((words + 255) / 256), 256, 0, st >>>(codes, n, k, l.blocks, words, reinterpret_cast< uint32_t* >(base));
   if((rc = check_launch("k_int4_pack"))) return rc;
   k_int4_pack_groups<<< (unsigned)((entries + 255) / 256), 256, 0, st >>>(
      static_cast< const __half* >(scales), zeros, n, k / group, l.groups, entries,
      reinterpret_cast< __half* >(base + l.scales), zeros ? reinterpret_cast< unsigned char* >(base + l.zeros) : nullptr);
   return check_launch("k_int4_pack_groups");
}

int relm_mp_int4_matvec(relm_mp_dtype dtype, int x_e4m3, const void* x, int64_t x_stride, const float* x_scale,
                        int64_t rows, const void* packed, int64_t n, int64_t k, int64_t group, int has_zeros, void* y,
                        void* stream)
{
   int rc;
   if((rc = check_shape(n, k, group, "int4_matvec"))) return rc;
   if(rows < 0) return fail(RELM_MP_ERR_INVALID_ARGUMENT, "int4_matvec: rows must be >= 0.");
   if(dtype != RELM_MP_FLOAT32 && dtype != RELM_MP_BFLOAT16 && dtype != RELM_MP_FLOAT16)
      return fail(RELM_MP_ERR_UNSUPPORTED, "int4_matvec: unsupported dtype (float32, bfloat16, float16).");
   if(rows == 0) return RELM_MP_OK;
   if(!x || !packed || !y) return fail(RELM_MP_ERR_INVALID_ARGUMENT, "int4_matvec: pointers must not be NULL.");
   const Layout l = layout(n, k, group, has_zeros != 0);
   const char* base = static_cast< const char* >(packed);
   const size_t es = x_e4m3 ? 1 : dtype_size(dtype);
   MatvecArgs a{};
   a.x = x, a.x_stride = x_stride, a.x_scale = x_scale;
   a.codes = reinterpret_cast< const uint4* >(base);
   a.scales = reinterpret_cast< const __half2* >(base + l.scales);
   a.zeros = has_zeros ? reinterpret_cast< const uchar2* >(base + l.zeros) : nullptr;
   a.n = n, a.k = k, a.groups = l.groups, a.blocks = (int)l.blocks;
   a.group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
   a.vec = (reinterpret_cast< uintptr_t >(x) & 15) == 0 && (x_stride * es) % 16 == 0;
   a.y = y;
   cudaStream_t st = static_cast< cudaStream_t >(stream);
   if(x_e4m3) {
      switch(dtype) {
         case RELM_MP_FLOAT32: return matvec< __half, kE4m3, float >(a, rows, st);
         case RELM_MP_BFLOAT16: return matvec< __half, kE4m3, __nv_bfloat16 >(a, rows, st);
         default: return matvec< __half, kE4m3, __half >(a, rows, st);
      }
   }
   switch(dtype) {
      case RELM_MP_FLOAT32: return matvec< __nv_bfloat16, kF32, float >(a, rows, st);
      case RELM_MP_BFLOAT16: return matvec< __nv_bfloat16, kSame, __nv_bfloat16 >(a, rows, st);
      default: return matvec< __half, kSame, __half >(a, rows, st);
   }
}
