// Cross attention on the CUDA cores: float32 inputs, head dims and strides that
// the tensor-core kernels do not take.
//
// Forward, per query tile: one pass over the keys with the running maximum m
// and sum l of each row (log2 domain, float32):
//   m' = max(m, s_j), c = 2^(m - m'), l = l c + sum 2^(s_j - m'), o = o c + sum 2^(s_j - m') v_j
// Backward, from lse = m + log l and delta = sum_d do o:
//   p = e^(s - lse), ds = p (do . v - delta)
// in two kernels without atomics: one per key tile (dk, dv; the loop runs over
// the query tiles of all heads of the group) and one per query tile (dq).
//
// Tiles are float32 in shared memory, rows DP + 4 apart (16-byte reads of 8
// consecutive rows cover all banks), zero beyond the length and dim, so that
// nothing outside a sequence, and no masked value row, enters a sum. Each of
// the 256 threads computes R x R scores of a (16 R) x (16 R) tile.
#include <math_constants.h>

#include "relm_mp_attn.cuh"

namespace relm_mp {
namespace attn {
namespace {

constexpr int kBlock = 256;

// DP: dim rounded up; R: rows (and keys) of a tile per thread row. Tiles of
// wide heads are smaller so that four of them fit shared memory.
template < int DP_ >
struct Shape {
   static constexpr int DP = DP_, R = DP_ > 128 ? 2 : 4, B = 16 * R, LD = DP_ + 4, LP = B + 4;
   static constexpr size_t tile = (size_t)B * LD * 4, square = (size_t)B * LP * 4;
};

// Rows [row0, row0 + B) of one head into shared memory, zero where row >= len,
// column >= dim or keep[row] == 0.
template < typename T, typename S >
__device__ void load_tile(float* dst, const T* src, int64_t row_stride, int row0, int len, int dim,
                          const unsigned char* keep)
{
   for(int i = threadIdx.x; i < S::B * S::DP; i += kBlock) {
      const int r = i / S::DP, c = i % S::DP;
      float v = 0.f;
      if(row0 + r < len && c < dim && (!keep || keep[row0 + r])) v = to_f32(src[(int64_t)(row0 + r) * row_stride + c]);
      dst[r * S::LD + c] = v;
   }
}

// s[i][j] = a[ty + 16 i] . b[tx + 16 j]
template < typename S >
__device__ __forceinline__ void dots(const float* a, const float* b, int ty, int tx, float (&s)[S::R][S::R])
{
#pragma unroll
   for(int i = 0; i < S::R; ++i)
#pragma unroll
      for(int j = 0; j < S::R; ++j) s[i][j] = 0.f;
#pragma unroll 4
   for(int d = 0; d < S::DP; d += 4) {
      float4 x[S::R], y[S::R];
#pragma unroll
      for(int i = 0; i < S::R; ++i) x[i] = *reinterpret_cast< const float4* >(a + (ty + 16 * i) * S::LD + d);
#pragma unroll
      for(int j = 0; j < S::R; ++j) y[j] = *reinterpret_cast< const float4* >(b + (tx + 16 * j) * S::LD + d);
#pragma unroll
      for(int i = 0; i < S::R; ++i)
#pragma unroll
         for(int j = 0; j < S::R; ++j) {
            s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
            s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
            s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
            s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
         }
   }
}

// acc[i][c] += sum_j w[ty + 16 i][j] x[j][tx + 16 c]
template < typename S >
__device__ __forceinline__ void accumulate(const float* w, const float* x, int ty, int tx, float (&acc)[S::R][S::DP / 16])
{
#pragma unroll 2
   for(int j = 0; j < S::B; ++j) {
      float p[S::R];
#pragma unroll
      for(int i = 0; i < S::R; ++i) p[i] = w[(ty + 16 * i) * S::LP + j];
#pragma unroll
      for(int c = 0; c < S::DP / 16; ++c) {
         const float v = x[j * S::LD + tx + 16 * c];
#pragma unroll
         for(int i = 0; i < S::R; ++i) acc[i][c] = fmaf(p[i], v, acc[i][c]);
      }
   }
}

template < typename S >
__device__ __forceinline__ void clear(float (&acc)[S::R][S::DP / 16])
{
#pragma unroll
   for(int i = 0; i < S::R; ++i)
#pragma unroll
      for(int c = 0; c < S::DP / 16; ++c) acc[i][c] = 0.f;
}

template < typename T, typename S >
__global__ void __launch_bounds__(kBlock) k_attn_forward(Args a)
{
   extern __shared__ float sm[];
   float *sq = sm, *sk = sq + S::B * S::LD, *sv = sk + S::B * S::LD, *sp = sv + S::B * S::LD;
   const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
   constexpr int PER = kTileRows / S::B; // sub-tiles of a plan's tile
   const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
   const Item it = item(a.q_tiles, a.max_q, kTileRows, blockIdx.x / PER);
   const Seq qs = locate(a.q_off, a.max_q, a.qs, it.seq), ks = locate(a.kv_off, a.max_kv, a.ks, it.seq);
   const Seq vs = locate(a.kv_off, a.max_kv, a.vs, it.seq);
   const int row0 = it.tile * kTileRows + (blockIdx.x % PER) * S::B;
   if(row0 >= qs.len) return;
   const T* q = static_cast< const T* >(a.q) + qs.base + head * a.qs[2];
   const T* k = static_cast< const T* >(a.k) + ks.base + kv_head * a.ks[2];
   const T* v = static_cast< const T* >(a.v) + vs.base + kv_head * a.vs[2];
   const unsigned char* keep = a.mask ? a.mask + ks.first : nullptr;
   load_tile< T, S >(sq, q, a.qs[1], row0, qs.len, a.dim, nullptr);
   float acc[S::R][S::DP / 16], m[S::R], l[S::R];
   clear< S >(acc);
#pragma unroll
   for(int i = 0; i < S::R; ++i) m[i] = -CUDART_INF_F, l[i] = 0.f;
   const float sc = a.scale * kLog2e;
   for(int key0 = 0; key0 < ks.len; key0 += S::B) {
      __syncthreads();
      load_tile< T, S >(sk, k, a.ks[1], key0, ks.len, a.dim, nullptr);
      load_tile< T, S >(sv, v, a.vs[1], key0, ks.len, a.dim, keep);
      __syncthreads();
      float s[S::R][S::R];
      dots< S >(sq, sk, ty, tx, s);
#pragma unroll
      for(int j = 0; j < S::R; ++j) {
         const int key = key0 + tx + 16 * j;
         const bool in = key < ks.len && (!keep || keep[key]);
#pragma unroll
         for(int i = 0; i < S::R; ++i) s[i][j] = in ? s[i][j] * sc : -CUDART_INF_F;
      }
#pragma unroll
      for(int i = 0; i < S::R; ++i) {
         float top = m[i];
#pragma unroll
         for(int j = 0; j < S::R; ++j) top = fmaxf(top, s[i][j]);
#pragma unroll
         for(int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
         // A row without a kept key so far has no maximum: its weights are 0 whatever the reference.
         const float ref = top == -CUDART_INF_F ? 0.f : top;
         const float c = exp2_fast(m[i] - ref);
         m[i] = top;
         float sum = 0.f;
#pragma unroll
         for(int j = 0; j < S::R; ++j) {
            const float p = exp2_fast(s[i][j] - ref);
            sum += p;
            sp[(ty + 16 * i) * S::LP + tx + 16 * j] = p;
         }
#pragma unroll
         for(int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
         l[i] = l[i] * c + sum;
#pragma unroll
         for(int d = 0; d < S::DP / 16; ++d) acc[i][d] *= c;
      }
      __syncwarp(); // a thread row's weights are written and read by the same half warp
      accumulate< S >(sp, sv, ty, tx, acc);
   }
   T* o = static_cast< T* >(a.o);
#pragma unroll
   for(int i = 0; i < S::R; ++i) {
      const int row = row0 + ty + 16 * i;
      if(row >= qs.len) continue;
      const bool none = l[i] == 0.f; // no kept key (a NaN score leaves l NaN)
      const float inv = none ? 0.f : 1.f / l[i];
      const int64_t out = ((qs.first + row) * a.heads + head) * a.dim;
#pragma unroll
      for(int d = 0; d < S::DP / 16; ++d)
         if(tx + 16 * d < a.dim) {
            const float v = none ? 0.f : acc[i][d] * inv;
            const T r = from_f32< T >(v);
            o[out + tx + 16 * d] = r;
            if(a.o_rest) static_cast< T* >(a.o_rest)[out + tx + 16 * d] = from_f32< T >(v - to_f32(r));
         }
      if(a.lse && tx == 0) a.lse[(int64_t)head * a.q_rows + qs.first + row] = none ? -CUDART_INF_F : m[i] * kLn2 + logf(l[i]);
   }
}

// p and ds of one tile pair into shared memory. TRANS: rows of the stored
// squares are keys. Both come out 0 where the key is masked, out of range, or
// the query row has no kept key.
template < typename S, bool TRANS >
__device__ __forceinline__ void weights(const Args& a, float (&s)[S::R][S::R], float (&dp)[S::R][S::R], const float* lse,
                                        const float* delta, int q0, int q_len, int key0, int kv_len,
                                        const unsigned char* keep, int ty, int tx, float* sp, float* sds)
{
   const float sc = a.scale * kLog2e;
#pragma unroll
   for(int i = 0; i < S::R; ++i)
#pragma unroll
      for(int j = 0; j < S::R; ++j) {
         const int r = ty + 16 * i, c = tx + 16 * j;
         const int row = q0 + (TRANS ? c : r), key = key0 + (TRANS ? r : c);
         float p = 0.f, ds = 0.f;
         if(row < q_len && key < kv_len && (!keep || keep[key])) {
            const float L = lse[row];
            if(L != -CUDART_INF_F) {
               p = exp2_fast(s[i][j] * sc - L * kLog2e);
               ds = p * (dp[i][j] - delta[row]);
            }
         }
         if(sp) sp[r * S::LP + c] = p;
         sds[r * S::LP + c] = ds;
      }
}

template < typename T, typename S >
__global__ void __launch_bounds__(kBlock) k_attn_backward_kv(Args a)
{
   extern __shared__ float sm[];
   float *sk = sm, *sv = sk + S::B * S::LD, *sq = sv + S::B * S::LD, *sg = sq + S::B * S::LD;
   float *sp = sg + S::B * S::LD, *sds = sp + S::B * S::LP;
   const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
   constexpr int PER = kTileRows / S::B;
   const int kv_head = blockIdx.y, group = a.heads / a.kv_heads;
   const Item it = item(a.kv_tiles, a.max_kv, kTileRows, blockIdx.x / PER);
   const Seq qs = locate(a.q_off, a.max_q, a.qs, it.seq), ks = locate(a.kv_off, a.max_kv, a.ks, it.seq);
   const Seq vs = locate(a.kv_off, a.max_kv, a.vs, it.seq);
   const int key0 = it.tile * kTileRows + (blockIdx.x % PER) * S::B;
   if(key0 >= ks.len) return;
   const unsigned char* keep = a.mask ? a.mask + ks.first : nullptr;
   load_tile< T, S >(sk, static_cast< const T* >(a.k) + ks.base + kv_head * a.ks[2], a.ks[1], key0, ks.len, a.dim, keep);
   load_tile< T, S >(sv, static_cast< const T* >(a.v) + vs.base + kv_head * a.vs[2], a.vs[1], key0, ks.len, a.dim, keep);
   float dk[S::R][S::DP / 16], dv[S::R][S::DP / 16];
   clear< S >(dk);
   clear< S >(dv);
   for(int h = kv_head * group; h < (kv_head + 1) * group; ++h) {
      const T* q = static_cast< const T* >(a.q) + qs.base + h * a.qs[2];
      const T* g = static_cast< const T* >(a.go) + (qs.first * a.heads + h) * a.dim;
      const float* lse = a.lse_in + (int64_t)h * a.q_rows + qs.first;
      const float* delta = a.delta + (int64_t)h * a.q_rows + qs.first;
      for(int q0 = 0; q0 < qs.len; q0 += S::B) {
         __syncthreads();
         load_tile< T, S >(sq, q, a.qs[1], q0, qs.len, a.dim, nullptr);
         load_tile< T, S >(sg, g, (int64_t)a.heads * a.dim, q0, qs.len, a.dim, nullptr);
         __syncthreads();
         float s[S::R][S::R], dp[S::R][S::R];
         dots< S >(sk, sq, ty, tx, s);
         dots< S >(sv, sg, ty, tx, dp);
         weights< S, true >(a, s, dp, lse, delta, q0, qs.len, key0, ks.len, keep, ty, tx, sp, sds);
         __syncwarp();
         accumulate< S >(sp, sg, ty, tx, dv);
         accumulate< S >(sds, sq, ty, tx, dk);
      }
   }
#pragma unroll
   for(int i = 0; i < S::R; ++i) {
      const int key = key0 + ty + 16 * i;
      if(key >= ks.len) continue;
      const int64_t out = ((ks.first + key) * a.kv_heads + kv_head) * a.dim;
#pragma unroll
      for(int d = 0; d < S::DP / 16; ++d) {
         const int c = tx + 16 * d;
         if(c >= a.dim) continue;
         static_cast< T* >(a.dk)[out + c] = from_f32< T >(dk[i][d] * a.scale);
         static_cast< T* >(a.dv)[out + c] = from_f32< T >(dv[i][d]);
      }
   }
}

template < typename T, typename S >
__global__ void __launch_bounds__(kBlock) k_attn_backward_q(Args a)
{
   extern __shared__ float sm[];
   float *sq = sm, *sg = sq + S::B * S::LD, *sk = sg + S::B * S::LD, *sv = sk + S::B * S::LD, *sds = sv + S::B * S::LD;
   const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
   constexpr int PER = kTileRows / S::B;
   const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
   const Item it = item(a.q_tiles, a.max_q, kTileRows, blockIdx.x / PER);
   const Seq qs = locate(a.q_off, a.max_q, a.qs, it.seq), ks = locate(a.kv_off, a.max_kv, a.ks, it.seq);
   const Seq vs = locate(a.kv_off, a.max_kv, a.vs, it.seq);
   const int q0 = it.tile * kTileRows + (blockIdx.x % PER) * S::B;
   if(q0 >= qs.len) return;
   const unsigned char* keep = a.mask ? a.mask + ks.first : nullptr;
   load_tile< T, S >(sq, static_cast< const T* >(a.q) + qs.base + head * a.qs[2], a.qs[1], q0, qs.len, a.dim, nullptr);
   load_tile< T, S >(sg, static_cast< const T* >(a.go) + (qs.first * a.heads + head) * a.dim, (int64_t)a.heads * a.dim, q0,
                     qs.len, a.dim, nullptr);
   const T* k = static_cast< const T* >(a.k) + ks.base + kv_head * a.ks[2];
   const T* v = static_cast< const T* >(a.v) + vs.base + kv_head * a.vs[2];
   const float* lse = a.lse_in + (int64_t)head * a.q_rows + qs.first;
   const float* delta = a.delta + (int64_t)head * a.q_rows + qs.first;
   float dq[S::R][S::DP / 16];
   clear< S >(dq);
   for(int key0 = 0; key0 < ks.len; key0 += S::B) {
      __syncthreads();
      load_tile< T, S >(sk, k, a.ks[1], key0, ks.len, a.dim, keep);
      load_tile< T, S >(sv, v, a.vs[1], key0, ks.len, a.dim, keep);
      __syncthreads();
      float s[S::R][S::R], dp[S::R][S::R];
      dots< S >(sq, sk, ty, tx, s);
      dots< S >(sg, sv, ty, tx, dp);
      weights< S, false >(a, s, dp, lse, delta, q0, qs.len, key0, ks.len, keep, ty, tx, nullptr, sds);
      __syncwarp();
      accumulate< S >(sds, sk, ty, tx, dq);
   }
#pragma unroll
   for(int i = 0; i < S::R; ++i) {
      const int row = q0 + ty + 16 * i;
      if(row >= qs.len) continue;
      const int64_t out = ((qs.first + row) * a.heads + head) * a.dim;
#pragma unroll
      for(int d = 0; d < S::DP / 16; ++d)
         if(tx + 16 * d < a.dim) static_cast< T* >(a.dq)[out + tx + 16 * d] = from_f32< T >(dq[i][d] * a.scale);
   }
}

int launch(SmemLimit& limit, const void* fn, dim3 grid, size_t smem, const Args& a, cudaStream_t st, const char* what)
{
   if(grid.x == 0 || grid.y == 0) return RELM_MP_OK;
   int rc = limit(fn, smem, what);
   if(rc) return rc;
   Args copy = a;
   void* args[] = {&copy};
   rc = check_cuda(cudaLaunchKernel(fn, grid, dim3(kBlock), args, smem, st), what);
   return rc ? rc : check_launch(what);
}

template < typename T, int DP >
int forward(const Args& a, int64_t items, cudaStream_t st)
{
   using S = Shape< DP >;
   static SmemLimit limit;
   return launch(limit, (const void*)k_attn_forward< T, S >, dim3((unsigned)(items * (kTileRows / S::B)), a.heads),
                 3 * S::tile + S::square, a, st, "k_attn_forward");
}

template < typename T, int DP >
int backward(const Args& a, int64_t q_items, int64_t kv_items, cudaStream_t st)
{
   using S = Shape< DP >;
   constexpr int PER = kTileRows / S::B;
   static SmemLimit kv_limit, q_limit;
   int rc = launch(kv_limit, (const void*)k_attn_backward_kv< T, S >, dim3((unsigned)(kv_items * PER), a.kv_heads),
                   4 * S::tile + 2 * S::square, a, st, "k_attn_backward_kv");
   if(rc) return rc;
   return launch(q_limit, (const void*)k_attn_backward_q< T, S >, dim3((unsigned)(q_items * PER), a.heads),
                 4 * S::tile + S::square, a, st, "k_attn_backward_q");
}

template < typename T, typename F32, typename F64, typename F128, typename F256 >
int by_dim(int dim, F32 f32, F64 f64, F128 f128, F256 f256)
{
   return dim <= 32 ? f32() : dim <= 64 ? f64() : dim <= 128 ? f128() : f256();
}

template < typename T >
int forward_dim(const Args& a, int64_t items, cudaStream_t st)
{
   return by_dim< T >(a.dim, [&] { return forward< T, 32 >(a, items, st); }, [&] { return forward< T, 64 >(a, items, st); },
                      [&] { return forward< T, 128 >(a, items, st); }, [&] { return forward< T, 256 >(a, items, st); });
}

template < typename T >
int backward_dim(const Args& a, int64_t qi, int64_t ki, cudaStream_t st)
{
   return by_dim< T >(a.dim, [&] { return backward< T, 32 >(a, qi, ki, st); }, [&] { return backward< T, 64 >(a, qi, ki, st); },
                      [&] { return backward< T, 128 >(a, qi, ki, st); }, [&] { return backward< T, 256 >(a, qi, ki, st); });
}

}  // namespace

int simt_forward(relm_mp_dtype dtype, const Args& a, int64_t items, cudaStream_t st)
{
   switch(dtype) {
      case RELM_MP_FLOAT32: return forward_dim< float >(a, items, st);
      case RELM_MP_BFLOAT16: return forward_dim< __nv_bfloat16 >(a, items, st);
      default: return forward_dim< __half >(a, items, st);
   }
}

int simt_backward(relm_mp_dtype dtype, const Args& a, int64_t q_items, int64_t kv_items, cudaStream_t st)
{
   switch(dtype) {
      case RELM_MP_FLOAT32: return backward_dim< float >(a, q_items, kv_items, st);
      case RELM_MP_BFLOAT16: return backward_dim< __nv_bfloat16 >(a, q_items, kv_items, st);
      default: return backward_dim< __half >(a, q_items, kv_items, st);
   }
}

}  // namespace attn
}  // namespace relm_mp
