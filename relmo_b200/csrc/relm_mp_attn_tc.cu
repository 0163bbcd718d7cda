// Cross attention on the tensor cores (tcgen05): 2-byte types, head dims up to
// 128, forward.
//
// A block owns QT tiles of 128 query rows of one head and walks the keys in
// tiles of 128. One thread copies k and v tiles by tensor map, one thread issues
// the products, and four warps per query tile do the softmax, a thread per row:
//
//   S = Q K^T          both operands in shared memory, S (float32) in tensor memory
//   P = 2^(sc S - m)   rounded to the inputs' type, written over S
//   O += P V           P in tensor memory, V in shared memory, O in tensor memory
//
// The reference m of a row follows its running maximum only when that has grown
// by more than 8 (in log2): any reference gives the same quotient, weights stay
// below 2^8, and O is rescaled rarely. l, the sum of the unrounded weights, is
// float32. With two tiles per block the products of one overlap the softmax of
// the other, and both read the same k and v from shared memory.
//
// Keys outside the sequence or masked get weight 0; their rows of v are zeroed
// in shared memory first, as 0 times an infinity or NaN would not be 0.
#include <math_constants.h>

#include <type_traits>

#include "relm_mp_attn_tc.cuh"

namespace relm_mp {
namespace attn {
namespace {

using namespace tc;

constexpr float kGrow = 8.f;

template < int DP, int QT >
struct Fwd {
   static constexpr int ST = QT == 1 && DP == 128 ? 1 : 2; // stages of k and of v
   static constexpr int PANELS = DP / 64;
   static constexpr uint32_t PANEL = kTileRows * 128, TILE = PANELS * PANEL;
   static constexpr uint32_t Q = 0, K = QT * TILE, V = K + ST * TILE, BYTES = V + ST * TILE;
   static constexpr uint32_t COLS = QT == 2 ? 512 : 256, O = QT * 128; // tensor memory: S tiles, then O tiles
   static constexpr int THREADS = QT * 128 + 64;
};

template < typename T, int DP, int QT >
__global__ void __launch_bounds__(Fwd< DP, QT >::THREADS, QT == 1 ? 2 : 1)
   k_attn_tc_forward(Args a, const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                     const __grid_constant__ CUtensorMap vm)
{
   using L = Fwd< DP, QT >;
   extern __shared__ unsigned char raw[];
   unsigned char* sm = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
   __shared__ uint64_t q_full[QT], k_full[L::ST], k_empty[L::ST], v_full[L::ST], v_empty[L::ST], s_full[QT], p_full[QT], o_full[QT];
   __shared__ uint32_t tmem_base;
   __shared__ int gave_up;
   const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
   const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
   const Item it = item(QT == 2 ? a.q_pairs : a.q_tiles, a.max_q, QT * kTileRows, blockIdx.x);
   const Seq qs = locate(a.q_off, a.max_q, a.qs, it.seq), ks = locate(a.kv_off, a.max_kv, a.ks, it.seq);
   const int row0 = it.tile * QT * kTileRows;
   const int active = QT == 1 || row0 + kTileRows >= qs.len ? 1 : QT;
   const int tiles = (ks.len + kTileRows - 1) / kTileRows;
   constexpr bool BF = std::is_same< T, __nv_bfloat16 >::value;

   if(threadIdx.x == 0) {
      for(int t = 0; t < QT; ++t) {
         mbar_init(&q_full[t], 1);
         mbar_init(&s_full[t], 1);
         mbar_init(&p_full[t], 128);
         mbar_init(&o_full[t], 1);
      }
      for(int s = 0; s < L::ST; ++s) {
         mbar_init(&k_full[s], 1);
         mbar_init(&k_empty[s], 1);
         mbar_init(&v_full[s], 1);
         mbar_init(&v_empty[s], 1);
      }
      mbar_init_fence();
      gave_up = 0;
   }
   if(warp == QT * 4) tmem_alloc(&tmem_base, L::COLS);
   fence_before();
   __syncthreads();
   fence_after();
   const uint32_t tmem = tmem_base;
   const uint32_t base = smem_addr(sm);

   if(warp == QT * 4 + 1) { // copies
      if(lane == 0 && tiles > 0) {
         const int qr = (int)(a.q_off ? qs.first : 0) + row0, kr = (int)(a.kv_off ? ks.first : 0);
         const int b = a.q_off ? 0 : it.seq;
         auto load = [&](uint32_t dst, const CUtensorMap* m, uint64_t* bar, int row, int h) {
            mbar_expect(bar, L::TILE);
            for(int p = 0; p < L::PANELS; ++p) tma_load(dst + p * L::PANEL, m, bar, p * 64, row, h, b);
         };
         bool ok = true;
         for(int t = 0; t < active; ++t) load(base + L::Q + t * L::TILE, &qm, &q_full[t], qr + t * kTileRows, head);
         int issued = 0;
         for(int j = 0; j < tiles && ok; ++j) {
            const int s = j % L::ST, round = j / L::ST;
            if(round) ok = mbar_wait(&k_empty[s], (round - 1) & 1);
            if(!ok) break;
            load(base + L::K + s * L::TILE, &km, &k_full[s], kr + j * kTileRows, kv_head);
            if(round) ok = mbar_wait(&v_empty[s], (round - 1) & 1);
            if(!ok) { // k of this round is on its way, v is not
               mbar_wait(&k_full[s], round & 1);
               break;
            }
            load(base + L::V + s * L::TILE, &vm, &v_full[s], kr + j * kTileRows, kv_head);
            issued = j + 1;
         }
         if(!ok) { // nothing may still be written to shared memory when the block ends
            gave_up = 1;
            for(int t = 0; t < active; ++t) mbar_wait(&q_full[t], 0);
            for(int j = issued > L::ST ? issued - L::ST : 0; j < issued; ++j) {
               mbar_wait(&k_full[j % L::ST], (j / L::ST) & 1);
               mbar_wait(&v_full[j % L::ST], (j / L::ST) & 1);
            }
         }
      }
   } else if(warp == QT * 4) { // products
      if(lane == 0 && tiles > 0) {
         const int steps = (a.dim + 15) / 16;
         const uint32_t pv = instruction(BF, 128, steps * 16, true);
         auto keys16 = [&](int j) { return min(kTileRows, (ks.len - j * kTileRows + 15) / 16 * 16); };
         auto scores = [&](int t, int j) {
            const uint32_t qa = base + L::Q + t * L::TILE, ka = base + L::K + (j % L::ST) * L::TILE;
            const uint32_t id = instruction(BF, 128, keys16(j), false);
            for(int i = 0; i < steps; ++i) {
               const uint32_t off = (i >> 2) * L::PANEL + (i & 3) * 32;
               mma_ss(tmem + t * 128, operand(qa + off, 16, 1024), operand(ka + off, 16, 1024), id, i > 0);
            }
            mma_commit(&s_full[t]);
         };
         bool ok = mbar_wait(&k_full[0], 0);
         for(int t = 0; t < active && ok; ++t) {
            ok = mbar_wait(&q_full[t], 0);
            if(ok) scores(t, 0);
         }
         if(ok) mma_commit(&k_empty[0]);
         for(int j = 0; j < tiles && ok; ++j) {
            const int n = keys16(j) / 16;
            for(int t = 0; t < active && ok; ++t) {
               ok = mbar_wait(&p_full[t], j & 1) && mbar_wait(&v_full[j % L::ST], (j / L::ST) & 1);
               if(!ok) break;
               fence_after();
               const uint32_t va = base + L::V + (j % L::ST) * L::TILE;
               for(int i = 0; i < n; ++i)
                  mma_ts(tmem + L::O + t * DP, tmem + t * 128 + i * 8, operand(va + i * 2048, L::PANEL, 1024), pv, j > 0 || i > 0);
               if(j + 1 == tiles) mma_commit(&o_full[t]);
               else {
                  ok = mbar_wait(&k_full[(j + 1) % L::ST], ((j + 1) / L::ST) & 1);
                  if(ok) scores(t, j + 1);
               }
            }
            if(!ok) break;
            mma_commit(&v_empty[j % L::ST]);
            if(j + 1 < tiles) mma_commit(&k_empty[(j + 1) % L::ST]);
         }
         if(!ok) {
            gave_up = 1;
            // Products in flight read shared and tensor memory: wait for them before the block ends.
            mma_commit(&q_full[0]);
            mbar_wait(&q_full[0], 1);
         }
      }
   } else { // softmax: thread = row of tile t
      const int t = warp >> 2, row = threadIdx.x & 127;
      const uint32_t lanes = tmem + ((uint32_t)(warp & 3) * 32 << 16), st = lanes + t * 128, ot = lanes + L::O + t * DP;
      const unsigned char* keep = a.mask ? a.mask + ks.first : nullptr;
      const float sc = a.scale * kLog2e;
      float m = -CUDART_INF_F, l = 0.f;
      bool ok = true;
      if(t < active) {
         for(int j = 0; j < tiles && ok; ++j) {
            const int left = ks.len - j * kTileRows, chunks = min(4, (left + 31) / 32);
            unsigned bits[4];
            bool all = left >= kTileRows && !keep;
#pragma unroll
            for(int c = 0; c < 4; ++c) {
               if(all) bits[c] = ~0u;
               else {
                  const int key = c * 32 + lane;
                  bits[c] = __ballot_sync(~0u, key < left && (!keep || keep[j * kTileRows + key]));
               }
            }
            all = all || (bits[0] & bits[1] & bits[2] & bits[3]) == ~0u;
            if(!all && t == 0) { // rows of v that take no part
               ok = __all_sync(~0u, mbar_wait(&v_full[j % L::ST], (j / L::ST) & 1));
               if(!ok) break;
               const bool in = bits[0] >> lane & 1, in1 = bits[1] >> lane & 1, in2 = bits[2] >> lane & 1, in3 = bits[3] >> lane & 1;
               const bool mine = (warp & 3) == 0 ? in : (warp & 3) == 1 ? in1 : (warp & 3) == 2 ? in2 : in3;
               if(!mine) {
                  for(int p = 0; p < L::PANELS; ++p) {
                     uint4* line = reinterpret_cast< uint4* >(sm + L::V + (j % L::ST) * L::TILE + p * L::PANEL + row * 128);
#pragma unroll
                     for(int i = 0; i < 8; ++i) line[i] = make_uint4(0, 0, 0, 0);
                  }
               }
               fence_async_proxy();
            }
            ok = __all_sync(~0u, mbar_wait(&s_full[t], j & 1));
            if(!ok) break;
            fence_after();
            uint32_t s[128];
#pragma unroll
            for(int c = 0; c < 4; ++c)
               if(c < chunks) tmem_ld32(s + c * 32, st + c * 32);
            wait_ld();
            loaded< 128 >(s);
            float top = -CUDART_INF_F;
#pragma unroll
            for(int c = 0; c < 4; ++c) {
               if(c >= chunks) continue;
               if(!all) {
#pragma unroll
                  for(int i = 0; i < 32; ++i)
                     if(!(bits[c] >> i & 1)) s[c * 32 + i] = 0xff800000u;
               }
#pragma unroll
               for(int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(s[c * 32 + i]));
            }
            top *= sc;
            float f = 1.f;
            if(top > m + kGrow || (m == -CUDART_INF_F && top > m)) {
               f = exp2_fast(m - top);
               m = top;
               l *= f;
            }
            if(j > 0 && __any_sync(~0u, f != 1.f)) { // the products into O so far were done before this S
               for(int c = 0; c < a.dim; c += 16) {
                  uint32_t o[16];
                  tmem_ld16(o, ot + c);
                  wait_ld();
                  loaded< 16 >(o);
#pragma unroll
                  for(int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                  tmem_st16(ot + c, o);
               }
            }
            const float ref = m == -CUDART_INF_F ? 0.f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for(int c = 0; c < 4; ++c) {
               if(c >= chunks) continue;
               uint32_t p[16];
#pragma unroll
               for(int i = 0; i < 16; ++i) {
                  const float x = exp2_fast(fmaf(__uint_as_float(s[c * 32 + 2 * i]), sc, -ref));
                  const float y = exp2_fast(fmaf(__uint_as_float(s[c * 32 + 2 * i + 1]), sc, -ref));
                  sum[i & 3] += x + y;
                  p[i] = pack2< T >(x, y);
               }
               tmem_st16(st + c * 16, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            wait_st();
            fence_before();
            mbar_arrive(&p_full[t]);
         }
         if(ok && tiles > 0) ok = __all_sync(~0u, mbar_wait(&o_full[t], 0));
         fence_after();
         // Rows leave through the q tile's shared memory (its products are done), 16 bytes a lane along the rows.
         const bool none = l == 0.f;
         const float inv = none ? 0.f : 1.f / l;
         const int r0 = row0 + t * kTileRows + (warp & 3) * 32;
         unsigned char* stage = sm + L::Q + t * L::TILE + (warp & 3) * 32 * (DP * 2);
         for(int pass = 0; pass < (a.o_rest ? 2 : 1); ++pass) {
#pragma unroll
            for(int c = 0; c < DP; c += 16) {
               if(c >= a.dim) break;
               uint32_t o[16];
               if(tiles > 0) {
                  tmem_ld16(o, ot + c);
                  wait_ld();
                  loaded< 16 >(o);
               }
               uint32_t w[8];
#pragma unroll
               for(int i = 0; i < 8; ++i) {
                  float x = tiles == 0 || none ? 0.f : __uint_as_float(o[2 * i]) * inv, y = tiles == 0 || none ? 0.f : __uint_as_float(o[2 * i + 1]) * inv;
                  if(!ok) x = y = CUDART_NAN_F; // a wait gave up: nothing here is a result
                  w[i] = pack2< T >(x, y);
                  if(pass) w[i] = pack2< T >(x - low2< T >(w[i]), y - high2< T >(w[i]));
               }
#pragma unroll
               for(int h = 0; h < 2; ++h)
                  *reinterpret_cast< uint4* >(stage + lane * (DP * 2) + (((c >> 3) + h) ^ (lane & 7)) * 16) =
                     make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
            }
            __syncwarp();
            T* out = static_cast< T* >(pass ? a.o_rest : a.o);
            constexpr int CH = DP / 8;
#pragma unroll 4
            for(int i = lane; i < 32 * CH; i += 32) {
               const int r = i / CH, c = i % CH;
               if(r0 + r < qs.len && c * 8 < a.dim)
                  *reinterpret_cast< uint4* >(out + ((qs.first + r0 + r) * a.heads + head) * a.dim + c * 8) =
                     *reinterpret_cast< const uint4* >(stage + r * (DP * 2) + ((c ^ (r & 7)) * 16));
            }
            __syncwarp();
         }
         if(a.lse && r0 + lane < qs.len) {
            float v = none ? -CUDART_INF_F : m * kLn2 + logf(l);
            a.lse[(int64_t)head * a.q_rows + qs.first + r0 + lane] = ok ? v : CUDART_NAN_F;
         }
         if(!ok) gave_up = 1;
      }
   }
   fence_before();
   __syncthreads();
   fence_after();
   if(warp == QT * 4) tmem_free(tmem, L::COLS);
   if(threadIdx.x == 0 && gave_up) atomicExch(a.gave_up, 1);
}

template < typename T, int DP, int QT >
int launch(const Args& a, const TcMaps& m, int64_t items, cudaStream_t st)
{
   using L = Fwd< DP, QT >;
   constexpr int bytes = (int)L::BYTES + 1024;
   int rc = check_cuda(cudaFuncSetAttribute(k_attn_tc_forward< T, DP, QT >, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "k_attn_tc_forward");
   if(rc) return rc;
   k_attn_tc_forward< T, DP, QT ><<< dim3((unsigned)items, a.heads), L::THREADS, bytes, st >>>(a, m.q, m.k, m.v);
   return check_launch("k_attn_tc_forward");
}

template < typename T >
int forward(const Args& a, const TcMaps& m, int64_t tiles, int64_t pairs, cudaStream_t st)
{
   const bool two = a.max_q > kTileRows && pairs * a.heads >= 148;
   if(a.dim <= 64) return two ? launch< T, 64, 2 >(a, m, pairs, st) : launch< T, 64, 1 >(a, m, tiles, st);
   return two ? launch< T, 128, 2 >(a, m, pairs, st) : launch< T, 128, 1 >(a, m, tiles, st);
}

}  // namespace

int tc_forward(relm_mp_dtype dtype, const Args& a, int64_t tiles, int64_t pairs, cudaStream_t st)
{
   TcMaps m;
   int rc;
   if((rc = tc_map(&m.q, dtype, a.q, a.qs, a.dim, a.heads, a.q_off ? a.q_rows : a.max_q, a.q_off ? 1 : a.seqs)) ||
      (rc = tc_map(&m.k, dtype, a.k, a.ks, a.dim, a.kv_heads, a.kv_off ? a.kv_rows : a.max_kv, a.kv_off ? 1 : a.seqs)) ||
      (rc = tc_map(&m.v, dtype, a.v, a.vs, a.dim, a.kv_heads, a.kv_off ? a.kv_rows : a.max_kv, a.kv_off ? 1 : a.seqs)))
      return rc;
   return dtype == RELM_MP_BFLOAT16 ? forward< __nv_bfloat16 >(a, m, tiles, pairs, st) : forward< __half >(a, m, tiles, pairs, st);
}

}  // namespace attn
}  // namespace relm_mp
