// Cross attention on the tensor cores (tcgen05): 2-byte types, head dims up to
// 128, forward.
//
// A block owns QT tiles of 128 query rows of one head and walks the keys in
// tiles of 128. One thread copies k and v tiles by tensor map, one thread issues
// the products, two warps see to masked keys, and four warps per query tile do
// the softmax, a thread per row:
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
constexpr int kBitSlots = 4;

template < int DP, int QT >
struct Fwd {
   static constexpr int ST = QT == 1 && DP == 128 ? 1 : 2; // stages of k and of v
   static constexpr int PANELS = DP / 64;
   static constexpr uint32_t PANEL = kTileRows * 128, TILE = PANELS * PANEL;
   static constexpr uint32_t Q = 0, K = QT * TILE, V = K + ST * TILE, BYTES = V + ST * TILE;
   static constexpr uint32_t COLS = QT == 2 ? 512 : 256, O = QT * 128; // tensor memory: S tiles, then O tiles
   static constexpr int THREADS = QT * 128 + 128;
};

// Largest of 32 scores, in four independent chains.
__device__ __forceinline__ float largest(const uint32_t* s, float top)
{
   float m[4] = {top, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
   for(int i = 0; i < 32; i += 8)
#pragma unroll
      for(int k = 0; k < 4; ++k) m[k] = fmaxf(fmaxf(m[k], __uint_as_float(s[i + 2 * k])), __uint_as_float(s[i + 2 * k + 1]));
   return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

__device__ __forceinline__ void hide(uint32_t* s, unsigned bits)
{
#pragma unroll
   for(int i = 0; i < 32; ++i)
      if(!(bits >> i & 1)) s[i] = 0xff800000u;
}

// 32 scores to weights 2^(sc s - ref), added to `sum` unrounded and packed.
template < typename T >
__device__ __forceinline__ void exponents(const uint32_t* s, uint32_t* p, uint64_t sc, uint64_t ref, uint64_t (&sum)[2])
{
#pragma unroll
   for(int i = 0; i < 16; ++i) {
      float x, y;
      unpair(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc, ref), x, y);
      x = exp2_fast(x);
      y = exp2_fast(y);
      sum[i & 1] = add2(sum[i & 1], pair(x, y));
      p[i] = pack2< T >(x, y);
   }
}

template < typename T, int DP, int QT >
__global__ void __launch_bounds__(Fwd< DP, QT >::THREADS, QT == 1 ? 2 : 1)
   k_attn_tc_forward(Args a, const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                     const __grid_constant__ CUtensorMap vm)
{
   using L = Fwd< DP, QT >;
   extern __shared__ unsigned char raw[];
   unsigned char* sm = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
   __shared__ uint64_t q_full[QT], k_full[L::ST], k_empty[L::ST], v_full[L::ST], v_empty[L::ST], v_clean[L::ST];
   __shared__ uint64_t s_full[QT], p_full[QT][2], o_full[QT], bits_full[kBitSlots], v_last;
   __shared__ unsigned s_bits[kBitSlots][4];
   __shared__ uint32_t tmem_base;
   __shared__ int gave_up;
   const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
   const int head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
   const Item it = item(QT == 2 ? a.q_pairs : a.q_tiles, a.max_q, QT * kTileRows, blockIdx.x);
   const Seq qs = locate(a.q_off, a.max_q, a.qs, it.seq), ks = locate(a.kv_off, a.max_kv, a.ks, it.seq);
   const int row0 = it.tile * QT * kTileRows;
   const int active = QT == 1 || row0 + kTileRows >= qs.len ? 1 : QT;
   const int tiles = (ks.len + kTileRows - 1) / kTileRows;
   const unsigned char* keep = a.mask ? a.mask + ks.first : nullptr;
   constexpr bool BF = std::is_same< T, __nv_bfloat16 >::value;

   if(threadIdx.x == 0) {
      for(int t = 0; t < QT; ++t) {
         mbar_init(&q_full[t], 1);
         mbar_init(&s_full[t], 1);
         mbar_init(&p_full[t][0], 128);
         mbar_init(&p_full[t][1], 128);
         mbar_init(&o_full[t], 1);
      }
      for(int s = 0; s < L::ST; ++s) {
         mbar_init(&k_full[s], 1);
         mbar_init(&k_empty[s], 1);
         mbar_init(&v_full[s], 1);
         mbar_init(&v_empty[s], 1);
         mbar_init(&v_clean[s], 2);
      }
      for(int s = 0; s < kBitSlots; ++s) mbar_init(&bits_full[s], 2);
      mbar_init(&v_last, 1);
      mbar_init_fence();
      gave_up = 0;
   }
   if(warp == QT * 4) tmem_alloc(&tmem_base, L::COLS);
   fence_before();
   __syncthreads();
   fence_after();
   const uint32_t tmem = tmem_base;
   const uint32_t base = smem_addr(sm);
   // Tiles with keys that take no part: all where there is a mask, else the last if it ends inside.
   auto dirty = [&](int j) { return keep != nullptr || ks.len - j * kTileRows < kTileRows; };
   auto dirty_parity = [&](int round) { return keep ? round & 1 : 0; };

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
      if(elect_one() && tiles > 0) {
         const int steps = (a.dim + 15) / 16;
         const uint32_t pv = instruction(BF, 128, steps * 16, true);
         auto keys16 = [&](int j) { return min(kTileRows, (ks.len - j * kTileRows + 15) / 16 * 16); };
         auto scores = [&](int t, int j) {
            product_columns< DP, kTileRows, kTileRows >(tmem + t * 128, base + L::Q + t * L::TILE, base + L::K + (j % L::ST) * L::TILE,
                                                        instruction(BF, 128, keys16(j), false), steps);
            mma_commit(&s_full[t]);
         };
         bool ok = mbar_wait(&k_full[0], 0);
         for(int t = 0; t < active && ok; ++t) {
            ok = mbar_wait(&q_full[t], 0);
            if(ok) scores(t, 0);
         }
         if(ok) mma_commit(&k_empty[0]);
         for(int j = 0; j < tiles && ok; ++j) {
            const int n = keys16(j) / 16, s = j % L::ST, round = j / L::ST;
            ok = mbar_wait(&v_full[s], round & 1);
            if(ok && dirty(j)) {
               if(!keep) mbar_arrive(&v_last);
               ok = mbar_wait(&v_clean[s], dirty_parity(round));
            }
            for(int t = 0; t < active && ok; ++t) {
               const uint32_t va = base + L::V + s * L::TILE;
               // The weights come in two halves of 64 keys.
               if(!(ok = mbar_wait(&p_full[t][0], j & 1))) break;
               fence_after();
               product_rows< 0, 4, 0, kTileRows >(tmem + L::O + t * DP, tmem + t * 128, va, pv, n, j > 0);
               if(!(ok = mbar_wait(&p_full[t][1], j & 1))) break;
               fence_after();
               product_rows< 4, 4, 0, kTileRows >(tmem + L::O + t * DP, tmem + t * 128, va, pv, n, true);
               if(j + 1 == tiles) mma_commit(&o_full[t]);
               else {
                  ok = mbar_wait(&k_full[(j + 1) % L::ST], ((j + 1) / L::ST) & 1);
                  if(ok) scores(t, j + 1);
               }
            }
            if(!ok) break;
            mma_commit(&v_empty[s]);
            if(j + 1 < tiles) mma_commit(&k_empty[(j + 1) % L::ST]);
         }
         if(!ok) {
            gave_up = 1;
            // Products in flight read shared and tensor memory: wait for them before the block ends.
            mma_commit(&q_full[0]);
            mbar_wait(&q_full[0], 1);
         }
      }
   } else if(warp >= QT * 4 + 2) { // masks: 64 keys of each tile per warp
      const int w = warp - (QT * 4 + 2);
      for(int j = keep ? 0 : max(tiles - 1, 0); j < tiles; ++j) {
         if(!dirty(j)) break;
         const int left = ks.len - j * kTileRows, s = j % L::ST;
         unsigned bits[2];
#pragma unroll
         for(int c = 0; c < 2; ++c) {
            const int key = w * 64 + c * 32 + lane;
            bits[c] = __ballot_sync(~0u, key < left && (!keep || keep[j * kTileRows + key]));
         }
         // The slot's last reader was tile j - 4; v of tile j - 1 arrived after the products of tile j - 3 or later.
         if(keep && lane == 0) {
            s_bits[j % kBitSlots][2 * w] = bits[0];
            s_bits[j % kBitSlots][2 * w + 1] = bits[1];
            mbar_arrive(&bits_full[j % kBitSlots]);
         }
         // Without a mask this warp has not followed the phases of v_full: it is called for the last tile.
         if(!__all_sync(~0u, (keep || mbar_wait(&v_last, 0)) && mbar_wait(&v_full[s], (j / L::ST) & 1))) {
            gave_up = 1;
            break;
         }
#pragma unroll
         for(int c = 0; c < 2; ++c)
            if(!(bits[c] >> lane & 1))
               for(int p = 0; p < L::PANELS; ++p) {
                  uint4* line = reinterpret_cast< uint4* >(sm + L::V + s * L::TILE + p * L::PANEL + (w * 64 + c * 32 + lane) * 128);
#pragma unroll
                  for(int i = 0; i < 8; ++i) line[i] = make_uint4(0, 0, 0, 0);
               }
         fence_async_proxy();
         __syncwarp();
         if(lane == 0) mbar_arrive(&v_clean[s]);
      }
   } else { // softmax: thread = row of tile t
      const int t = warp >> 2;
      const uint32_t lanes = tmem + ((uint32_t)(warp & 3) * 32 << 16), st = lanes + t * 128, ot = lanes + L::O + t * DP;
      const float sc = a.scale * kLog2e;
      const uint64_t sc2 = pair(sc, sc);
      float m = -CUDART_INF_F;
      uint64_t sum[2] = {0, 0};
      bool ok = true;
      if(t < active) {
         for(int j = 0; j < tiles && ok; ++j) {
            const int left = ks.len - j * kTileRows, chunks = min(4, (left + 31) / 32);
            unsigned bits[4] = {~0u, ~0u, ~0u, ~0u};
            const bool partial = dirty(j);
            if(keep) {
               ok = __all_sync(~0u, mbar_wait(&bits_full[j % kBitSlots], (j / kBitSlots) & 1));
#pragma unroll
               for(int c = 0; c < 4; ++c) bits[c] = s_bits[j % kBitSlots][c];
            } else if(partial) {
#pragma unroll
               for(int c = 0; c < 4; ++c) bits[c] = left >= 32 * c + 32 ? ~0u : left <= 32 * c ? 0u : (1u << (left - 32 * c)) - 1u;
            }
            ok = ok && __all_sync(~0u, mbar_wait(&s_full[t], j & 1));
            if(!ok) break;
            fence_after();
            uint32_t s[QT == 2 ? 128 : 64];
            float top = -CUDART_INF_F;
            if constexpr(QT == 2) {
#pragma unroll
               for(int c = 0; c < 4; ++c)
                  if(c < chunks) tmem_ld32(s + c * 32, st + c * 32);
               wait_ld();
               loaded< 128 >(s);
#pragma unroll
               for(int c = 0; c < 4; ++c) {
                  if(c >= chunks) continue;
                  if(partial) hide(s + c * 32, bits[c]);
                  top = largest(s + c * 32, top);
               }
            } else { // two blocks share the registers: the scores are read twice, 32 at a time
               tmem_ld32(s, st);
#pragma unroll
               for(int c = 0; c < 4; ++c) {
                  if(c >= chunks) continue;
                  wait_ld();
                  loaded< 32 >(s + (c & 1) * 32);
                  if(c + 1 < chunks) tmem_ld32(s + (~c & 1) * 32, st + (c + 1) * 32);
                  if(partial) hide(s + (c & 1) * 32, bits[c]);
                  top = largest(s + (c & 1) * 32, top);
               }
               tmem_ld32(s, st);
            }
            top *= sc;
            float f = 1.f;
            if(top > m + kGrow || (m == -CUDART_INF_F && top > m)) {
               f = exp2_fast(m - top);
               m = top;
               sum[0] = mul2(sum[0], pair(f, f));
               sum[1] = mul2(sum[1], pair(f, f));
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
            const uint64_t ref2 = pair(-ref, -ref);
#pragma unroll
            for(int c = 0; c < 4; ++c) {
               if(c < chunks) {
                  uint32_t p[16];
                  if constexpr(QT == 2) {
                     exponents< T >(s + c * 32, p, sc2, ref2, sum);
                  } else {
                     wait_ld();
                     loaded< 32 >(s + (c & 1) * 32);
                     if(c + 1 < chunks) tmem_ld32(s + (~c & 1) * 32, st + (c + 1) * 32);
                     if(partial) hide(s + (c & 1) * 32, bits[c]);
                     exponents< T >(s + (c & 1) * 32, p, sc2, ref2, sum);
                     // The next scores lie from column 32 (c + 1) on, these weights before column 16 (c + 1).
                  }
                  tmem_st16(st + c * 16, p);
               }
               if(c & 1) {
                  wait_st();
                  fence_before();
                  mbar_arrive(&p_full[t][c >> 1]);
               }
            }
         }
         float l, l1;
         unpair(add2(sum[0], sum[1]), l, l1);
         l += l1;
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
   static SmemLimit limit;
   int rc = limit((const void*)k_attn_tc_forward< T, DP, QT >, bytes, "k_attn_tc_forward");
   if(rc) return rc;
   k_attn_tc_forward< T, DP, QT ><<< dim3((unsigned)items, a.heads), L::THREADS, bytes, st >>>(a, m.q, m.k, m.v);
   return check_launch("k_attn_tc_forward");
}

template < typename T >
int forward(const Args& a, const TcMaps& m, int64_t tiles, int64_t pairs, cudaStream_t st)
{
   const bool two = 2 * tiles >= 3 * pairs && pairs * a.heads >= 148;
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
