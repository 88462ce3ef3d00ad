// Attention of single tokens over a packed cache (packed_kv.cuh) on the tensor cores: bfloat16 activations, heads of 64 or 128
// channels, pages of 16 tokens or more.
//
//   score(j, h) = scale q_h . k_j,  k_j = s_jg code_j + o_jg in group g of 64 channels
//               = scale sum_g ( s_jg (q_h . code_j)_g + o_jg (sum of q_h over g) )
//   out_h       = sum_j p_jh v_j / sum_j p_jh = sum_j ( (p_jh s'_jg) code'_j + p_jh o'_jg ) / sum_j p_jh
// so the matrix products run on the codes themselves, which half precision holds exactly, and scales and offsets are applied to
// the 16 x 8 results in float32.  A code needs one AND to become a half: its bits in the low end of a half are the subnormal
// code * 2^-24 (4 bits: every second code stands four bits higher and counts sixteenfold; its q, or its row of the output, is
// divided by 16).  q is scaled by a power of two into the range of half precision (common to the heads of a kv head); the
// weights p s' are rounded to half precision under a running power of two.
//
// The products are transposed, keys (16) x heads (8) and channels (16) x heads (8): with 8 query heads to a kv head or fewer no
// row of a tensor core instruction is empty.  Both operands' other index may be permuted freely, so codes go from shared memory
// to the tensor core in their plain layout: a lane takes 16 neighbouring channels of a key for the scores, and 8 neighbouring
// channels of four keys for the output, whose pairs (key, key) are put together by byte permutation.  The weights pass from the
// score layout to the B operand by a register transpose of 8 x 8.
//
// Bytes are what bounds it (4.5 or 8.5 bits a channel; two products on 16 keys cost ~170 instructions a warp), so the work is cut
// into equal ranges of tiles of 32 keys over all (token, kv head) pairs: one range a block, tile after tile to the block's
// warps.  A warp brings its tiles by bulk copies (one per page and kv head) into a ring of its own, ahead of the pair it works
// on, and shares nothing with the others until the block's part of a pair is merged.  Pairs that were cut between blocks are
// joined by a second kernel.
#include "attention_common.cuh"
#include "packed_kv.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>

#define PD_TILE 32                 // keys of a tile
#define PD_WARPS 8
#define PD_MAX_TOKENS 1024         // tokens of one launch
#define PD_STATUS 71               // reported where a copy did not arrive
#define PD_LOG2E 1.4426950408889634f
#define PD_NO_KEY (-3.0e38f)       // the running maximum before the first key: below every finite score

struct PackedDecode {
  const __nv_bfloat16* q;
  long long q_stride;
  const unsigned char* pages;
  int num_pages;
  const int* tables;
  int bt_stride;
  const int* cu_q_lens;
  const int* context_lens;
  const int* seqs;
  int n;
  __nv_bfloat16* out;
  int nh, nkv, group, chunks;      // heads of a kv head, in chunks of 8 NT
  int page_log2, page_bytes;
  int window;
  float scale, softcap;
  const float* sink;
  const float* slopes;
  float temp_coef, temp_every;
  float* part;                     // [2 * blocks][8 NT * D + 2 * 8 NT]: outputs, then (max, sum) pairs
  int* prefix;                     // [n + 1]
  int blocks, stages;
  int* status;
};

__device__ __forceinline__ void mma_f16(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ unsigned half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ unsigned lds32(unsigned a) { unsigned v; asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a)); return v; }
__device__ __forceinline__ uint2 lds64(unsigned a) { uint2 v; asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a)); return v; }
__device__ __forceinline__ uint4 lds128(unsigned a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

// The keys in sight of token i: [lo, context), counted in tiles from the tile of lo.  A context that its block table
// cannot hold is cut there.
__device__ __forceinline__ void token_keys(const PackedDecode& a, int i, int* seq, int* context, int* lo) {
  const int b = a.seqs ? a.seqs[i] : i;
  long long most = (long long)a.bt_stride << a.page_log2;
  const int c = b >= 0 ? (int)min((long long)a.context_lens[b], most) : 0;
  *seq = b;
  *context = max(c, 0);
  *lo = a.window > 0 ? max(0, c - a.window) : 0;
}
__device__ __forceinline__ int token_tiles(const PackedDecode& a, int i) {
  int b, c, lo;
  token_keys(a, i, &b, &c, &lo);
  return c > lo ? (c + PD_TILE - 1) / PD_TILE - lo / PD_TILE : 0;
}

// prefix[i] = tiles of the tokens before i (of all their pairs), for every block alike
template <int THREADS>
__device__ __forceinline__ void scan_tiles(const PackedDecode& a, int pairs, int* prefix, int* wsum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int i0 = 0; i0 < a.n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const int mine = i < a.n ? token_tiles(a, i) * pairs : 0;
    int v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) wsum[warp] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += wsum[w];
      all += wsum[w];
    }
    if (i < a.n) prefix[i] = base + before + v - mine;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[a.n] = base;
  __syncthreads();
}
__device__ __forceinline__ int range_start(int block, int blocks, int total) { return (int)((long long)total * block / blocks); }

// A place in the sequence of all tiles: tile f lies in pair `pair` of token i, whose tiles are [base, base + tiles).
struct TileCursor {
  int i, pair, base, tiles;
  __device__ __forceinline__ void settle(const int* prefix, int pairs) {   // tiles of token i
    tiles = (prefix[i + 1] - prefix[i]) / pairs;
  }
  __device__ __forceinline__ void start(const int* prefix, int n, int pairs, int f) {
    int lo = 0, hi = n - 1;                       // the last token whose tiles start at f or before and that has any
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (prefix[m] <= f) lo = m; else hi = m - 1;
    }
    i = lo;
    settle(prefix, pairs);
    pair = (f - prefix[i]) / tiles;
    base = prefix[i] + pair * tiles;
  }
  __device__ __forceinline__ void advance(const int* prefix, int pairs, int f) {   // f < prefix[n]
    while (f >= base + tiles) {
      base += tiles;
      if (++pair == pairs) {
        pair = 0;
        do { ++i; settle(prefix, pairs); } while (tiles == 0);
      }
    }
  }
};

template <int D, int BITS, int NT, bool OPT>
__global__ void __launch_bounds__(PD_WARPS * 32, (D == 128 && NT == 1 && BITS == 4) || (D == 64 && NT == 1) ? 2 : 1)
packed_decode_kernel(PackedDecode a) {
  constexpr int GR = D / 64, ROW = D * BITS / 8, HEADS = 8 * NT;
  constexpr int STAGE = 2 * PD_TILE * (ROW + 4 * GR);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int wsum[PD_WARPS];
  __shared__ float top_s[PD_WARPS][HEADS], sum_s[PD_WARPS][HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int pairs = a.nkv * a.chunks;
  // shared memory: rings, merge buffer [WARPS / 2][HEADS * D], barriers, which chunks of a stage are there, prefix
  unsigned char* ring_p = smem + (size_t)warp * a.stages * STAGE;
  float* merge = reinterpret_cast<float*>(smem + (size_t)PD_WARPS * a.stages * STAGE);
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(merge + PD_WARPS / 2 * HEADS * D);
  unsigned* there = reinterpret_cast<unsigned*>(bars + PD_WARPS * a.stages);
  int* prefix = reinterpret_cast<int*>(there + PD_WARPS * a.stages);
  const unsigned ring = tc_smem(ring_p), bar0 = tc_smem(bars + warp * a.stages);
  there += warp * a.stages;
  if (lane == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(bar0 + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();
  scan_tiles<PD_WARPS * 32>(a, pairs, prefix, wsum);
  const int total = prefix[a.n];
  if (blockIdx.x == 0)
    for (int i = tid; i <= a.n; i += PD_WARPS * 32) a.prefix[i] = prefix[i];
  const int f_lo = range_start(blockIdx.x, a.blocks, total), f_hi = range_start(blockIdx.x + 1, a.blocks, total);
  if (f_lo >= f_hi) return;
  if (lane == 0) asm volatile("fence.proxy.async;" ::: "memory");    // pages that the kernel ahead wrote, read by bulk copies

  // chunks: the tokens of a tile that lie in one page, 16 or 32
  const int chunk = a.page_log2 == 4 ? 16 : 32, chunks = PD_TILE / chunk;
  const int chunk_bytes = 2 * chunk * (ROW + 4 * GR);
  const int page_mask = (1 << a.page_log2) - 1;

  // ---- the ring: tile f = f_lo + warp + PD_WARPS * k of this warp goes to stage k % stages
  TileCursor ahead;
  int f_ahead = f_lo + warp, ahead_id = -1;       // the next tile to be asked for, and (lane < chunks) its page
  int ahead_seq = -1, ahead_token = -1, ahead_first = 0, ahead_ctx = 0;
  if (f_ahead < f_hi) ahead.start(prefix, a.n, pairs, f_ahead);
  const int* ahead_row = nullptr;
  auto look_up = [&]() {                          // load the page id of the tile at f_ahead
    if (f_ahead >= f_hi) return;
    ahead.advance(prefix, pairs, f_ahead);
    if (ahead.i != ahead_token) {
      int lo;
      token_keys(a, ahead.i, &ahead_seq, &ahead_ctx, &lo);
      ahead_token = ahead.i;
      ahead_first = lo / PD_TILE * PD_TILE;
      ahead_row = a.tables + (size_t)ahead_seq * a.bt_stride;
    }
    const int key = ahead_first + (f_ahead - ahead.base) * PD_TILE + lane * chunk;
    ahead_id = lane < chunks && key < ahead_ctx ? ahead_row[key >> a.page_log2] : -1;
  };
  auto ask = [&](int stage) {                     // start the copies of the tile at f_ahead
    if (f_ahead >= f_hi) return;
    const bool ok = ahead_id >= 0 && ahead_id < a.num_pages;
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    const unsigned bar = bar0 + 8 * stage;
    if (lane == 0) {
      there[stage] = mask;
      mbar_expect_tx(bar, __popc(mask) * chunk_bytes);
    }
    __syncwarp();
    if (ok) {
      const int key = ahead_first + (f_ahead - ahead.base) * PD_TILE + lane * chunk;
      const unsigned char* block = a.pages + ((size_t)ahead_id * a.nkv + ahead.pair / a.chunks) * a.page_bytes;
      const unsigned dst = ring + stage * STAGE + lane * chunk_bytes;
      if (a.page_log2 == 4) {
        bulk_load(dst, block, chunk_bytes, bar);
      } else {
        const int place = key & page_mask, P = page_mask + 1;
        bulk_load(dst, block + place * ROW, chunk * ROW, bar);
        bulk_load(dst + chunk * ROW, block + (P + place) * ROW, chunk * ROW, bar);
        bulk_load(dst + 2 * chunk * ROW, block + 2 * P * ROW + place * GR * 4, chunk * GR * 4, bar);
        bulk_load(dst + 2 * chunk * ROW + chunk * GR * 4, block + 2 * P * ROW + (P + place) * GR * 4, chunk * GR * 4, bar);
      }
    }
    f_ahead += PD_WARPS;
  };
  look_up();
  for (int s = 0; s < a.stages; ++s) { ask(s); look_up(); }

  // ---- the pairs of this block's range, one after the other
  const int key_g = (g >> 1) + 4 * (g & 1);       // the key (of 16) in row g of the scores; row g + 8 has key_g + 8
  const int step_c = chunk == 16 ? chunk_bytes : 16 * ROW, step_p = chunk == 16 ? chunk_bytes : 16 * GR * 4;   // from 16 keys to the next
  const unsigned off_k = key_g * ROW + t * (2 * BITS);                     // a lane's 16 channels of its key
  const unsigned off_v = chunk * ROW + t * ROW + g * BITS;                 // its 8 channels of keys t, t + 4, t + 8, t + 12
  const unsigned off_kp = 2 * chunk * ROW + key_g * GR * 4, off_vp = off_kp + chunk * GR * 4;
  int stage = 0, f = f_lo + warp;
  unsigned phase = 0;
  bool broken = false;
  TileCursor at;
  at.start(prefix, a.n, pairs, f_lo);
  for (int seg = f_lo; seg < f_hi;) {
    at.advance(prefix, pairs, seg);
    const int seg_end = min(at.base + at.tiles, f_hi);
    int b, ctx, lo;
    token_keys(a, at.i, &b, &ctx, &lo);
    const int first_key = lo / PD_TILE * PD_TILE;
    const int kvh = at.pair / a.chunks, head0 = (at.pair % a.chunks) * HEADS;
    const int heads = min(HEADS, a.group - head0);
    const int row = a.cu_q_lens ? a.cu_q_lens[b] : b;

    float o[GR * 4][NT][4], l[NT][2], r[GR][NT][2], ref[NT][2];
#pragma unroll
    for (int i = 0; i < GR * 4; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt][0] = l[nt][1] = 0.f;
      ref[nt][0] = ref[nt][1] = PD_NO_KEY;
#pragma unroll
      for (int gr = 0; gr < GR; ++gr) r[gr][nt][0] = r[gr][nt][1] = 0.f;
    }
    int vexp = -120;                               // weights are held times 2^(6 - vexp)

    if (f < seg_end) {
      // ---- q of this pair: B operands, and its sums over each group
      unsigned qf[GR][4][NT][2];
      float qsum[GR][NT][2], qfac;
      {
        const float temp = OPT && a.temp_every > 0.f ? 1.f + a.temp_coef * logf(floorf(__fdiv_rn((float)ctx, a.temp_every)) + 1.f) : 1.f;
        const float fac = a.scale * temp * (OPT ? 1.f : PD_LOG2E);
        float x[GR][NT][16];
        float big = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bool mine = nt * 8 + g < heads;
          const __nv_bfloat16* qp = a.q + (size_t)row * a.q_stride + (size_t)(kvh * a.group + head0 + (mine ? nt * 8 + g : 0)) * D + t * 16;
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const uint4 u = mine ? *reinterpret_cast<const uint4*>(qp + gr * 64 + v * 8) : make_uint4(0, 0, 0, 0);
              const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x[gr][nt][v * 8 + 2 * i] = __uint_as_float(w[i] << 16);
                x[gr][nt][v * 8 + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
              }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              sum += x[gr][nt][i];
              big = fmaxf(big, fabsf(x[gr][nt][i]));
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= fac;
            qsum[gr][nt][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
            qsum[gr][nt][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
          }
        }
        big = warp_max(big);
        const int e = max(-90, min(100, 139 - (int)(__float_as_uint(big) >> 23)));   // big * 2^e lies in [2^12, 2^13)
        const float up = power_of_two(e);
        qfac = fac * power_of_two(24 - e);
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const float* y = x[gr][nt];
              if (BITS == 4) {                     // m = 2 * word + (codes four bits up)
                const int c = 8 * (m >> 1) + (m & 1);
                const float u = m & 1 ? up * 0.0625f : up;
                qf[gr][m][nt][0] = half_pair(y[c] * u, y[c + 4] * u);
                qf[gr][m][nt][1] = half_pair(y[c + 2] * u, y[c + 6] * u);
              } else {
                qf[gr][m][nt][0] = half_pair(y[4 * m] * up, y[4 * m + 2] * up);
                qf[gr][m][nt][1] = half_pair(y[4 * m + 1] * up, y[4 * m + 3] * up);
              }
            }
      }
      float slope[NT][2];
      if (OPT) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int h = nt * 8 + 2 * t + j;
            slope[nt][j] = a.slopes && h < heads ? a.slopes[kvh * a.group + head0 + h] : 0.f;
          }
      }

      for (; f < seg_end; f += PD_WARPS) {
        if (!broken) broken = __any_sync(0xffffffffu, !mbar_wait(bar0 + 8 * stage, phase));
        if (broken) {
          if (lane == 0 && a.status) *a.status = PD_STATUS;
        } else {
          const unsigned base = ring + stage * STAGE;
          const int key0 = first_key + (f - at.base) * PD_TILE;
          const unsigned mask = there[stage];
          const bool whole = key0 >= lo && key0 + PD_TILE <= ctx && mask == (1u << chunks) - 1;
          // ---- scores of 32 keys
          float s[2][NT][4];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[kb][nt][0] = s[kb][nt][1] = s[kb][nt][2] = s[kb][nt][3] = 0.f;
            unsigned kp[2][GR];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const unsigned p = base + off_kp + kb * step_p + half * 8 * GR * 4;
              if (GR == 2) {
                const uint2 u = lds64(p);
                kp[half][0] = u.x;
                kp[half][GR - 1] = u.y;
              } else {
                kp[half][0] = lds32(p);
              }
            }
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
              float acc[NT][4];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
              const unsigned kc = base + off_k + kb * step_c + gr * (8 * BITS);
              if (BITS == 4) {
                const uint2 ua = lds64(kc), ub = lds64(kc + 8 * ROW);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  const unsigned wa = w ? ua.y : ua.x, wb = w ? ub.y : ub.x, xa = wa >> 8, xb = wb >> 8;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    mma_f16(acc[nt], wa & 0x000f000fu, wb & 0x000f000fu, xa & 0x000f000fu, xb & 0x000f000fu, qf[gr][2 * w][nt][0], qf[gr][2 * w][nt][1]);
                    mma_f16(acc[nt], wa & 0x00f000f0u, wb & 0x00f000f0u, xa & 0x00f000f0u, xb & 0x00f000f0u, qf[gr][2 * w + 1][nt][0], qf[gr][2 * w + 1][nt][1]);
                  }
                }
              } else {
                const uint4 ua = lds128(kc), ub = lds128(kc + 8 * ROW);
                const unsigned wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma_f16(acc[nt], wa[w] & 0x00ff00ffu, wb[w] & 0x00ff00ffu, (wa[w] >> 8) & 0x00ff00ffu, (wb[w] >> 8) & 0x00ff00ffu,
                            qf[gr][w][nt][0], qf[gr][w][nt][1]);
              }
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float sc = __uint_as_float(kp[half][gr] << 16) * qfac, of = __uint_as_float(kp[half][gr] & 0xffff0000u);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int j = 0; j < 2; ++j)
                    s[kb][nt][2 * half + j] = fmaf(of, qsum[gr][nt][j], fmaf(sc, acc[nt][2 * half + j], s[kb][nt][2 * half + j]));
              }
            }
          }
          if (OPT) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float v = s[kb][nt][i];
                  if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
                  v -= slope[nt][i & 1] * (float)(ctx - 1 - (key0 + 16 * kb + 8 * (i >> 1) + key_g));
                  s[kb][nt][i] = v * PD_LOG2E;
                }
          }
          // pairs of the values, and what is out of sight
          float sv[2][2][GR], ov[2][2][GR];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              unsigned u[GR];
              const unsigned p = base + off_vp + kb * step_p + half * 8 * GR * 4;
              if (GR == 2) {
                const uint2 w = lds64(p);
                u[0] = w.x;
                u[GR - 1] = w.y;
              } else {
                u[0] = lds32(p);
              }
#pragma unroll
              for (int gr = 0; gr < GR; ++gr) {
                sv[kb][half][gr] = __uint_as_float(u[gr] << 16);
                ov[kb][half][gr] = __uint_as_float(u[gr] & 0xffff0000u);
              }
            }
          if (!whole) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int key = key0 + 16 * kb + 8 * half + key_g;
                if (key < lo || key >= ctx || !((mask >> (chunk == 16 ? kb : 0)) & 1)) {
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) s[kb][nt][2 * half] = s[kb][nt][2 * half + 1] = -INFINITY;
#pragma unroll
                  for (int gr = 0; gr < GR; ++gr) sv[kb][half][gr] = ov[kb][half][gr] = 0.f;
                }
              }
          }
          // ---- the running maximum moves only where some score is 2^8 above it
          float mx[NT][2];
          bool over = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mx[nt][j] = fmaxf(fmaxf(s[0][nt][j], s[0][nt][2 + j]), fmaxf(s[1][nt][j], s[1][nt][2 + j]));
              over = over || mx[nt][j] > ref[nt][j] + 8.f;
            }
          if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float m = mx[nt][j];
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                m = fmaxf(m, ref[nt][j]);
                const float al = fast_exp2(ref[nt][j] - m);
                ref[nt][j] = m;
                l[nt][j] *= al;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) r[gr][nt][j] *= al;
#pragma unroll
                for (int i = 0; i < GR * 4; ++i) { o[i][nt][j] *= al; o[i][nt][2 + j] *= al; }
              }
          }
          float pmax = 0.f, smax = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
              for (int gr = 0; gr < GR; ++gr) smax = fmaxf(smax, sv[kb][half][gr]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const float p = fast_exp2(s[kb][nt][2 * half + j] - ref[nt][j]);
                  s[kb][nt][2 * half + j] = p;
                  l[nt][j] += p;
                  pmax = fmaxf(pmax, p);
#pragma unroll
                  for (int gr = 0; gr < GR; ++gr) r[gr][nt][j] = fmaf(p, ov[kb][half][gr], r[gr][nt][j]);
                }
            }
          // ---- the weights' power of two: p s' stays below 2^9 times it
          if (__any_sync(0xffffffffu, pmax * smax > power_of_two(vexp) * 512.f)) {
            float w = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                float p = 0.f, z = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p = fmaxf(p, fmaxf(s[kb][nt][2 * half], s[kb][nt][2 * half + 1]));
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) z = fmaxf(z, sv[kb][half][gr]);
                w = fmaxf(w, p * z);
              }
            w = warp_max(w);
            const int e = max(vexp, min(100, (int)(__float_as_uint(w) >> 23) - 127));
            const float down = vexp - e < -126 ? 0.f : power_of_two(vexp - e);
            vexp = e;
#pragma unroll
            for (int i = 0; i < GR * 4; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][nt][j] *= down;
          }
          const float inv = power_of_two(6 - vexp);
          // ---- output: channels x heads
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
              unsigned pb[NT][2];
              const float w0 = sv[kb][0][gr] * inv, w1 = sv[kb][1][gr] * inv;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                pb[nt][0] = transpose8(half_pair(s[kb][nt][0] * w0, s[kb][nt][1] * w0));
                pb[nt][1] = transpose8(half_pair(s[kb][nt][2] * w1, s[kb][nt][3] * w1));
              }
              const unsigned vc = base + off_v + kb * step_c + gr * (8 * BITS);
              if (BITS == 4) {
                const unsigned w0 = lds32(vc), w1 = lds32(vc + 4 * ROW), w2 = lds32(vc + 8 * ROW), w3 = lds32(vc + 12 * ROW);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                  unsigned x = __byte_perm(w0, w1, v ? 0x7632 : 0x5410), y = __byte_perm(w2, w3, v ? 0x7632 : 0x5410);
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                      mma_f16(o[gr * 4 + 2 * v + i][nt], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[nt][0], pb[nt][1]);
                    x >>= 8;
                    y >>= 8;
                  }
                }
              } else {
                const uint2 w0 = lds64(vc), w1 = lds64(vc + 4 * ROW), w2 = lds64(vc + 8 * ROW), w3 = lds64(vc + 12 * ROW);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  const unsigned sel = v & 1 ? 0x7632 : 0x5410;
                  const unsigned x = v < 2 ? __byte_perm(w0.x, w1.x, sel) : __byte_perm(w0.y, w1.y, sel);
                  const unsigned y = v < 2 ? __byte_perm(w2.x, w3.x, sel) : __byte_perm(w2.y, w3.y, sel);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma_f16(o[gr * 4 + v][nt], x & 0x00ff00ffu, (x >> 8) & 0x00ff00ffu, y & 0x00ff00ffu, (y >> 8) & 0x00ff00ffu, pb[nt][0], pb[nt][1]);
                }
              }
            }
        }
        __syncwarp();                              // every lane has read the stage
        if (!broken) { ask(stage); look_up(); }
        if (++stage == a.stages) { stage = 0; phase ^= 1; }
      }
    }

    // ---- the warps' parts of the pair become one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], m);
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) r[gr][nt][j] += __shfl_xor_sync(0xffffffffu, r[gr][nt][j], m);
        }
    if (g == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top_s[warp][nt * 8 + 2 * t + j] = ref[nt][j];
          sum_s[warp][nt * 8 + 2 * t + j] = l[nt][j];
        }
    }
    __syncthreads();
    float M[NT][2], L[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = nt * 8 + 2 * t + j;
        M[nt][j] = PD_NO_KEY;
        L[nt][j] = 0.f;
        for (int w = 0; w < PD_WARPS; ++w) M[nt][j] = fmaxf(M[nt][j], top_s[w][h]);
        for (int w = 0; w < PD_WARPS; ++w) L[nt][j] += sum_s[w][h] * fast_exp2(top_s[w][h] - M[nt][j]);
        const float fc = fast_exp2(ref[nt][j] - M[nt][j]);
#pragma unroll
        for (int i = 0; i < GR * 4; ++i) {
          const float off = r[i / 4][nt][j];
          o[i][nt][j] = (scalbnf(o[i][nt][j], 18 + vexp) + off) * fc;
          o[i][nt][2 + j] = (scalbnf(o[i][nt][2 + j], (BITS == 4 ? 14 : 18) + vexp) + off) * fc;
        }
      }
    // float4 slots [half of the warps][i, nt][lane]
    float4* slot = reinterpret_cast<float4*>(merge);
    constexpr int REGS = GR * 4 * NT;
#pragma unroll
    for (int w = PD_WARPS / 2; w >= 1; w >>= 1) {
      if (warp >= w && warp < 2 * w) {
#pragma unroll
        for (int i = 0; i < GR * 4; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            slot[((warp - w) * REGS + i * NT + nt) * 32 + lane] = make_float4(o[i][nt][0], o[i][nt][1], o[i][nt][2], o[i][nt][3]);
      }
      __syncthreads();
      if (warp < w) {
#pragma unroll
        for (int i = 0; i < GR * 4; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float4 v = slot[(warp * REGS + i * NT + nt) * 32 + lane];
            o[i][nt][0] += v.x; o[i][nt][1] += v.y; o[i][nt][2] += v.z; o[i][nt][3] += v.w;
          }
      }
      __syncthreads();
    }
    if (warp == 0) {
      const bool complete = seg == at.base && seg_end == at.base + at.tiles;
      // a part that is not the whole pair is the block's first (slot 0) or its last
      float* part = a.part + (size_t)(2 * blockIdx.x + (seg == f_lo ? 0 : 1)) * (HEADS * D + 2 * HEADS);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = nt * 8 + 2 * t + j;
          if (h >= heads) continue;
          float fac = 1.f;
          if (complete) {
            float sum = L[nt][j];
            if (OPT && a.sink) {
              const float sk = a.sink[kvh * a.group + head0 + h] * PD_LOG2E, top = fmaxf(M[nt][j], sk);
              fac = fast_exp2(M[nt][j] - top);
              sum = sum * fac + fast_exp2(sk - top);
            }
            fac = sum != 0.f ? fac / sum : 0.f;
          } else if (g == 0) {
            part[HEADS * D + 2 * h] = M[nt][j];
            part[HEADS * D + 2 * h + 1] = L[nt][j];
          }
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) { y[2 * i] = o[gr * 4 + i][nt][j] * fac; y[2 * i + 1] = o[gr * 4 + i][nt][2 + j] * fac; }
            const int c = gr * 64 + g * 8;
            if (complete) {
              const uint4 u = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
              *reinterpret_cast<uint4*>(a.out + ((size_t)row * a.nh + kvh * a.group + head0 + h) * D + c) = u;
            } else {
              float4* p = reinterpret_cast<float4*>(part + h * D + c);
              p[0] = make_float4(y[0], y[1], y[2], y[3]);
              p[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
          }
        }
    }
    seg = seg_end;
  }
  if (broken) {                                    // leave no copy in flight behind
    for (int s = 0; s < a.stages; ++s) mbar_wait(bar0 + 8 * ((stage + s) % a.stages), stage + s >= a.stages ? phase ^ 1 : phase);
  }
}

// One block per (token, kv head, chunk of heads): joins the parts of a pair that was cut between blocks; a token without a
// key in sight gets zeros.
template <int D, int NT>
__global__ void __launch_bounds__(256) packed_join_kernel(PackedDecode a) {
  constexpr int HEADS = 8 * NT, PART = HEADS * D + 2 * HEADS;
  pdl_trigger();
  pdl_wait();
  const int pairs = a.nkv * a.chunks, i = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  const int b = a.seqs ? a.seqs[i] : i;
  if (b < 0) return;
  const int lo = a.prefix[i], total = a.prefix[a.n], tiles = (a.prefix[i + 1] - lo) / pairs;
  const int kvh = pair / a.chunks, head0 = (pair % a.chunks) * HEADS, heads = min(HEADS, a.group - head0);
  const int row = a.cu_q_lens ? a.cu_q_lens[b] : b;
  const int f0 = lo + pair * tiles, f1 = f0 + tiles;
  int first = 0, last = -1;
  if (tiles) {
    // the block that holds tile f: the largest c with total * c / blocks <= f
    auto holder = [&](int f) {
      int c = (int)(((long long)f * a.blocks) / total);
      while (c + 1 < a.blocks && range_start(c + 1, a.blocks, total) <= f) ++c;
      while (c > 0 && range_start(c, a.blocks, total) > f) --c;
      return c;
    };
    first = holder(f0);
    last = holder(f1 - 1);
    if (first == last) return;                     // whole in one block, which wrote the result
  }
  for (int e = threadIdx.x * 4; e < heads * D; e += blockDim.x * 4) {
    const int h = e / D;
    float M = PD_NO_KEY, L = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    auto part_of = [&](int c) { return a.part + (size_t)(2 * c + (c == first && range_start(c, a.blocks, total) != f0 ? 1 : 0)) * PART; };
    for (int c = first; c <= last; ++c) M = fmaxf(M, part_of(c)[HEADS * D + 2 * h]);
    for (int c = first; c <= last; ++c) {
      const float* p = part_of(c);
      const float w = fast_exp2(p[HEADS * D + 2 * h] - M);
      const float4 v = *reinterpret_cast<const float4*>(p + e);
      L = fmaf(w, p[HEADS * D + 2 * h + 1], L);
      y.x = fmaf(w, v.x, y.x); y.y = fmaf(w, v.y, y.y); y.z = fmaf(w, v.z, y.z); y.w = fmaf(w, v.w, y.w);
    }
    float fac = 1.f;
    if (a.sink) {
      const float sk = a.sink[kvh * a.group + head0 + h] * PD_LOG2E, top = fmaxf(M, sk);
      fac = fast_exp2(M - top);
      L = L * fac + fast_exp2(sk - top);
    }
    fac = L != 0.f ? fac / L : 0.f;
    const uint2 u = make_uint2(pack_bf16(y.x * fac, y.y * fac), pack_bf16(y.z * fac, y.w * fac));
    *reinterpret_cast<uint2*>(a.out + ((size_t)row * a.nh + kvh * a.group + head0) * D + e) = u;
  }
}

// ---------------------------------------------------------------- launchers
extern "C" int gg_packed_decode_mma_ok(int dtype, int d, int page_size, int bits) {
  return dtype == GG_BF16 && (d == 64 || d == 128) && page_size >= 16 && packed_sizes_ok(bits, d, page_size);
}

static int pd_sms() {
  static int n = 0;
  if (!n) {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) n = v;
  }
  return n > 0 ? n : 148;
}

struct PdShape { int nt, chunks, blocks, stages; size_t smem; long long part_floats; };
static size_t pd_smem(int d, int bits, int nt, int n, int stages) {
  const size_t stage = 2 * PD_TILE * (d * bits / 8 + 4 * (d / 64));
  return PD_WARPS * (stages * (stage + 12)) + PD_WARPS / 2 * 8 * nt * d * 4 + (n + 1) * 4;
}
static PdShape pd_shape(int n, int nh, int nkv, int d, int bits, int max_context, int window) {
  PdShape s;
  const int group = nh / nkv;
  s.nt = group > 8 ? 2 : 1;
  s.chunks = (group + 8 * s.nt - 1) / (8 * s.nt);
  const bool two = (d == 128 && s.nt == 1 && bits == 4) || (d == 64 && s.nt == 1);
  const size_t most = two ? 111 * 1024 : 225 * 1024;      // of 228 KB, with what a block has besides
  s.stages = 6;
  while (s.stages > 2 && pd_smem(d, bits, s.nt, n, s.stages) > most) --s.stages;
  s.smem = pd_smem(d, bits, s.nt, n, s.stages);
  const long long reach = window > 0 && window < max_context ? (long long)window + PD_TILE - 1 : max_context;
  const long long tiles = (long long)n * nkv * s.chunks * ((reach + PD_TILE - 1) / PD_TILE);
  const long long want = (tiles + PD_WARPS - 1) / PD_WARPS, fit = (long long)pd_sms() * (two ? 2 : 1);
  s.blocks = (int)(want < 1 ? 1 : want < fit ? want : fit);
  s.part_floats = 2LL * s.blocks * (8 * s.nt * d + 16 * s.nt);
  return s;
}

// Scratch of gg_packed_decode_mma, in floats (the prefix lies behind the parts).
extern "C" long long gg_packed_decode_scratch(int n, int nh, int nkv, int d, int bits, int max_context, int window) {
  return pd_shape(n, nh, nkv, d, bits, max_context, window).part_floats + n + 1;
}

template <int D, int BITS, int NT, bool OPT>
static int pd_launch(const PackedDecode& a, size_t smem, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(packed_decode_kernel<D, BITS, NT, OPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return gg_fail(GG_ERR_CUDA, "packed_decode: %s", cudaGetErrorString(e));
  gg_launch(packed_decode_kernel<D, BITS, NT, OPT>, dim3(a.blocks), dim3(PD_WARPS * 32), smem, stream, a);
  int rc = gg_check_launch("packed_decode");
  if (rc) return rc;
  gg_launch(packed_join_kernel<D, NT>, dim3(a.n * a.nkv * a.chunks), dim3(256), 0, stream, a);
  return gg_check_launch("packed_join");
}

extern "C" int gg_packed_decode_mma(const void* q, long long q_stride, const void* pages, int num_pages, const int* tables, int bt_stride,
                                    const int* cu_q_lens, const int* context_lens, const int* seqs, int n, int max_context, float* scratch,
                                    long long scratch_floats, void* out, int nh, int nkv, int d, int page_size, int bits, int window,
                                    float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every,
                                    int* status, cudaStream_t stream) {
  GG_REQUIRE(gg_packed_decode_mma_ok(GG_BF16, d, page_size, bits), "packed_decode: head size %d, pages of %d tokens or %d bits are not taken", d, page_size, bits);
  GG_REQUIRE(nkv > 0 && nh > 0 && nh % nkv == 0, "packed_decode: %d heads are not a multiple of %d kv heads", nh, nkv);
  GG_REQUIRE(n >= 0 && n <= PD_MAX_TOKENS && num_pages >= 0 && bt_stride > 0 && window >= 0 && max_context >= 0,
             "packed_decode: bad sizes n=%d pages=%d table width=%d window=%d", n, num_pages, bt_stride, window);
  GG_REQUIRE(((size_t)q % 16) == 0 && q_stride % 8 == 0 && ((size_t)out % 16) == 0 && ((size_t)pages % 16) == 0,
             "packed_decode: q, its rows, the output and the pages must start on 16 bytes");
  if (n == 0) return GG_OK;
  const PdShape s = pd_shape(n, nh, nkv, d, bits, max_context, window);
  GG_REQUIRE(scratch && ((size_t)scratch % 16) == 0 && scratch_floats >= s.part_floats + n + 1, "packed_decode: scratch too small");
  PackedDecode a = {};
  a.q = (const __nv_bfloat16*)q; a.q_stride = q_stride; a.pages = (const unsigned char*)pages; a.num_pages = num_pages;
  a.tables = tables; a.bt_stride = bt_stride; a.cu_q_lens = cu_q_lens; a.context_lens = context_lens; a.seqs = seqs; a.n = n;
  a.out = (__nv_bfloat16*)out; a.nh = nh; a.nkv = nkv; a.group = nh / nkv; a.chunks = s.chunks;
  a.page_log2 = 31 - __builtin_clz(page_size);
  a.page_bytes = PackedRows(bits, d, page_size).page_bytes();
  a.window = window; a.scale = scale; a.softcap = softcap; a.sink = sink; a.slopes = slopes; a.temp_coef = temp_coef; a.temp_every = temp_every;
  a.part = scratch; a.prefix = reinterpret_cast<int*>(scratch + s.part_floats); a.blocks = s.blocks; a.stages = s.stages; a.status = status;
  const bool opt = softcap > 0.f || sink || slopes || temp_every > 0.f;
#define PD_OPT(D, BITS, NT) return opt ? pd_launch<D, BITS, NT, true>(a, s.smem, stream) : pd_launch<D, BITS, NT, false>(a, s.smem, stream)
#define PD_NT(D, BITS) do { if (s.nt == 1) PD_OPT(D, BITS, 1); else PD_OPT(D, BITS, 2); } while (0)
  if (d == 64 && bits == 4) PD_NT(64, 4);
  if (d == 64) PD_NT(64, 8);
  if (bits == 4) PD_NT(128, 4);
  PD_NT(128, 8);
}
