// Attention of single tokens, and in float32 of prompt portions, over a packed cache (packed_kv.cuh) on the tensor cores: heads of 64 or
// 128 channels, pages of 16 tokens or more.
//
//   score(j, h) = scale q_h . k_j,  k_j = s_jg code_j + o_jg in group g of 64 channels
//               = scale sum_g ( s_jg (q_h . code_j)_g + o_jg (sum of q_h over g) )
//   out_h       = sum_j p_jh v_j / sum_j p_jh = sum_j ( (p_jh s'_jg) code'_j + p_jh o'_jg ) / sum_j p_jh
// so the matrix products run on the codes themselves, and scales and offsets are applied to the 16 x 8 results in float32.
//
// A code needs one AND to become a half, which holds it exactly: its bits in the low end of a half are the subnormal
// code * 2^-24 (4 bits: every second code stands four bits higher and counts sixteenfold; its q, or its row of the output, is
// divided by 16).  (Codes as e4m3 numbers, four an AND, are slower: their products become conversions and products of halves, 75
// us where this takes 56.)  q is brought into the range of half precision by a power of two for each head; the weights p s' are
// rounded to half precision under a running power of two of each head.
//
// The products are transposed, keys (16) x heads (8) and channels (16) x heads (8): with 8 query heads to a kv head or fewer no
// row of a tensor core instruction is empty.  Both operands' other index may be permuted freely, so codes go from shared memory
// to the tensor core in their plain layout: a lane takes 16 neighbouring channels of a key for the scores, and 8 neighbouring
// channels of four keys for the output, whose pairs (key, key) are put together by byte permutation.  The weights pass from the
// score layout to the B operand by a register transpose of 8 x 8.
//
// Its floor are the bytes (4.5 or 8.5 bits a channel); what bounds it are warps that wait on their own chains, no unit being busy for more than
// 60 %, the instructions that make operands of codes most.  The work is cut into equal ranges of tiles over all (token, kv head) pairs, a range for each warp.  A warp brings its tiles into a
// ring of its own by 16-byte asynchronous copies (bulk copies, one a page, were started by one lane after the other with more
// instructions than ten copies of all lanes take), the pages of its next 16 or 32 tiles found by one lane each, and shares
// nothing until it is done: a pair that lies inside its range is written out, parts of pairs are joined inside the block and
// then, by a second kernel, between blocks.  Measured (32 and 8 heads of 128, 4 bits): 64 contexts of 2730 tokens on average, 215 MB, 56 us =
// 3.8 TB/s (copies alone 44 us, products alone on what is there 48 us, 10 us of launch, look-ups and joins in all of them); a context
// of 100003, 115 MB, 37.7 us; one of 700, 10 us.
//
// float32 (EXACT): a query or weight is two halves, each with 11 bits of it, and codes are exact, so two products keep float32's precision (off by
// 2e-7 of 64 bits up to 4000 keys, 1e-6 at 120000; products of float32 values on the general kernels were 4e-7 and took 30 times as long).
// Codes are taken less the middle one there, and a tile's output is summed apart, for tensor cores truncate where they add: with sums carried
// through them 120000 keys were off by 7e-6 (and 4 to 6 % faster).  Prompt portions are single tokens too, as many neighbouring rows to an item
// as fill the eight columns, each with its own context: two portions of 350 rows behind 3000 keys, 32 and 8 heads, 419 us (reading the
// cache back into plain pages for the float32 prompt kernel took 9126).
#include "attention_common.cuh"
#include "packed_kv.cuh"

#include <cuda_fp16.h>

#include <atomic>

#define PD_MAX_TOKENS 512          // tokens of one launch
// Tiles of a block below which fewer blocks are launched (us for 1, 2, 4 and 8: one token of 4000 keys of one kv head 16.0 14.0
// 12.4 12.6; 2000 keys of eight 12.1 12.1 11.9 11.5, 4000 keys 11.1 11.1 11.1 12.5).
#define PD_EACH 4
// Tiles a warp up to which a single token's pairs get a block each (us with and without, eight kv heads of 128 in 4 bits: 200 keys
// 7.2 9.1, 700 keys 10.1 11.0, 1400 keys 12.7 11.3).
#define PD_ALONE 2
// Warps of a block for float32 (us with 8 and 12: the portions above 445 419, one of 600 rows of 40 heads 243 189, a context of 20000 of 40 heads 54 53, three
// of 8000 of four kv heads 15.1 17.1; with 16, heads of 128 spill 132 to 296 bytes, with 12 4 to 28).
#define PD_EXACT_WARPS 12
// Keys of all (token, kv head) pairs from which more than eight heads of a kv head take sixteen columns at a time (twice the registers, so 8 warps for
// 16), below which they go eight by eight, each key read as often (us, sixteen and eight, 4 bits: 16 heads on one kv head of 128, one token of 20000
// keys 19.2 16.3, 24 of up to 4000 18.6 15.7, 64 of 8000 33.6 32.0; 32 on two, 64 of 8000 51.2 54.5; 128 on eight, one of 20000 23.1 22.0, 40 of
// 600 25.5 21.7, 24 of 4000 43.4 44.3, in 8 bits 52.3 54.7).
#define PD_WIDE 640000
#define PD_SMEM (222 * 1024)       // dynamic shared memory: of 227 KB, with what a block has besides
#define PD_LOG2E 1.4426950408889634f
#define PD_NO_KEY (-3.0e38f)       // the running maximum before the first key: below every finite score

struct PackedDecode {
  const void* q;                   // bfloat16, or float32 (EXACT), as the result
  long long q_stride;
  const unsigned char* pages;
  int num_pages;
  const int* tables;
  int bt_stride;
  const int* cu_q_lens;
  const int* context_lens;
  const int* seqs;
  const int* q0;                   // EXACT, prompts: item i is rows q0[i] .. of sequence seqs[i], at most `fold` of them; else items are tokens
  int fold;
  int n, B;                        // items; sequences (rows of the tables): an item of none is padding
  void* out;
  int nh, nkv, group, chunks;      // heads of a kv head, in chunks of 8 NT
  int page_log2, page_bytes;
  int window;
  float scale, softcap;
  const float* sink;
  const float* slopes;
  float temp_coef, temp_every;
  float* part;                     // parts of pairs, [8 NT * D + 2 * 8 NT] each (outputs, then max and sum of each head): two of every block,
                                   // then one of every warp
  int4* cut;                       // of each block: what the second kernel joins (see there)
  int blocks, early;               // early: the lists are not the output of the kernel ahead
};

__device__ __forceinline__ void mma_f16(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (no volatile in these: the order of independent products and exponentials is the compiler's to choose)
__device__ __forceinline__ float exp2_near(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ unsigned half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
// x u and y u as halves.  EXACT: x and y become what is left of them, v = 1 / u; two such parts have every one of a float's 24 bits
// but the last (11 each, and the second one's sign).
template <bool EXACT> __device__ __forceinline__ unsigned half_parts(float& x, float& y, float u, float v) {
  const __half2 h = __floats2half2_rn(x * u, y * u);
  if (EXACT) {
    const float2 f = __half22float2(h);
    x = fmaf(-f.x, v, x);
    y = fmaf(-f.y, v, y);
  }
  return *reinterpret_cast<const unsigned*>(&h);
}
// Codes as halves, times 2^-24.  EXACT: as they are, less the middle code (8 or 128), so that sums of them are no larger than those of the
// values: 1024 + code first.  Not times 2^-24, since a tensor core lines products up by their operands' exponents: a small subnormal loses bits
// (of the float32 result of 4-bit codes it left 4e-6).  `center`: -(1024 + middle), of codes that stand where they are or count sixteenfold.
#define PD_LOW 0xe408e408u
#define PD_HIGH 0xe480e480u
template <bool EXACT> __device__ __forceinline__ unsigned codes(unsigned x, unsigned mask, unsigned center) {
  if (!EXACT) return x & mask;
  const unsigned v = (x & mask) | 0x64006400u;
  const __half2 h = __hadd2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&center));
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T> __device__ __forceinline__ T ld(const unsigned char* p) { return *reinterpret_cast<const T*>(p); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

// The sequence of token i, or -1.
__device__ __forceinline__ int sequence_of(const PackedDecode& a, int i) {
  const int b = a.seqs ? a.seqs[i] : i;
  return b < a.B ? b : -1;
}
// Tokens of sequence b that can be in sight: a context that its block table cannot hold is cut there.
__device__ __forceinline__ int context_of(const PackedDecode& a, int b) {
  const long long most = (long long)a.bt_stride << a.page_log2;
  return b >= 0 ? max(0, (int)min((long long)a.context_lens[b], most)) : 0;
}
// Its keys in sight are [first_key, context), counted in tiles from the tile of the first.  An item of w tokens has the context of
// its last one, and sees what its first one does.
__device__ __forceinline__ int first_key(const PackedDecode& a, int context) { return a.window > 0 ? max(0, context - a.window) : 0; }
struct Item { int tokens, row, context, first; };
template <bool EXACT> __device__ __forceinline__ Item item_of(const PackedDecode& a, int i, int b) {
  Item it = {1, 0, context_of(a, b), 0};
  if (b >= 0) {
    it.row = a.cu_q_lens ? a.cu_q_lens[b] : b;
    if (EXACT && a.q0) {
      const int q_len = a.cu_q_lens[b + 1] - it.row, q0 = a.q0[i];
      it.tokens = min(a.fold, q_len - q0);
      it.row += q0;
      it.context = max(0, it.context - q_len + q0 + it.tokens);
    }
  }
  it.first = first_key(a, max(0, it.context - it.tokens + 1));
  return it;
}
// what scan_tiles keeps of item i
template <bool EXACT> __device__ __forceinline__ int first_of(const PackedDecode& a, const int* contexts, int i) {
  return EXACT ? contexts[a.n + i] : first_key(a, contexts[i]);
}
// Pairs of a token are (kv head, chunk of its query heads), chunk by chunk.
__device__ __forceinline__ int kv_head(const PackedDecode& a, int pair) { return a.chunks == 1 ? pair : pair / a.chunks; }

// prefix[i] = tiles of the tokens before i (of all their pairs), contexts[i] = context of token i, for every block alike
template <int TILE, int THREADS, bool EXACT>
__device__ __forceinline__ void scan_tiles(const PackedDecode& a, int pairs, int* prefix, int* contexts, int* wsum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int i0 = 0; i0 < a.n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    int mine = 0;
    if (i < a.n) {
      const Item it = item_of<EXACT>(a, i, sequence_of(a, i));
      const int c = it.context, lo = it.first;
      contexts[i] = c;
      if (EXACT) contexts[a.n + i] = lo;
      mine = c > lo ? ((c + TILE - 1) / TILE - lo / TILE) * pairs : 0;
    }
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
// `total` tiles over `blocks` blocks: the first total % blocks have one more than the others.
struct BlockRanges {
  int each, more;
  __device__ __forceinline__ BlockRanges(int total, int blocks) : each((unsigned)total / (unsigned)blocks), more(total - each * blocks) {}
  __device__ __forceinline__ int start(int block) const { return block * each + min(block, more); }
  __device__ __forceinline__ int holder(int f) const {                // the block that has tile f
    const int edge = more * (each + 1);
    return f < edge ? (unsigned)f / (unsigned)(each + 1) : more + (unsigned)(f - edge) / (unsigned)each;
  }
};

// A place in the sequence of all tiles: tile f lies in pair `pair` of token i, whose tiles are [base, base + tiles).
template <int TILE, bool EXACT> struct TileCursor {
  int i, pair, base, tiles;
  __device__ __forceinline__ void settle(const PackedDecode& a, const int* contexts) {   // tiles of token i
    tiles = (int)((unsigned)(contexts[i] + TILE - 1) / TILE - (unsigned)first_of<EXACT>(a, contexts, i) / TILE);
  }
  // from all lanes of a warp, the same f
  __device__ __forceinline__ void start(const PackedDecode& a, const int* prefix, const int* contexts, int f) {
    int lo = 0, hi = a.n - 1;                     // the last token whose tiles start at f or before and that has any
    if (hi < 32) {
      const int lane = threadIdx.x & 31;
      lo = 31 - __clz(__ballot_sync(0xffffffffu, lane <= hi && prefix[min(lane, hi)] <= f));
    } else {
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (prefix[m] <= f) lo = m; else hi = m - 1;
      }
    }
    i = lo;
    settle(a, contexts);
    const int rest = f - prefix[i];
    pair = (int)__fdividef((float)rest, (float)tiles);      // a small number: off by one at most
    if (pair * tiles > rest) --pair;
    if ((pair + 1) * tiles <= rest) ++pair;
    base = prefix[i] + pair * tiles;
  }
  __device__ __forceinline__ void advance(const PackedDecode& a, const int* contexts, int pairs, int f) {   // f < prefix[n]
    while (f >= base + tiles) {
      base += tiles;
      if (++pair == pairs) {
        pair = 0;
        do { ++i; settle(a, contexts); } while (tiles <= 0);
      }
    }
  }
};

// Shapes of the kernel: warps of a block (16 at 128 registers a thread, or 8), keys of a tile, stages of a ring.  Twice the heads
// take twice the registers, so half the warps (PD_WIDE); a tile is about the same bytes in 4 and in 8 bits; as many stages as shared
// memory holds beside the lists of the most tokens.
template <int D, int BITS, int NT, bool EXACT> struct PdSizes {
  static constexpr int WARPS = EXACT ? PD_EXACT_WARPS : NT == 1 ? 16 : 8, TILE = BITS == 4 ? 32 : 16, THREADS = WARPS * 32;
  static constexpr int GR = D / 64, ROW = D * BITS / 8, HEADS = 8 * NT, PART = HEADS * D + 2 * HEADS;      // PART in floats
  static constexpr int STAGE = 2 * TILE * (ROW + 4 * GR);
  static constexpr int bytes(int stages) { return WARPS * stages * (STAGE + 4) + ((EXACT ? 3 : 2) * PD_MAX_TOKENS + 1) * 4; }
  static constexpr int most(int stages) { return stages < 8 && bytes(stages + 1) <= PD_SMEM ? most(stages + 1) : stages; }
  static constexpr int STAGES = most(2), SMEM = bytes(most(2));
};

// Where column h of the kernel's results stands in the result, counted in rows of D from the item's first: of the next token after `fold` heads.
template <bool EXACT> __device__ __forceinline__ int token_of(const PackedDecode& a, int h) { return EXACT && a.fold > 1 ? h / a.group : 0; }
template <bool EXACT> __device__ __forceinline__ int head_of(const PackedDecode& a, int h) { return EXACT && a.fold > 1 ? h % a.group : h; }
template <bool EXACT> __device__ __forceinline__ int place_of(const PackedDecode& a, int h) { return token_of<EXACT>(a, h) * a.nh + head_of<EXACT>(a, h); }
// Four values of the result.
template <bool EXACT> __device__ __forceinline__ void put4(const PackedDecode& a, size_t at, float x, float y, float z, float w) {
  if (EXACT) *reinterpret_cast<float4*>((float*)a.out + at) = make_float4(x, y, z, w);
  else *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + at) = make_uint2(pack_bf16(x, y), pack_bf16(z, w));
}

template <int D, int BITS, int NT, bool OPT, bool EXACT>
__global__ void __launch_bounds__(PdSizes<D, BITS, NT, EXACT>::THREADS, 1) packed_decode_kernel(PackedDecode a) {
  typedef PdSizes<D, BITS, NT, EXACT> Z;
  constexpr int PARTS = EXACT ? 2 : 1;             // halves that a query or weight is held in
  constexpr float MIDDLE = BITS == 4 ? 8.f : 128.f;
  constexpr int GR = Z::GR, ROW = Z::ROW, HEADS = Z::HEADS, STAGE = Z::STAGE, TILE = Z::TILE, WARPS = Z::WARPS, KB = TILE / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int wsum[WARPS];
  // a warp's two parts: which pair (its first tile) they belong to, or -1; maximum and sum of each head; weight in the joined pair
  __shared__ int part_base[2 * WARPS];
  __shared__ int4 part_pair[2 * WARPS];            // tiles and heads of that pair, its first row of the result
  __shared__ float part_top[2 * WARPS][HEADS], part_sum[2 * WARPS][HEADS], part_weight[2 * WARPS][HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int pairs = a.nkv * a.chunks;
  constexpr int S = Z::STAGES;
  // shared memory: a ring per warp, the chunks of a stage that are there, prefix, contexts
  unsigned* here = reinterpret_cast<unsigned*>(smem + (size_t)WARPS * S * STAGE) + warp * S;
  int* prefix = reinterpret_cast<int*>(smem + (size_t)WARPS * S * STAGE) + WARPS * S;
  int* contexts = prefix + a.n + 1;
  float* parts = a.part + ((size_t)2 * a.blocks + (size_t)blockIdx.x * WARPS) * Z::PART;
  const unsigned ring = smem_u32(smem) + warp * S * STAGE;
  if (tid < 2 * WARPS) part_base[tid] = -1;
  pdl_trigger();
  if (!a.early) pdl_wait();
  scan_tiles<TILE, Z::THREADS, EXACT>(a, pairs, prefix, contexts, wsum);
  const int total = prefix[a.n];
  auto zeros = [&]() {                             // tokens without a key in sight, spread over the blocks
    for (int i = blockIdx.x; i < a.n; i += a.blocks) {
      const int b = sequence_of(a, i);
      if (contexts[i] > 0 || b < 0) continue;
      const Item it = item_of<EXACT>(a, i, b);
      for (int e = tid * 4; e < it.tokens * a.nh * D; e += Z::THREADS * 4) put4<EXACT>(a, (size_t)it.row * a.nh * D + e, 0.f, 0.f, 0.f, 0.f);
    }
  };
  const int blocks = min(a.blocks, total);         // each has a tile at least
  if ((int)blockIdx.x >= blocks) {
    if (a.early) pdl_wait();
    if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    zeros();
    return;
  }
  const BlockRanges ranges(total, blocks);
  const int b_lo = ranges.start(blockIdx.x), b_hi = ranges.start(blockIdx.x + 1);

  // chunks: the tokens of a tile that lie in one page
  const int chunk = a.page_log2 == 4 ? 16 : TILE, chunks = TILE / chunk, two = chunks >> 1;      // two: log2 of chunks
  const int chunk_bytes = 2 * chunk * (ROW + 4 * GR);
  const int w_lo = b_lo + (b_hi - b_lo) * warp / WARPS, w_hi = b_lo + (b_hi - b_lo) * (warp + 1) / WARPS;

  // ---- the ring.  Lane j knows chunk j of the tiles [batch, batch + 32 / chunks): its page, kv head and place in the page;
  // the ones of the batch that follows are being looked up.
  int batch = w_lo, f_ask = w_lo, id = -1, id_next = -1, spot = 0, spot_next = 0;
  unsigned there = 0;
  TileCursor<TILE, EXACT> at;                             // of the first tile that was looked up last
  auto look_up = [&](int from) {
    id_next = -1;
    if (from >= w_hi) return;
    at.start(a, prefix, contexts, from);
    const int f = from + (lane >> two);
    if (f >= w_hi) return;
    TileCursor<TILE, EXACT> mine = at;
    mine.advance(a, contexts, pairs, f);
    const int ctx = contexts[mine.i], b = a.seqs ? a.seqs[mine.i] : mine.i;
    const int key = first_of<EXACT>(a, contexts, mine.i) / TILE * TILE + (f - mine.base) * TILE + (lane & (chunks - 1)) * chunk;
    if (key < ctx) id_next = a.tables[(size_t)b * a.bt_stride + (key >> a.page_log2)];
    spot_next = kv_head(a, mine.pair) << 8 | (key & ((1 << a.page_log2) - 1));
  };
  auto ask = [&](int stage) {                      // start the copies of tile f_ask; a group of copies whether there is one or not
    if (f_ask < w_hi) {
      if (f_ask == batch + (32 >> two) || f_ask == w_lo) {
        batch = f_ask;
        id = id_next;
        spot = spot_next;
        there = __ballot_sync(0xffffffffu, id >= 0 && id < a.num_pages);
      }
      const int k = f_ask - batch;
      if (k == S) look_up(batch + (32 >> two));    // not before the first stages are on their way
      const unsigned mask = (there >> (k << two)) & ((1u << chunks) - 1);
      const int spot_k = __shfl_sync(0xffffffffu, spot, k << two);
      const unsigned char* head = a.pages + (size_t)(spot_k >> 8) * a.page_bytes;
      const size_t page = (size_t)a.nkv * a.page_bytes;
      if (lane == 0) here[stage] = mask;
      const unsigned dst = ring + stage * STAGE + lane * 16;
      if (a.page_log2 == 4) {                      // a chunk is a whole block
        constexpr int BYTES = 32 * (ROW + 4 * GR);
#pragma unroll
        for (int c = 0; c < TILE / 16; ++c) {
          const int there_c = (mask >> c) & 1 ? 16 : 0;
          const int id_c = __shfl_sync(0xffffffffu, id, (k << two) + c);
          const unsigned char* src = head + (there_c ? id_c * page : 0) + lane * 16;
#pragma unroll
          for (int u = 0; u < BYTES; u += 512)
            if (u + 512 <= BYTES || lane * 16 < BYTES - u) cp_async16(dst + c * BYTES + u, src + u, there_c);
        }
      } else {                                     // codes and pairs of TILE tokens, each apart in the block
        const int place = spot_k & 255, P = 1 << a.page_log2;
        const unsigned char* block = head + (mask ? __shfl_sync(0xffffffffu, id, k << two) * page : 0);
        constexpr int CODES = TILE * ROW, PAIRS = TILE * GR * 4;
        for (int u = lane * 16; u < STAGE; u += 512) {
          const int from = u < CODES ? place * ROW + u : u < 2 * CODES ? (P + place) * ROW + u - CODES
                           : u < 2 * CODES + PAIRS ? 2 * P * ROW + place * GR * 4 + u - 2 * CODES
                                                   : 2 * P * ROW + (P + place) * GR * 4 + u - 2 * CODES - PAIRS;
          cp_async16(dst + u - lane * 16, block + from, mask ? 16 : 0);
        }
      }
      ++f_ask;
    }
    cp_async_commit();
  };
  look_up(w_lo);
  if (a.early) pdl_wait();
  TileCursor<TILE, EXACT> now = at;                       // the pair the warp is at
  if (!EXACT && w_lo < w_hi) {
    const int b = a.seqs ? a.seqs[at.i] : at.i, row = a.cu_q_lens ? a.cu_q_lens[b] : b;
    const int kvh = kv_head(a, at.pair), head = kvh * a.group + (at.pair - kvh * a.chunks) * HEADS;
    // the queries are on their way while the first pages are looked up: 64 bytes a lane
    if (lane < min(HEADS, a.nh - head) * D / 32)
      asm volatile("prefetch.global.L1 [%0];" ::"l"((const __nv_bfloat16*)a.q + (size_t)row * a.q_stride + (size_t)head * D + lane * 32));
  }
#pragma unroll 1
  for (int s = 0; s < S; ++s) ask(s);
  if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
  zeros();

  // ---- the pairs of the warp's range, one after the other
  const int key_g = (g >> 1) + 4 * (g & 1);       // the key (of 16) in row g of the scores; row g + 8 has key_g + 8
  const int step_c = chunk == 16 ? chunk_bytes : 16 * ROW, step_p = chunk == 16 ? chunk_bytes : 16 * GR * 4;   // from 16 keys to the next
  const unsigned off_k = key_g * ROW + t * (2 * BITS);                     // a lane's 16 channels of its key
  const unsigned off_v = chunk * ROW + t * ROW + g * BITS;                 // its 8 channels of keys t, t + 4, t + 8, t + 12
  const unsigned off_kp = 2 * chunk * ROW + key_g * GR * 4, off_vp = off_kp + chunk * GR * 4;
  int stage = 0, f = w_lo;
  while (f < w_hi) {
    now.advance(a, contexts, pairs, f);
    const int seg = f, seg_end = min(now.base + now.tiles, w_hi);
    const int b = a.seqs ? a.seqs[now.i] : now.i, ctx = contexts[now.i], lo = first_of<EXACT>(a, contexts, now.i);
    const Item it = item_of<EXACT>(a, now.i, b);
    const int tile0 = lo / TILE * TILE;
    const int kvh = kv_head(a, now.pair), head0 = (now.pair - kvh * a.chunks) * HEADS;
    const int row = it.row, heads = EXACT && a.fold > 1 ? it.tokens * a.group : min(HEADS, a.group - head0);      // columns
    int ends[NT][2];                               // the contexts of this lane's columns
    if (EXACT)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) ends[nt][j] = ctx - it.tokens + 1 + min(it.tokens - 1, token_of<EXACT>(a, nt * 8 + 2 * t + j));

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
    float unit[NT][2], one[NT][2];                 // a head's scores and maxima are held in units of `unit`
    // weights of a head are held times a power of two, `inv`: 2^2 over the largest p s' when it was last set.  Columns without a head have one
    // that nothing exceeds.
    float inv[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) inv[nt][j] = nt * 8 + 2 * t + j < heads ? 0x1p106f : 0x1p-121f;

    {
      // ---- q of this pair: B operands, and its sums over each group
      unsigned qf[PARTS][GR][4][NT][2];
      float qsum[GR][NT][2];
      {
        constexpr int CODE = EXACT ? 0 : 24;       // a code is an operand times 2^-CODE
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bool mine = nt * 8 + g < heads;
          const int col = mine ? nt * 8 + g : 0, tok = token_of<EXACT>(a, col);
          const float held = (float)(ctx - it.tokens + 1 + tok);
          const float temp = OPT && a.temp_every > 0.f ? 1.f + a.temp_coef * logf(floorf(__fdiv_rn(held, a.temp_every)) + 1.f) : 1.f;
          const float fac = a.scale * temp * (OPT ? 1.f : PD_LOG2E), size = fmaxf(fabsf(fac), 1e-30f);
          const size_t q_at = (size_t)(row + tok) * a.q_stride + (size_t)(kvh * a.group + head0 + head_of<EXACT>(a, col)) * D + t * 16;
          float x[GR][16], sum[GR], big = 0.f;
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
#pragma unroll
            for (int v = 0; v < (EXACT ? 4 : 2); ++v) {
              const uint4 u = !mine ? make_uint4(0, 0, 0, 0) : EXACT ? *reinterpret_cast<const uint4*>((const float*)a.q + q_at + gr * 64 + v * 4)
                                    : *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + q_at + gr * 64 + v * 8);
              const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (EXACT) {
                  x[gr][(v * 4 + i) & 15] = __uint_as_float(w[i]);
                } else {
                  x[gr][(v * 8 + 2 * i) & 15] = __uint_as_float(w[i] << 16);
                  x[gr][(v * 8 + 2 * i + 1) & 15] = __uint_as_float(w[i] & 0xffff0000u);
                }
              }
            }
            sum[gr] = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              sum[gr] += x[gr][i];
              big = fmaxf(big, fabsf(x[gr][i]));
            }
            sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
            sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
            if (!(sum[gr] - sum[gr] == 0.f)) sum[gr] = __int_as_float(0x7fffffff);       // an infinity or NaN in q: NaN scores
          }
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          const int e = max(-90, min(100, 139 - (int)(__float_as_uint(big) >> 23)));   // big * 2^e lies in [2^12, 2^13)
          const float up = copysignf(power_of_two(e), fac), down = copysignf(power_of_two(e - CODE), fac), mul = fmaxf(size * power_of_two(CODE - e), 1e-37f);
#pragma unroll
          for (int j = 0; j < 2; ++j) {            // of the heads whose scores this lane will hold
            unit[nt][j] = __shfl_sync(0xffffffffu, mul, 8 * t + 4 * j);
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) qsum[gr][nt][j] = __shfl_sync(0xffffffffu, sum[gr] * down, 8 * t + 4 * j);
          }
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            float* y = x[gr];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] *= up;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                if (BITS == 4) {                   // m = 2 * word + (codes four bits up)
                  const int c = 8 * (m >> 1) + (m & 1);
                  const float u = m & 1 ? 0.0625f : 1.f, v = m & 1 ? 16.f : 1.f;
                  qf[part][gr][m][nt][0] = half_parts<EXACT>(y[c], y[c + 4], u, v);
                  qf[part][gr][m][nt][1] = half_parts<EXACT>(y[c + 2], y[c + 6], u, v);
                } else {
                  qf[part][gr][m][nt][0] = half_parts<EXACT>(y[4 * m], y[4 * m + 2], 1.f, 1.f);
                  qf[part][gr][m][nt][1] = half_parts<EXACT>(y[4 * m + 1], y[4 * m + 3], 1.f, 1.f);
                }
              }
            }
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
            slope[nt][j] = a.slopes && h < heads ? a.slopes[kvh * a.group + head0 + head_of<EXACT>(a, h)] : 0.f;
          }
      }

      if (OPT) {                                   // options are applied to scores as they are
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) one[nt][0] = one[nt][1] = 1.f;
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) { one[nt][0] = unit[nt][0]; one[nt][1] = unit[nt][1]; }
      }

      for (; f < seg_end; ++f) {
        cp_async_wait<S - 1>();
        __syncwarp();                              // every lane's copies of this stage are there
        {
          const unsigned char* base = smem + (size_t)(warp * S + stage) * STAGE;
          const int key0 = tile0 + (f - now.base) * TILE;
          const unsigned mask = here[stage];
          const bool whole = key0 >= (EXACT ? first_key(a, ctx) : lo) && key0 + TILE <= (EXACT ? ctx - it.tokens + 1 : ctx) && mask == (1u << chunks) - 1;
          // ---- scores
          float s[KB][NT][4];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[kb][nt][0] = s[kb][nt][1] = s[kb][nt][2] = s[kb][nt][3] = 0.f;
            unsigned kp[2][GR];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const unsigned char* p = base + off_kp + kb * step_p + half * 8 * GR * 4;
              if (GR == 2) {
                const uint2 u = ld<uint2>(p);
                kp[half][0] = u.x;
                kp[half][GR - 1] = u.y;
              } else {
                kp[half][0] = ld<unsigned>(p);
              }
            }
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
              float acc[NT][4];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
              const unsigned char* kc = base + off_k + kb * step_c + gr * (8 * BITS);
              unsigned x[4][4];
              if (BITS == 4) {
                const uint2 ua = ld<uint2>(kc), ub = ld<uint2>(kc + 8 * ROW);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  const unsigned wa = w ? ua.y : ua.x, wb = w ? ub.y : ub.x, xa = wa >> 8, xb = wb >> 8;
                  x[2 * w][0] = codes<EXACT>(wa, 0x000f000fu, PD_LOW);
                  x[2 * w][1] = codes<EXACT>(wb, 0x000f000fu, PD_LOW);
                  x[2 * w][2] = codes<EXACT>(xa, 0x000f000fu, PD_LOW);
                  x[2 * w][3] = codes<EXACT>(xb, 0x000f000fu, PD_LOW);
                  x[2 * w + 1][0] = codes<EXACT>(wa, 0x00f000f0u, PD_HIGH);
                  x[2 * w + 1][1] = codes<EXACT>(wb, 0x00f000f0u, PD_HIGH);
                  x[2 * w + 1][2] = codes<EXACT>(xa, 0x00f000f0u, PD_HIGH);
                  x[2 * w + 1][3] = codes<EXACT>(xb, 0x00f000f0u, PD_HIGH);
                }
              } else {
                const uint4 ua = ld<uint4>(kc), ub = ld<uint4>(kc + 8 * ROW);
                const unsigned wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  x[w][0] = codes<EXACT>(wa[w], 0x00ff00ffu, PD_HIGH);
                  x[w][1] = codes<EXACT>(wb[w], 0x00ff00ffu, PD_HIGH);
                  x[w][2] = codes<EXACT>(wa[w] >> 8, 0x00ff00ffu, PD_HIGH);
                  x[w][3] = codes<EXACT>(wb[w] >> 8, 0x00ff00ffu, PD_HIGH);
                }
              }
              // (small parts first: a tensor core may truncate where it adds)
#pragma unroll
              for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma_f16(acc[nt], x[w][0], x[w][1], x[w][2], x[w][3], qf[part][gr][w][nt][0], qf[part][gr][w][nt][1]);
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float sc = __uint_as_float(kp[half][gr] << 16);
                float of = __uint_as_float(kp[half][gr] & 0xffff0000u);
                if (EXACT) of = fmaf(MIDDLE, sc, of);
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
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float v = s[kb][nt][i] * unit[nt][i & 1];
                  if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
                  v -= slope[nt][i & 1] * (float)((EXACT ? ends[nt][i & 1] : ctx) - 1 - (key0 + 16 * kb + 8 * (i >> 1) + key_g));
                  s[kb][nt][i] = v * PD_LOG2E;
                }
          }
          // pairs of the values, and what is out of sight
          float sv[KB][2][GR], ov[KB][2][GR];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              unsigned u[GR];
              const unsigned char* p = base + off_vp + kb * step_p + half * 8 * GR * 4;
              if (GR == 2) {
                const uint2 w = ld<uint2>(p);
                u[0] = w.x;
                u[GR - 1] = w.y;
              } else {
                u[0] = ld<unsigned>(p);
              }
#pragma unroll
              for (int gr = 0; gr < GR; ++gr) {
                sv[kb][half][gr] = __uint_as_float(u[gr] << 16);
                ov[kb][half][gr] = __uint_as_float(u[gr] & 0xffff0000u);
                if (EXACT) ov[kb][half][gr] = fmaf(MIDDLE, sv[kb][half][gr], ov[kb][half][gr]);
              }
            }
          unsigned hide = 0;                       // EXACT: scores that some of the columns do not see, whose value may be a NaN
          if (!whole) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int key = key0 + 16 * kb + 8 * half + key_g;
                if (key < lo || key >= ctx || !((mask >> (chunk == 16 ? kb : 0)) & 1)) {
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) s[kb][nt][2 * half] = s[kb][nt][2 * half + 1] = -INFINITY;
#pragma unroll
                  for (int gr = 0; gr < GR; ++gr) sv[kb][half][gr] = ov[kb][half][gr] = 0.f;
                } else if (EXACT) {
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                      if (key >= ends[nt][j] || key < first_key(a, ends[nt][j])) {
                        s[kb][nt][2 * half + j] = -INFINITY;
                        hide |= 1u << ((kb * NT + nt) * 4 + 2 * half + j);
                      }
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
              mx[nt][j] = fmaxf(s[0][nt][j], s[0][nt][2 + j]);
              if (KB == 2) mx[nt][j] = fmaxf(mx[nt][j], fmaxf(s[KB - 1][nt][j], s[KB - 1][nt][2 + j]));
              over = over || (mx[nt][j] - ref[nt][j]) * one[nt][j] > 8.f;
            }
          float smax = 0.f;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) smax = fmaxf(smax, fmaxf(sv[kb][0][gr], sv[kb][1][gr]));
          if (__any_sync(0xffffffffu, over)) {
            const int loudest = (int)(__float_as_uint(warp_max(smax)) >> 23);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float m = mx[nt][j];
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                m = fmaxf(m, ref[nt][j]);
                const float al = exp2_near((ref[nt][j] - m) * one[nt][j]);
                ref[nt][j] = m;
                l[nt][j] *= al;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) r[gr][nt][j] *= al;
                // what the output had is that much smaller, so the weights' power of two may grow by as much: up to 2^2 over the largest s'
                const int has = (int)(__float_as_uint(inv[nt][j]) >> 23), shrunk = 127 - (int)(__float_as_uint(al) >> 23);
                const float more = power_of_two(max(0, min(min(120, shrunk), min(233 - has, 255 - loudest - has))));
                inv[nt][j] *= more;
#pragma unroll
                for (int i = 0; i < GR * 4; ++i) { o[i][nt][j] *= al * more; o[i][nt][2 + j] *= al * more; }
              }
          }
          float base2[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) base2[nt][j] = fmaxf(ref[nt][j] * one[nt][j], PD_NO_KEY);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const float p = exp2_near(fmaf(s[kb][nt][2 * half + j], one[nt][j], -base2[nt][j]));
                  s[kb][nt][2 * half + j] = p;           // (times inv where the products are made)
                  l[nt][j] += p;
#pragma unroll
                  for (int gr = 0; gr < GR; ++gr) {
                    const float of = EXACT && (hide >> ((kb * NT + nt) * 4 + 2 * half + j)) & 1 ? 0.f : ov[kb][half][gr];
                    r[gr][nt][j] = fmaf(p, of, r[gr][nt][j]);
                  }
                }
            }
          // ---- the weights' powers of two: p s' inv stays below 2^15 (p is below 2^8)
          float most = inv[0][0];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) most = fmaxf(most, fmaxf(inv[nt][0], inv[nt][1]));
          if (__any_sync(0xffffffffu, smax * most > 128.f)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float w = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                  for (int half = 0; half < 2; ++half) {
                    float z = 0.f;
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) z = fmaxf(z, sv[kb][half][gr]);
                    w = fmaxf(w, s[kb][nt][2 * half + j] * z);
                  }
                w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 4));
                w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 8));
                w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 16));
                if (nt * 8 + 2 * t + j < heads && w * inv[nt][j] > 64.f) {
                  const float next = power_of_two(2 - min(123, (int)(__float_as_uint(w) >> 23) - 127)), down = next / inv[nt][j];
                  inv[nt][j] = next;
#pragma unroll
                  for (int i = 0; i < GR * 4; ++i) { o[i][nt][j] *= down; o[i][nt][2 + j] *= down; }
                }
              }
          }
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) s[kb][nt][i] *= inv[nt][i & 1];
          // ---- output: channels x heads
          // (EXACT: a tile's sums are made apart)
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            float tile_o[4][NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) tile_o[i][nt][j] = EXACT ? 0.f : o[gr * 4 + i][nt][j];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              unsigned pb[PARTS][NT][2];
              const float w0 = sv[kb][0][gr], w1 = sv[kb][1][gr];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  y[i] = EXACT && (hide >> ((kb * NT + nt) * 4 + i)) & 1 ? 0.f : s[kb][nt][i] * (i < 2 ? w0 : w1);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                  pb[part][nt][0] = transpose8(half_parts<EXACT>(y[0], y[1], 1.f, 1.f));
                  pb[part][nt][1] = transpose8(half_parts<EXACT>(y[2], y[3], 1.f, 1.f));
                }
              }
              const unsigned char* vc = base + off_v + kb * step_c + gr * (8 * BITS);
              unsigned a4[4][4];                   // operands of channels 2 i and 2 i + 1 of the lane's eight
              if (BITS == 4) {
                const unsigned w0 = ld<unsigned>(vc), w1 = ld<unsigned>(vc + 4 * ROW), w2 = ld<unsigned>(vc + 8 * ROW), w3 = ld<unsigned>(vc + 12 * ROW);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  const unsigned sel = v & 2 ? 0x7632 : 0x5410;
                  const unsigned x = __byte_perm(w0, w1, sel) >> (v & 1 ? 8 : 0), y = __byte_perm(w2, w3, sel) >> (v & 1 ? 8 : 0);
                  a4[v][0] = codes<EXACT>(x, 0x000f000fu, PD_LOW);
                  a4[v][1] = codes<EXACT>(x, 0x00f000f0u, PD_HIGH);
                  a4[v][2] = codes<EXACT>(y, 0x000f000fu, PD_LOW);
                  a4[v][3] = codes<EXACT>(y, 0x00f000f0u, PD_HIGH);
                }
              } else {
                const uint2 w0 = ld<uint2>(vc), w1 = ld<uint2>(vc + 4 * ROW), w2 = ld<uint2>(vc + 8 * ROW), w3 = ld<uint2>(vc + 12 * ROW);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  const unsigned sel = v & 1 ? 0x7632 : 0x5410;
                  const unsigned x = v < 2 ? __byte_perm(w0.x, w1.x, sel) : __byte_perm(w0.y, w1.y, sel);
                  const unsigned y = v < 2 ? __byte_perm(w2.x, w3.x, sel) : __byte_perm(w2.y, w3.y, sel);
                  a4[v][0] = codes<EXACT>(x, 0x00ff00ffu, PD_HIGH);
                  a4[v][1] = codes<EXACT>(x >> 8, 0x00ff00ffu, PD_HIGH);
                  a4[v][2] = codes<EXACT>(y, 0x00ff00ffu, PD_HIGH);
                  a4[v][3] = codes<EXACT>(y >> 8, 0x00ff00ffu, PD_HIGH);
                }
              }
#pragma unroll
              for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int part = PARTS - 1; part >= 0; --part)
                    mma_f16(tile_o[v][nt], a4[v][0], a4[v][1], a4[v][2], a4[v][3], pb[part][nt][0], pb[part][nt][1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[gr * 4 + i][nt][j] = EXACT ? o[gr * 4 + i][nt][j] + tile_o[i][nt][j] : tile_o[i][nt][j];
          }
        }
        __syncwarp();                              // every lane has read the stage
        ask(stage);
        if (++stage == S) stage = 0;
      }
    }

    // ---- the pair's result, or this warp's part of it (maxima as powers of two from here)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) ref[nt][j] = fmaxf(ref[nt][j] * one[nt][j], PD_NO_KEY);
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
    const bool complete = seg == now.base && seg_end == now.base + now.tiles;
    // the last part of the range goes where the ring was (all its copies have arrived and been read), the first to the scratch
    const bool last = seg_end == w_hi;
    float* part = last ? reinterpret_cast<float*>(smem + (size_t)warp * S * STAGE) : parts + warp * Z::PART;
    if (!complete && lane == 0) {
      part_base[2 * warp + last] = now.base;
      part_pair[2 * warp + last] = make_int4(now.tiles, heads, row * a.nh + kvh * a.group + head0, 0);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = nt * 8 + 2 * t + j;
        float fac = 1.f;
        if (complete) {
          float sum = l[nt][j];
          if (OPT && a.sink && h < heads) {
            const float sk = a.sink[kvh * a.group + head0 + head_of<EXACT>(a, h)] * PD_LOG2E, top = fmaxf(ref[nt][j], sk);
            fac = exp2_near(ref[nt][j] - top);
            sum = sum * fac + exp2_near(sk - top);
          }
          fac = sum != 0.f ? fac / sum : 0.f;
        } else if (g == 0) {
          part_top[2 * warp + last][h] = ref[nt][j];
          part_sum[2 * warp + last][h] = l[nt][j];
        }
        // codes stood at 2^-24 or, EXACT, 1 (in 4 bits every second one at 16 times that), weights at inv
        const float even = 0x1p2f / inv[nt][j] * fac, up = EXACT ? 0x1p-2f : 0x1p22f, odd = BITS == 4 ? up * 0.0625f : up;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
          const float off = r[gr][nt][j] * fac;
          float y[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = fmaf(o[gr * 4 + i][nt][j] * up, even, off);
            y[2 * i + 1] = fmaf(o[gr * 4 + i][nt][2 + j] * odd, even, off);
          }
          const int c = gr * 64 + g * 8;
          if (!complete) {
            float4* p = reinterpret_cast<float4*>(part + h * D + c);
            p[0] = make_float4(y[0], y[1], y[2], y[3]);
            p[1] = make_float4(y[4], y[5], y[6], y[7]);
          } else if (h < heads) {
            const size_t to = ((size_t)row * a.nh + kvh * a.group + head0 + place_of<EXACT>(a, h)) * D + c;
            if (EXACT) {
              put4<EXACT>(a, to, y[0], y[1], y[2], y[3]);
              put4<EXACT>(a, to + 4, y[4], y[5], y[6], y[7]);
            } else {
              const uint4 u = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
              *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + to) = u;
            }
          }
        }
      }
  }
  // ---- the parts of one pair become the result, or this block's part of the pair
  __syncthreads();
  const int lane_base = lane < 2 * WARPS ? part_base[lane] : -1;
  const unsigned same = __match_any_sync(0xffffffffu, lane_base);           // the parts of the same pair
  unsigned leaders = __ballot_sync(0xffffffffu, lane_base >= 0 && (same & ((1u << lane) - 1)) == 0);
  if (!leaders) return;
  // lane i of the warps takes part i; a pair's parts lie between its first one and the next pair's
  const int from = max(0, 31 - __clz(leaders & ((2u << lane) - 1)));
  const unsigned beyond = lane == 31 ? 0u : leaders >> (lane + 1);
  const int to = beyond ? lane + __ffs(beyond) - 1 : 31;
  for (int h = warp; h < HEADS; h += WARPS) {
    const bool real = lane_base >= 0;
    float top = real ? part_top[lane][h] : PD_NO_KEY;
    const float mine = top;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, top, o);
      if (lane - o >= from) top = fmaxf(top, v);
    }
    const float M = __shfl_sync(0xffffffffu, top, to);
    float w = real ? exp2_near(mine - M) : 0.f, L = real ? part_sum[lane][h] * w : 0.f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, L, o);
      if (lane - o >= from) L += v;
    }
    L = __shfl_sync(0xffffffffu, L, to);
    if (!real) continue;
    const int4 pair = part_pair[lane];
    if (lane_base >= b_lo && lane_base + pair.x <= b_hi) {        // the weight in the result
      if (OPT && a.sink && h < pair.y) {
        const float sk = a.sink[pair.z % a.nh + head_of<EXACT>(a, h)] * PD_LOG2E, all = fmaxf(M, sk), u = exp2_near(M - all);
        w *= u;
        L = L * u + exp2_near(sk - all);
      }
      w = L != 0.f ? w / L : 0.f;
    } else if (lane == from) {
      float* out = a.part + (size_t)(2 * blockIdx.x + (lane_base < b_lo ? 0 : 1)) * Z::PART;
      out[HEADS * D + 2 * h] = M;
      out[HEADS * D + 2 * h + 1] = L;
      // a pair that began in an earlier block and ends here is joined from there to here
      if (h == 0 && lane_base < b_lo && lane_base + pair.x <= b_hi)
        a.cut[blockIdx.x] = make_int4(ranges.holder(lane_base), pair.y, pair.z, 0);
    }
    part_weight[lane][h] = w;
  }
  __syncthreads();
  // four values a thread: pairs side by side, PART / 4 threads each
  constexpr int QUADS = HEADS * D / 4;
  const int runs = __popc(leaders);
  for (int e = tid; e < runs * QUADS; e += Z::THREADS) {                    // (whole warps: QUADS is a multiple of 32)
    const int run = e / QUADS, x = (e % QUADS) * 4, h = x / D;
    unsigned rest = leaders;
    for (int i = 0; i < run; ++i) rest &= rest - 1;
    const int k = __ffs(rest) - 1;
    const unsigned members = __shfl_sync(0xffffffffu, same, k);
    const int4 pair = part_pair[k];
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    const int end = 32 - __clz(members);
#pragma unroll 4
    for (int i = k | 1; i < end; i += 2) {         // last parts, in shared memory
      const bool in = (members >> i) & 1;
      const float4 v = in ? *reinterpret_cast<const float4*>(smem + (size_t)(i >> 1) * S * STAGE + x * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float w = in ? part_weight[i][h] : 0.f;
      y.x = fmaf(w, v.x, y.x); y.y = fmaf(w, v.y, y.y); y.z = fmaf(w, v.z, y.z); y.w = fmaf(w, v.w, y.w);
    }
    for (unsigned m = members & 0x55555555u; m; m &= m - 1) {               // first parts (a pair has one in the block, or two)
      const int i = __ffs(m) - 1;
      const float4 v = *reinterpret_cast<const float4*>(parts + (i >> 1) * Z::PART + x);
      const float w = part_weight[i][h];
      y.x = fmaf(w, v.x, y.x); y.y = fmaf(w, v.y, y.y); y.z = fmaf(w, v.z, y.z); y.w = fmaf(w, v.w, y.w);
    }
    if (part_base[k] >= b_lo && part_base[k] + pair.x <= b_hi) {
      if (h < pair.y) put4<EXACT>(a, ((size_t)pair.z + place_of<EXACT>(a, h)) * D + x % D, y.x, y.y, y.z, y.w);
    } else {
      *reinterpret_cast<float4*>(a.part + (size_t)(2 * blockIdx.x + (part_base[k] < b_lo ? 0 : 1)) * Z::PART + x) = y;
    }
  }
}

// Joins the pairs that were cut between blocks.  A block of threads for each block of the first kernel and head: where a pair
// from an earlier block ends in it, cut[c] = (block of the pair's first tile, heads, first row of the result); that block has
// its part second, the ones after it first.  Every 32 or 16 threads take some of the parts, four values each.
template <int D, int NT, bool EXACT>
__global__ void __launch_bounds__(256) packed_join_kernel(PackedDecode a) {
  constexpr int HEADS = 8 * NT, PART = HEADS * D + 2 * HEADS, LANES = D / 4, SETS = 256 / LANES;
  __shared__ float2 ml_s[SETS];
  __shared__ float4 y_s[SETS][LANES];
  pdl_trigger();
  pdl_wait();
  const int last = blockIdx.x, h = blockIdx.y, set = threadIdx.x / LANES, e = threadIdx.x % LANES;
  const int4 cut = a.cut[last];
  const int first = cut.x;
  if (first < 0 || h >= cut.y) return;
  float M = PD_NO_KEY, L = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = first + set; c <= last; c += SETS) {
    const float* p = a.part + (size_t)(2 * c + (c == first ? 1 : 0)) * PART;
    const float2 ml = *reinterpret_cast<const float2*>(p + HEADS * D + 2 * h);
    const float4 v = reinterpret_cast<const float4*>(p + h * D)[e];
    const float top = fmaxf(M, ml.x), u = exp2_near(M - top), w = exp2_near(ml.x - top);
    L = L * u + w * ml.y;
    y.x = fmaf(w, v.x, u * y.x); y.y = fmaf(w, v.y, u * y.y); y.z = fmaf(w, v.z, u * y.z); y.w = fmaf(w, v.w, u * y.w);
    M = top;
  }
  if (e == 0) ml_s[set] = make_float2(M, L);
  y_s[set][e] = y;
  __syncthreads();
  if (set) return;
  const float sk = a.sink ? a.sink[cut.z % a.nh + head_of<EXACT>(a, h)] * PD_LOG2E : PD_NO_KEY;
  const int sets = min(SETS, last - first + 1);
  float top = sk;
  for (int k = 0; k < sets; ++k) top = fmaxf(top, ml_s[k].x);
  float sum = a.sink ? exp2_near(sk - top) : 0.f;
  y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < sets; ++k) {
    const float w = exp2_near(ml_s[k].x - top);
    const float4 v = y_s[k][e];
    sum = fmaf(w, ml_s[k].y, sum);
    y.x = fmaf(w, v.x, y.x); y.y = fmaf(w, v.y, y.y); y.z = fmaf(w, v.z, y.z); y.w = fmaf(w, v.w, y.w);
  }
  const float fac = sum != 0.f ? 1.f / sum : 0.f;
  put4<EXACT>(a, ((size_t)cut.z + place_of<EXACT>(a, h)) * D + 4 * e, y.x * fac, y.y * fac, y.z * fac, y.w * fac);
}

// ---------------------------------------------------------------- launchers
extern "C" int gg_packed_decode_mma_ok(int dtype, int d, int page_size, int bits) {
  return (dtype == GG_BF16 || dtype == GG_F32) && (d == 64 || d == 128) && page_size >= 16 && packed_sizes_ok(bits, d, page_size);
}

static int pd_sms() {
  static int n = 0;
  if (!n) {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) n = v;
  }
  return n > 0 ? n : 148;
}

struct PdShape { int nt, chunks, blocks; bool join; long long part_floats; };
template <int D, int BITS, int NT, bool EXACT> static void pd_fill(PdShape* s, int n, int nkv, int max_context, int window) {
  typedef PdSizes<D, BITS, NT, EXACT> Z;
  const long long reach = window > 0 && window < max_context ? (long long)window + Z::TILE - 1 : max_context;
  const long long tiles = (long long)n * nkv * s->chunks * ((reach + Z::TILE - 1) / Z::TILE);
  const long long want = (tiles + PD_EACH - 1) / PD_EACH;
  s->blocks = (int)(want < 1 ? 1 : want < pd_sms() ? want : pd_sms());
  // one token of a short context: a block for each pair, which then is cut nowhere and needs no second kernel
  s->join = true;
  if (n == 1 && nkv * s->chunks <= pd_sms() && (reach + Z::TILE - 1) / Z::TILE <= PD_ALONE * Z::WARPS) {
    s->blocks = nkv * s->chunks;
    s->join = false;
  }
  s->part_floats = (long long)s->blocks * (2 + Z::WARPS) * Z::PART;
}
#define PD_SIZES_NT(CALL, D, BITS)                                      \
  do {                                                                  \
    if (exact) CALL(D, BITS, 1, true);                                  \
    else if (nt == 1) CALL(D, BITS, 1, false);                          \
    else CALL(D, BITS, 2, false);                                       \
  } while (0)
#define PD_SIZES(CALL)                                                  \
  do {                                                                  \
    if (d == 64 && bits == 4) PD_SIZES_NT(CALL, 64, 4);                 \
    else if (d == 64) PD_SIZES_NT(CALL, 64, 8);                         \
    else if (bits == 4) PD_SIZES_NT(CALL, 128, 4);                      \
    else PD_SIZES_NT(CALL, 128, 8);                                     \
  } while (0)
static PdShape pd_shape(int n, int nh, int nkv, int d, int bits, int max_context, int window, bool exact) {
  PdShape s;
  const long long keys = (long long)n * nkv * (window > 0 && window < max_context ? window : max_context);
  const int group = nh / nkv, nt = group > 8 && !exact && keys >= PD_WIDE ? 2 : 1;
  s.nt = nt;
  s.chunks = (group + 8 * nt - 1) / (8 * nt);
#define PD_FILL(D, BITS, NT, EXACT) pd_fill<D, BITS, NT, EXACT>(&s, n, nkv, max_context, window)
  PD_SIZES(PD_FILL);
  return s;
}

// Scratch of gg_packed_decode_mma, in floats (what is to be joined lies behind the parts).
extern "C" long long gg_packed_decode_scratch(int dtype, int n, int nh, int nkv, int d, int bits, int max_context, int window) {
  const PdShape s = pd_shape(n, nh, nkv, d, bits, max_context, window, dtype == GG_F32);
  return s.part_floats + 4LL * s.blocks;
}

// The shape of that launch as one number: calls for which this says the same spread their work alike.
extern "C" int gg_packed_decode_shape(int dtype, int n, int nh, int nkv, int d, int bits, int max_context, int window) {
  const PdShape s = pd_shape(n, nh, nkv, d, bits, max_context, window, dtype == GG_F32);
  return (s.blocks * 2 + s.join) * 2 + s.nt - 1;
}

template <int D, int BITS, int NT, bool OPT, bool EXACT>
static int pd_launch(const PackedDecode& a, bool join, cudaStream_t stream) {
  typedef PdSizes<D, BITS, NT, EXACT> Z;
  // once for each device
  static std::atomic<unsigned long long> allowed{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1))) {
    e = cudaFuncSetAttribute(packed_decode_kernel<D, BITS, NT, OPT, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM);
    if (e == cudaSuccess && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return gg_fail(GG_ERR_CUDA, "packed_decode: %s", cudaGetErrorString(e));
  gg_launch(packed_decode_kernel<D, BITS, NT, OPT, EXACT>, dim3(a.blocks), dim3(Z::THREADS), Z::SMEM, stream, a);
  int rc = gg_check_launch("packed_decode");
  if (rc) return rc;
  if (!join || a.blocks == 1) return GG_OK;
  const int columns = a.fold > 1 ? a.fold * a.group : a.group;
  gg_launch(packed_join_kernel<D, NT, EXACT>, dim3(a.blocks, columns < 8 * NT ? columns : 8 * NT), dim3(256), 0, stream, a);
  return gg_check_launch("packed_join");
}

static int pd_check(const char* who, const PackedDecode& a, int dtype, int d, int page_size, int bits) {
  const int size = dtype == GG_F32 ? 4 : 2;
  GG_REQUIRE(gg_packed_decode_mma_ok(dtype, d, page_size, bits), "%s: head size %d, pages of %d tokens, %d bits or type %d are not taken", who, d, page_size, bits, dtype);
  GG_REQUIRE(a.nkv > 0 && a.nh > 0 && a.nh % a.nkv == 0, "%s: %d heads are not a multiple of %d kv heads", who, a.nh, a.nkv);
  GG_REQUIRE(a.n >= 0 && a.B >= 0 && a.num_pages >= 0 && a.bt_stride > 0 && a.window >= 0, "%s: bad sizes n=%d pages=%d table width=%d window=%d", who, a.n,
             a.num_pages, a.bt_stride, a.window);
  GG_REQUIRE(((size_t)a.q % 16) == 0 && a.q_stride * size % 16 == 0 && ((size_t)a.out % 16) == 0 && ((size_t)a.pages % 16) == 0,
             "%s: q, its rows, the output and the pages must start on 16 bytes", who);
  return GG_OK;
}
// Tokens of one launch over such block tables: its tiles are counted in an int (0: one token has more).
extern "C" int gg_packed_decode_tokens(int nh, int bt_stride, int page_size) {
  if (nh < 1 || bt_stride < 1 || page_size < 1) return PD_MAX_TOKENS;
  const long long each = nh * (((long long)bt_stride * page_size + 15) / 16), most = ((1LL << 31) - 1) / each;
  return (int)(most < PD_MAX_TOKENS ? most : PD_MAX_TOKENS);
}
static int pd_fits(const PackedDecode& a, const PdShape& s, int page_size, const float* scratch, long long scratch_floats) {
  GG_REQUIRE(a.n <= gg_packed_decode_tokens(a.nh, a.bt_stride, page_size), "packed_decode: block tables of %d pages for %d tokens are too large for one launch", a.bt_stride, a.n);
  GG_REQUIRE(scratch && ((size_t)scratch % 16) == 0 && scratch_floats >= s.part_floats + 4LL * s.blocks, "packed_decode: scratch too small");
  return GG_OK;
}
static int pd_run(PackedDecode a, bool exact, int d, int page_size, int bits, int max_context, float* scratch, long long scratch_floats, cudaStream_t stream) {
  const PdShape s = pd_shape(a.n, a.nh, a.nkv, d, bits, max_context, a.window, exact);
  int rc = pd_fits(a, s, page_size, scratch, scratch_floats);
  if (rc) return rc;
  a.group = a.nh / a.nkv;
  a.chunks = s.chunks;
  a.page_log2 = 31 - __builtin_clz(page_size);
  a.page_bytes = PackedRows(bits, d, page_size).page_bytes();
  a.part = scratch; a.cut = reinterpret_cast<int4*>(scratch + s.part_floats); a.blocks = s.blocks;
  const bool opt = a.softcap > 0.f || a.sink || a.slopes || a.temp_every > 0.f;
  const int nt = s.nt;
#define PD_RUN(D, BITS, NT, EXACT) return opt ? pd_launch<D, BITS, NT, true, EXACT>(a, s.join, stream) : pd_launch<D, BITS, NT, false, EXACT>(a, s.join, stream)
  PD_SIZES(PD_RUN);
}

extern "C" int gg_packed_decode_mma(const void* q, long long q_stride, int dtype, const void* pages, int num_pages, const int* tables, int bt_stride, int B,
                                    const int* cu_q_lens, const int* context_lens, const int* seqs, int n, int max_context, float* scratch,
                                    long long scratch_floats, void* out, int nh, int nkv, int d, int page_size, int bits, int window,
                                    float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every,
                                    int early, cudaStream_t stream) {
  PackedDecode a = {};
  a.q = q; a.q_stride = q_stride; a.pages = (const unsigned char*)pages; a.num_pages = num_pages;
  a.tables = tables; a.bt_stride = bt_stride; a.cu_q_lens = cu_q_lens; a.context_lens = context_lens; a.seqs = seqs; a.fold = 1; a.n = n; a.B = B;
  a.out = out; a.nh = nh; a.nkv = nkv; a.early = early;
  a.window = window; a.scale = scale; a.softcap = softcap; a.sink = sink; a.slopes = slopes; a.temp_coef = temp_coef; a.temp_every = temp_every;
  int rc = pd_check("packed_decode", a, dtype, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(n <= PD_MAX_TOKENS && max_context >= 0, "packed_decode: %d tokens are too many for one launch", n);
  GG_REQUIRE(seqs || n <= B, "packed_decode: %d tokens of %d sequences", n, B);
  if (n == 0) return GG_OK;
  return pd_run(a, dtype == GG_F32, d, page_size, bits, max_context, scratch, scratch_floats, stream);
}

// ---------------------------------------------------------------- prompt portions in float32
// Rows of a prompt portion as items of `fold` rows: seq, q0 [count], -1 behind the last.  A block for each sequence.
__global__ void __launch_bounds__(256) packed_items_kernel(const int* cu_q_lens, int B, int least, int fold, int* seq, int* q0, int count) {
  __shared__ int red[8];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x;                        // B: what is behind the last
  int before = 0;
  for (int i = threadIdx.x; i < b; i += 256) {
    const int n = cu_q_lens[i + 1] - cu_q_lens[i];
    before += n >= least ? (n + fold - 1) / fold : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += red[w];
  const int n = b < B ? cu_q_lens[b + 1] - cu_q_lens[b] : 0;
  const int items = b == B ? count - before : n >= least ? (n + fold - 1) / fold : 0;
  for (int i = threadIdx.x; i < items && before + i < count; i += 256) {
    seq[before + i] = b < B ? b : -1;
    q0[before + i] = i * fold;
  }
}

// Rows of a prompt portion that share an item: what fills the eight columns of a product.
static int pd_fold(int group) { return group <= 4 ? 8 / group : 1; }
extern "C" int gg_packed_prompt_fold(int nh, int nkv) { return nkv > 0 && nh >= nkv ? pd_fold(nh / nkv) : 1; }

// Every row of the portions attends as a single token does, in float32: `count` items of gg_packed_prompt_fold rows in all, their lists in
// `items` [2 count], at most gg_packed_decode_tokens a launch.  scratch as for gg_packed_decode_mma with as many tokens as the first launch has.
extern "C" int gg_packed_prompt_f32(const void* q, long long q_stride, const void* pages, int num_pages, const int* tables, int bt_stride, int B,
                                    const int* cu_q_lens, const int* context_lens, int least, int count, int* items, int max_context, float* scratch,
                                    long long scratch_floats, void* out, int nh, int nkv, int d, int page_size, int bits, int window,
                                    float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every,
                                    cudaStream_t stream) {
  PackedDecode a = {};
  a.q = q; a.q_stride = q_stride; a.pages = (const unsigned char*)pages; a.num_pages = num_pages;
  a.tables = tables; a.bt_stride = bt_stride; a.cu_q_lens = cu_q_lens; a.context_lens = context_lens; a.n = count; a.B = B;
  a.out = out; a.nh = nh; a.nkv = nkv;
  a.window = window; a.scale = scale; a.softcap = softcap; a.sink = sink; a.slopes = slopes; a.temp_coef = temp_coef; a.temp_every = temp_every;
  int rc = pd_check("packed_prompt", a, GG_F32, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(cu_q_lens && items && max_context >= 0, "packed_prompt: no lists");
  if (count == 0) return GG_OK;
  a.fold = pd_fold(nh / nkv);
  const int tokens = gg_packed_decode_tokens(nh, bt_stride, page_size), most = tokens > 0 ? tokens : 1;        // (1: refused below)
  a.n = count < most ? count : most;
  rc = pd_fits(a, pd_shape(a.n, nh, nkv, d, bits, max_context, window, true), page_size, scratch, scratch_floats);
  if (rc) return rc;
  gg_launch(packed_items_kernel, dim3(B + 1), dim3(256), 0, stream, cu_q_lens, B, least > 1 ? least : 1, a.fold, items, items + count, count);
  rc = gg_check_launch("packed_items");
  for (int lo = 0; lo < count && !rc; lo += most) {
    a.n = count - lo < most ? count - lo : most;
    a.seqs = items + lo;
    a.q0 = items + count + lo;
    rc = pd_run(a, true, d, page_size, bits, max_context, scratch, scratch_floats, stream);
  }
  return rc;
}
