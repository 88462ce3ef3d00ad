// The packed cache (format: packed_kv.cuh): rotation and quantisation as keys and values are written, reading them back, and
// the launchers of attention over it.
#include "attention_common.cuh"
#include "packed_kv.cuh"

// ---------------------------------------------------------------- write
// Arithmetic: float32 for bfloat16 activations, float64 for float32 ones (whose last bits decide codes next to a border).
template <typename TA> struct PackMath;
template <> struct PackMath<__nv_bfloat16> { typedef float T; };
template <> struct PackMath<float> { typedef double T; };

__device__ __forceinline__ unsigned short bf16_down(float x) { return __bfloat16_as_ushort(__float2bfloat16_rd(x)); }
__device__ __forceinline__ unsigned short bf16_up(float x) { return __bfloat16_as_ushort(__float2bfloat16_ru(x)); }
__device__ __forceinline__ float bf16_value(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

// (scale, offset) of a group from its smallest and largest value, and a value's code.  Halves keep the range of a group
// that spans more than the largest float finite; halving is exact.
struct PackCoder {
  unsigned pair;
  float half_offset, half_scale;
  double offset, scale;
  int most;
  __device__ __forceinline__ void set(float mn, float mx, bool bad, int bits) {
    most = (1 << bits) - 1;
    if (bad) { pair = 0x7fff7fffu; half_offset = half_scale = 0.f; return; }
    const unsigned short o = bf16_down(mn);
    half_offset = 0.5f * bf16_value(o);
    const unsigned short s = bf16_up(__fdiv_ru(__fsub_ru(0.5f * mx, half_offset), 0.5f * (float)most));
    half_scale = 0.5f * bf16_value(s);
    pair = (unsigned)s | ((unsigned)o << 16);
  }
  __device__ __forceinline__ void set(double mn, double mx, bool bad, int bits) {
    most = (1 << bits) - 1;
    if (bad) { pair = 0x7fff7fffu; offset = scale = 0.0; return; }
    const unsigned short o = bf16_down(__double2float_rd(mn));
    offset = bf16_value(o);
    const unsigned short s = bf16_up(__double2float_ru((mx - offset) / most));
    scale = bf16_value(s);
    pair = (unsigned)s | ((unsigned)o << 16);
  }
  __device__ __forceinline__ unsigned code(float x) const {
    if (!(half_scale > 0.f)) return 0u;
    return (unsigned)fminf(fmaxf(rintf((0.5f * x - half_offset) / half_scale), 0.f), (float)most);
  }
  __device__ __forceinline__ unsigned code(double x) const {
    if (!(scale > 0.0)) return 0u;
    return (unsigned)fmin(fmax(rint((x - offset) / scale), 0.0), (double)most);
  }
};

__device__ __forceinline__ void turn_of(double pos, double freq, float mag, float* c, float* s) {
  // the angle is reduced modulo 2 pi in float64; float32 sine and cosine are exact to an ulp on the reduced argument
  const double two_pi = 6.283185307179586476925286766559;
  const double ang = pos * freq;
  sincosf((float)(ang - two_pi * rint(ang * (1.0 / two_pi))), s, c);
  *c *= mag;
  *s *= mag;
}
__device__ __forceinline__ void turn_of(double pos, double freq, float mag, double* c, double* s) {
  sincos(pos * freq, s, c);
  *c *= (double)mag;
  *s *= (double)mag;
}

// grid (T, ceil(heads / 8)): a warp takes one head (q, k or v) of one token.  A q head is rotated into q_out (which may be the
// row itself), a k or v head is rotated (k) and quantised into its page.  Every head's row passes through shared memory.
#define PACK_WARPS 8
template <typename TA>
__global__ void __launch_bounds__(PACK_WARPS * 32)
packed_write_kernel(const TA* __restrict__ qkv, long long row_stride, const int* __restrict__ positions, const int* __restrict__ slots,
                    const double* __restrict__ inv_freq, float mag, unsigned char* __restrict__ pages, int num_pages, TA* __restrict__ q_out,
                    long long q_stride, int nh, int nkv, int d, int rot, int page_size, int bits, int interleaved) {
  typedef typename PackMath<TA>::T TC;
  extern __shared__ double smem_d[];
  TC* cs = reinterpret_cast<TC*>(smem_d);             // cos[rot / 2], sin[rot / 2], then a row of each warp
  pdl_trigger();
  const int t = blockIdx.x, half = rot >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TC* row = cs + 2 * half + warp * d;
  if (half > 0) {
    const double pos = (double)positions[t];
    for (int p = threadIdx.x; p < half; p += blockDim.x) turn_of(pos, inv_freq[p], mag, &cs[p], &cs[half + p]);
  }
  const int slot = slots ? slots[t] : -1;
  __syncthreads();
  pdl_wait();
  const int h = blockIdx.y * PACK_WARPS + warp;
  if (h >= nh + 2 * nkv) return;
  if (h < nh ? q_out == nullptr : (slot < 0 || slot / page_size >= num_pages)) return;
  const TA* x = qkv + (size_t)t * row_stride + (size_t)h * d;
  for (int c = lane; c < d; c += 32) row[c] = (TC)to_f32(x[c]);
  __syncwarp();
  if (h < nh + nkv) {
    for (int p = lane; p < half; p += 32) {
      const int i0 = interleaved ? 2 * p : p, i1 = interleaved ? 2 * p + 1 : p + half;
      const TC u = row[i0], v = row[i1], c = cs[p], s = cs[half + p];
      row[i0] = u * c - v * s;
      row[i1] = u * s + v * c;
    }
    __syncwarp();
  }
  if (h < nh) {
    TA* o = q_out + (size_t)t * q_stride + (size_t)h * d;
    for (int c = lane; c < d; c += 32) o[c] = from_f32<TA>((float)row[c]);
    return;
  }
  const PackedRows r(bits, d, page_size);
  const int which = h >= nh + nkv, kvh = h - nh - which * nkv, place = slot % page_size;
  unsigned char* block = pages + ((size_t)(slot / page_size) * nkv + kvh) * r.page_bytes();
  for (int g = 0; g < r.groups(); ++g) {
    const bool mine = 2 * lane < r.group;
    const int c = g * r.group + (mine ? 2 * lane : 0);
    const TC a = row[c], b = row[c + 1];
    TC mn = a < b ? a : b, mx = a < b ? b : a;
    bool bad = !isfinite(a) || !isfinite(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const TC m2 = __shfl_xor_sync(0xffffffffu, mn, o), x2 = __shfl_xor_sync(0xffffffffu, mx, o);
      mn = m2 < mn ? m2 : mn;
      mx = x2 > mx ? x2 : mx;
    }
    bad = __any_sync(0xffffffffu, bad);
    PackCoder coder;
    coder.set(mn, mx, bad, bits);
    if (mine) {
      const unsigned qa = bad ? 0u : coder.code(a), qb = bad ? 0u : coder.code(b);
      if (bits == 4) block[r.codes(which, place) + (c >> 1)] = (unsigned char)(qa | (qb << 4));
      else *reinterpret_cast<unsigned short*>(block + r.codes(which, place) + c) = (unsigned short)(qa | (qb << 8));
    }
    if (lane == 0) *reinterpret_cast<unsigned*>(block + r.pairs(which, place) + g * 4) = coder.pair;
  }
}

// ---------------------------------------------------------------- read
// grid (pages of the longest sequence, B): a block turns one page of a sequence, all its kv heads, into keys and values
// [pages, nkv, P, d].  Rows behind the sequence's last token, and pages that were given back, read as zero.
template <typename TO>
__global__ void __launch_bounds__(256)
packed_read_kernel(const unsigned char* __restrict__ pages, int num_pages, const int* __restrict__ tables, int bt_stride,
                   const int* __restrict__ lens, const int* __restrict__ first_page, TO* __restrict__ k_out, TO* __restrict__ v_out,
                   int out_pages, int nkv, int d, int page_size, int bits) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, j = blockIdx.x, len = lens[b];
  if (j * page_size >= len) return;
  const int to = first_page[b] + j;
  if (to < 0 || to >= out_pages) return;
  const int page = tables[(size_t)b * bt_stride + j];
  const bool there = page >= 0 && page < num_pages;
  const PackedRows r(bits, d, page_size);
  const int per_row = d / 8, units = 2 * nkv * page_size * per_row;
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const int c = (u % per_row) * 8, place = (u / per_row) % page_size, hw = u / (per_row * page_size), kvh = hw >> 1, which = hw & 1;
    const unsigned char* block = pages + ((size_t)(there ? page : 0) * nkv + kvh) * r.page_bytes();
    TO* o = (which ? v_out : k_out) + (((size_t)to * nkv + kvh) * page_size + place) * d + c;
    const bool real = there && j * page_size + place < len;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = real ? r.value(block, which, place, c + i) : 0.f;
    store4(o, make_float4(y[0], y[1], y[2], y[3]));
    store4(o + 4, make_float4(y[4], y[5], y[6], y[7]));
  }
}

static int check_packed(const char* who, const void* pages, int num_pages, int nkv, int d, int page_size, int bits) {
  GG_REQUIRE(packed_sizes_ok(bits, d, page_size), "%s: a packed cache has 4 or 8 bits, heads of 16 to 256 channels in sixteens and pages of a power of two "
             "of 4 to 256 tokens (got %d bits, head size %d, pages of %d)", who, bits, d, page_size);
  GG_REQUIRE(nkv > 0 && num_pages >= 0, "%s: bad sizes nkv=%d pages=%d", who, nkv, num_pages);
  GG_REQUIRE(((size_t)pages % 16) == 0, "%s: the pages must start on 16 bytes", who);
  return GG_OK;
}

// positions, slots and inv_freq are read before the kernel ahead has finished
extern "C" int gg_packed_write(const void* qkv, long long row_stride, int act_dtype, const int* positions, const int* slots,
                               const double* inv_freq, float mag, void* pages, int num_pages, void* q_out, long long q_stride, int T,
                               int nh, int nkv, int d, int rot, int page_size, int bits, int interleaved, cudaStream_t stream) {
  int rc = check_packed("packed_write", pages, num_pages, nkv, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(T >= 0 && nh >= 0, "packed_write: bad sizes T=%d nh=%d", T, nh);
  GG_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0, "packed_write: rotary width %d must be even and <= head size %d", rot, d);
  GG_REQUIRE(rot == 0 || (inv_freq && positions), "packed_write: a rotation without frequencies or positions");
  if (T == 0) return GG_OK;
  const dim3 grid(T, (nh + 2 * nkv + PACK_WARPS - 1) / PACK_WARPS), block(PACK_WARPS * 32);
  GG_REQUIRE(grid.y <= 65535, "packed_write: too many heads");
  const int esize = act_dtype == GG_F32 ? 8 : 4;
  const size_t smem = (size_t)(rot + PACK_WARPS * d) * esize;
  if (act_dtype == GG_F32)
    gg_launch(packed_write_kernel<float>, grid, block, smem, stream, (const float*)qkv, row_stride, positions, slots, inv_freq, mag,
              (unsigned char*)pages, num_pages, (float*)q_out, q_stride, nh, nkv, d, rot, page_size, bits, interleaved);
  else if (act_dtype == GG_BF16)
    gg_launch(packed_write_kernel<__nv_bfloat16>, grid, block, smem, stream, (const __nv_bfloat16*)qkv, row_stride, positions, slots,
              inv_freq, mag, (unsigned char*)pages, num_pages, (__nv_bfloat16*)q_out, q_stride, nh, nkv, d, rot, page_size, bits, interleaved);
  else
    return gg_fail(GG_ERR_INVALID, "packed_write: unknown dtype %d", act_dtype);
  return gg_check_launch("packed_write");
}

extern "C" int gg_packed_read(const void* pages, int num_pages, const int* tables, int bt_stride, const int* lens, const int* first_page,
                              void* k_out, void* v_out, int out_dtype, int out_pages, int B, int most_pages, int nkv, int d, int page_size,
                              int bits, cudaStream_t stream) {
  int rc = check_packed("packed_read", pages, num_pages, nkv, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(B >= 0 && B <= 65535 && most_pages >= 0 && most_pages <= bt_stride, "packed_read: bad sizes B=%d pages=%d of %d", B, most_pages, bt_stride);
  GG_REQUIRE(((size_t)k_out % 16) == 0 && ((size_t)v_out % 16) == 0, "packed_read: the outputs must start on 16 bytes");
  if (B == 0 || most_pages == 0) return GG_OK;
  const dim3 grid(most_pages, B), block(256);
  if (out_dtype == GG_F32)
    gg_launch(packed_read_kernel<float>, grid, block, 0, stream, (const unsigned char*)pages, num_pages, tables, bt_stride, lens, first_page,
              (float*)k_out, (float*)v_out, out_pages, nkv, d, page_size, bits);
  else if (out_dtype == GG_BF16)
    gg_launch(packed_read_kernel<__nv_bfloat16>, grid, block, 0, stream, (const unsigned char*)pages, num_pages, tables, bt_stride, lens,
              first_page, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, out_pages, nkv, d, page_size, bits);
  else
    return gg_fail(GG_ERR_INVALID, "packed_read: unknown dtype %d", out_dtype);
  return gg_check_launch("packed_read");
}

// ---------------------------------------------------------------- attention
static AttnArgs packed_args(const void* q, long long q_stride, const void* pages, int num_pages, const int* tables, int bt_stride,
                            const int* cu_q_lens, const int* context_lens, void* out, int nh, int nkv, int d, int page_size, int bits,
                            int window, float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every) {
  AttnArgs a = {};
  a.q = q; a.q_stride = q_stride; a.kcache = pages; a.block_tables = tables; a.bt_stride = bt_stride; a.cu_q_lens = cu_q_lens;
  a.context_lens = context_lens; a.out = out; a.nh = nh; a.nkv = nkv; a.d = d; a.page_size = page_size; a.window = window;
  a.scale = scale; a.softcap = softcap; a.sink = sink; a.slopes = slopes; a.temp_coef = temp_coef; a.temp_every = temp_every;
  a.packed_bits = bits; a.num_pages = num_pages;
  return a;
}
static int check_heads(const char* who, int nh, int nkv, int bt_stride, int window) {
  GG_REQUIRE(nh > 0 && nh <= 65535 && nh % nkv == 0, "%s: %d heads are not a multiple of %d kv heads", who, nh, nkv);
  GG_REQUIRE(bt_stride > 0 && window >= 0, "%s: bad block table width %d or window %d", who, bt_stride, window);
  return GG_OK;
}

// Prompt portions on the general kernel: tiles of 16 query rows.
extern "C" int gg_packed_prefill(const void* q, long long q_stride, int act_dtype, const void* pages, int num_pages, const int* tables,
                                 int bt_stride, const int* cu_q_lens, const int* context_lens, const int* tile_seq, const int* tile_q0,
                                 int num_tiles, void* out, int nh, int nkv, int d, int page_size, int bits, int window, float scale,
                                 float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every, cudaStream_t stream) {
  int rc = check_packed("packed_prefill", pages, num_pages, nkv, d, page_size, bits);
  if (!rc) rc = check_heads("packed_prefill", nh, nkv, bt_stride, window);
  if (rc) return rc;
  AttnArgs a = packed_args(q, q_stride, pages, num_pages, tables, bt_stride, cu_q_lens, context_lens, out, nh, nkv, d, page_size, bits, window,
                           scale, softcap, sink, slopes, temp_coef, temp_every);
  a.tile_seq = tile_seq; a.tile_q0 = tile_q0;
  return attn_prefill_general(a, act_dtype, num_tiles, stream);
}

// Single tokens on the general kernel.  part_o float[n * nh * splits * d], part_ml float[n * nh * splits * 2].
extern "C" int gg_packed_decode(const void* q, long long q_stride, int act_dtype, const void* pages, int num_pages, const int* tables,
                                int bt_stride, const int* cu_q_lens, const int* context_lens, const int* seqs, int n, int splits,
                                float* part_o, float* part_ml, void* out, int nh, int nkv, int d, int page_size, int bits, int window,
                                float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every,
                                cudaStream_t stream) {
  int rc = check_packed("packed_decode", pages, num_pages, nkv, d, page_size, bits);
  if (!rc) rc = check_heads("packed_decode", nh, nkv, bt_stride, window);
  if (rc) return rc;
  GG_REQUIRE(n >= 0 && splits >= 1 && splits <= 65535, "packed_decode: bad n %d or splits %d", n, splits);
  if (n == 0) return GG_OK;
  AttnArgs a = packed_args(q, q_stride, pages, num_pages, tables, bt_stride, cu_q_lens, context_lens, out, nh, nkv, d, page_size, bits, window,
                           scale, softcap, sink, slopes, temp_coef, temp_every);
  a.dec_seqs = seqs; a.num_splits = splits; a.part_o = part_o; a.part_ml = part_ml;
  rc = attn_decode_general(a, act_dtype, n, stream);
  return rc ? rc : attn_merge_launch(a, act_dtype, n, stream);
}
