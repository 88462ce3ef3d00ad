// The packed cache (format: packed_kv.cuh): rotation and quantisation as keys and values are written, reading them back (plain, or in half
// precision for the prompt kernels), and the launchers of attention over it.
#include "attention_common.cuh"
#include "packed_kv.cuh"

// ---------------------------------------------------------------- write
// Which code a value gets is decided as float64 arithmetic decides, round((x - offset) / scale) with ties to even: for a bfloat16 value as it
// came in float32, with float64 where it lies on a border (its difference from the offset is a float but for values that lie far apart); for
// a rotated key, and whatever came in float32, in float64.

__device__ __forceinline__ unsigned short bf16_down(float x) { return __bfloat16_as_ushort(__float2bfloat16_rd(x)); }
__device__ __forceinline__ unsigned short bf16_up(float x) { return __bfloat16_as_ushort(__float2bfloat16_ru(x)); }
__device__ __forceinline__ float bf16_value(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

// (scale, offset) of a group from its smallest and largest value, and a float64 value's code.  In float32, halves keep the range
// of a group that spans more than the largest float finite; halving is exact.
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
// row itself), a k or v head is rotated (k) and quantised into its page.  Every head's row passes through shared memory.  float64 arithmetic and
// rows passed lane by lane bound it: 4000 float32 tokens of 32 + 2 x 8 heads of 128 in 116 us (1.4 TB/s).
#define PACK_WARPS 8
template <typename TA>
__global__ void __launch_bounds__(PACK_WARPS * 32)
packed_write_kernel(const TA* __restrict__ qkv, long long row_stride, const int* __restrict__ positions, const int* __restrict__ slots,
                    const double* __restrict__ inv_freq, float mag, unsigned char* __restrict__ pages, int num_pages, TA* __restrict__ q_out,
                    long long q_stride, int nh, int nkv, int d, int rot, int page_size, int bits, int interleaved, int early) {
  typedef double TC;
  extern __shared__ double smem_d[];
  TC* cs = reinterpret_cast<TC*>(smem_d);             // cos[rot / 2], sin[rot / 2], then a row of each warp
  pdl_trigger();
  if (!early) pdl_wait();
  const int t = blockIdx.x, half = rot >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TC* row = cs + 2 * half + warp * d;
  if (half > 0) {
    const double pos = (double)positions[t];
    for (int p = threadIdx.x; p < half; p += blockDim.x) turn_of(pos, inv_freq[p], mag, &cs[p], &cs[half + p]);
  }
  const int slot = slots ? slots[t] : -1;
  __syncthreads();
  if (early) pdl_wait();
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

// The codes of eight values, 4 or 8 bits each, as one or two words.  A quotient by the reciprocal is off by less than 2^-21
// of the largest code; where one lies that near to a border (half between two codes: with bfloat16 values and scales many lie
// on it) the remainder decides, which one multiply-add gives to the last bit of the difference (a difference and a border are whole
// multiples of the difference's last place there, so what the subtraction rounded away decides on the border alone).  Halves keep a wide
// group's differences finite, and a group of tiny values is brought up by 2^64 so that its scale has a reciprocal (one of equal values has none).
template <int BITS>
__device__ __forceinline__ uint2 codes8(const PackCoder& k, const float* x) {
  constexpr float MOST = (1 << BITS) - 1, NEAR = 0.5f - MOST * 0x1p-21f;
  constexpr float MAGIC = 12582912.f;                  // 1.5 * 2^23: added, the whole number stands in the low bits
  const float up = k.half_scale > 0.f && k.half_scale < 0x1p-60f ? 0x1p64f : 1.f, scale = k.half_scale * up, offset = k.half_offset * up, half = 0.5f * up;
  const float inv = scale > 0.f ? 1.f / scale : 0.f;
  unsigned w[2] = {0u, 0u};
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fmaf(half, x[i], -offset) * inv, m = t + MAGIC;
    far = fmaxf(far, fabsf(t - (m - MAGIC)));
    w[i * BITS / 32] |= (__float_as_uint(m) & ((1u << BITS) - 1)) << (i * BITS & 31);
  }
  if (far >= NEAR) {
    const float border = 0.5f * scale;
    w[0] = w[1] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float diff = fmaf(half, x[i], -offset), m = diff * inv + MAGIC, rest = fmaf(-(m - MAGIC), scale, diff);
      const unsigned q = __float_as_uint(m) & 255u;
      unsigned above = rest > border, below = rest < -border;
      if (fabsf(rest) == border) {                     // what the difference lost, in float64 as the formula has it; nothing: the even code
        const double lost = ((double)half * x[i] - offset) - diff;
        above = rest > 0.f && (lost > 0.0 || (lost == 0.0 && (q & 1u)));
        below = rest < 0.f && (lost < 0.0 || (lost == 0.0 && (q & 1u)));
      }
      w[i * BITS / 32] |= ((q + above - below) & ((1u << BITS) - 1)) << (i * BITS & 31);
    }
  }
  return k.pair == 0x7fff7fffu ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
}

// The same for float64 values (rotated keys).  1.5 * 2^28 added leaves a quotient in the low word without a conversion (those between the widths
// take eight clocks a warp), in steps of 2^-24: the code is its rounded upper byte.  The quotient by the reciprocal is off by far less than a
// step; where the rest lies within a step of one half (a rotation by nothing, as at position 0, leaves bfloat16 values, which lie on a border
// often; others one in 2^22), the remainder decides, which is exact there.
template <int BITS>
__device__ __forceinline__ uint2 codes8(const PackCoder& k, const double* x) {
  const double inv = k.scale > 0.0 ? 1.0 / k.scale : 0.0;
  auto quotient = [&](int i) { return (unsigned)__double2loint(fma(x[i] - k.offset, inv, 402653184.0)); };
  unsigned w[2] = {0u, 0u};
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned t = quotient(i);
    near = near || ((t - 0x7fffffu) & 0xffffffu) <= 2u;
    w[i * BITS / 32] |= (t + 0x800000u) >> 24 << (i * BITS & 31);
  }
  if (near) {
    const double border = 0.5 * k.scale;
    w[0] = w[1] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned q = (quotient(i) + 0x800000u) >> 24;
      const double rest = fma(-(double)(int)q, k.scale, x[i] - k.offset);
      const bool odd = q & 1u;
      const unsigned move = (rest > border || (rest == border && odd)) ? 1u : (rest < -border || (rest == -border && odd)) ? ~0u : 0u;
      w[i * BITS / 32] |= (q + move) << (i * BITS & 31);
    }
  }
  return k.pair == 0x7fff7fffu ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
}
// A bfloat16 value (as a float) as float64: the exponent moved over, in integer arithmetic.
__device__ __forceinline__ double widen(float x) {
  const unsigned b = __float_as_uint(x), e = b & 0x7f800000u;
  if (e == 0u || e == 0x7f800000u) return (double)x;                 // zeros, subnormal numbers, infinities and NaN
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), 0);
}

// One head of one token, channels p .. p + 7 (a) and D / 2 + p .. (c) in each of the head's lanes: the group's extremes, its pair, the codes.
__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return a < b ? a : b; }
__device__ __forceinline__ double most(double a, double b) { return a < b ? b : a; }
template <int D, int BITS, typename TC>
__device__ __forceinline__ void store_head(const TC* a, const TC* c, bool nan0, bool nan1, int p, unsigned char* block, const PackedRows& r, int which, int place) {
  constexpr int HALF = D / 2, LANES = D / 16;
  // (heads of 64: one group)
  TC mn[2] = {a[0], c[0]}, mx[2] = {a[0], c[0]};
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    mn[0] = least(mn[0], a[j]); mx[0] = most(mx[0], a[j]);
    mn[1] = least(mn[1], c[j]); mx[1] = most(mx[1], c[j]);
  }
  if (D == 64) { mn[0] = least(mn[0], mn[1]); mx[0] = most(mx[0], mx[1]); }
  const unsigned mates = ((1u << LANES) - 1) << ((threadIdx.x & 31) & ~(LANES - 1));
  PackCoder k[2];
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      mn[g] = least(mn[g], __shfl_xor_sync(mates, mn[g], o));
      mx[g] = most(mx[g], __shfl_xor_sync(mates, mx[g], o));
    }
    const bool bad = __any_sync(mates, g ? nan1 : nan0) || !(mx[g] - mx[g] == 0) || !(mn[g] - mn[g] == 0);
    k[g].set(mn[g], mx[g], bad, BITS);
  }
  if (D == 64) k[1] = k[0];
  unsigned char* o = block + r.codes(which, place) + p * BITS / 8;
  const uint2 c0 = codes8<BITS>(k[0], a), c1 = codes8<BITS>(k[1], c);
  if (BITS == 4) {
    *reinterpret_cast<unsigned*>(o) = c0.x;
    *reinterpret_cast<unsigned*>(o + HALF * BITS / 8) = c1.x;
  } else {
    *reinterpret_cast<uint2*>(o) = c0;
    *reinterpret_cast<uint2*>(o + HALF * BITS / 8) = c1;
  }
  if (p == 0) {
    unsigned* q = reinterpret_cast<unsigned*>(block + r.pairs(which, place));
    if (D == 128) *reinterpret_cast<uint2*>(q) = make_uint2(k[0].pair, k[1].pair);
    else *q = k[0].pair;
  }
}

// The common case: bfloat16, heads of 64 or 128, half-split pairs over the whole head or no rotation, rows in 16-byte steps.
// Blocks of y = 0 take the k and v heads of TOK tokens, blocks of y = 1 their q heads (a tenth of the work a row: apart, so that
// all warps of a block are busy as long).  A thread takes channels p .. p + 7 and D / 2 + p .. of one head (two 16-byte loads,
// those of its next row under way while it works), so that a head's extremes are found by 4 or 8 neighbouring lanes.  Bound by waiting for its
// rows and the chain from a row's extremes to its codes (issue slots 55 % busy): 2048 tokens of 32 + 2 x 8 heads of 128 in 18.3 us (2.4 TB/s), 8000 in 61 us
// (2.8 TB/s).  Three blocks a multiprocessor: with the 88 to 92 registers that 128 channels would take it has two, and 8000 tokens take 76 us.
#define WRITE_THREADS 256
template <int D, int BITS, int TOK>
__global__ void __launch_bounds__(WRITE_THREADS, 3)
packed_write_vec_kernel(const __nv_bfloat16* __restrict__ qkv, long long row_stride, const int* __restrict__ positions,
                        const int* __restrict__ slots, const double* __restrict__ inv_freq, float mag, unsigned char* __restrict__ pages,
                        int num_pages, __nv_bfloat16* __restrict__ q_out, long long q_stride, int T, int nh, int nkv, int page_log2, int early) {
  constexpr int HALF = D / 2, LANES = D / 16;         // lanes of a head
  __shared__ double cs[TOK][2][HALF];                 // (queries: the same as float32)
  pdl_trigger();
  if (!early) pdl_wait();
  const int t0 = blockIdx.x * TOK, tokens = min(TOK, T - t0);
  const bool queries = blockIdx.y == 1;
  const int first = queries ? 0 : nh, per = (queries ? nh : 2 * nkv) * LANES;
  float* cf = reinterpret_cast<float*>(cs);
  if (inv_freq) {
    for (int e = threadIdx.x; e < tokens * HALF; e += WRITE_THREADS) {
      const int p = e % HALF, i = e / HALF;
      const double pos = (double)positions[t0 + i];
      if (queries) turn_of(pos, inv_freq[p], mag, &cf[(2 * i) * HALF + p], &cf[(2 * i + 1) * HALF + p]);
      else turn_of(pos, inv_freq[p], mag, &cs[i][0][p], &cs[i][1][p]);
    }
  }
  if (early) pdl_wait();
  const int P = 1 << page_log2;
  const PackedRows r(BITS, D, P);
  int w = threadIdx.x, i = 0;                         // item w of token i
  auto settle = [&]() { while (w >= per) { w -= per; ++i; } };
  auto row_at = [&]() { return qkv + (size_t)(t0 + i) * row_stride + (size_t)(first + w / LANES) * D + (w % LANES) * 8; };
  uint4 lo, hi;
  settle();
  if (i < tokens) {
    lo = *reinterpret_cast<const uint4*>(row_at());
    hi = *reinterpret_cast<const uint4*>(row_at() + HALF);
  }
  __syncthreads();                                    // the angles are there
  // (every lane of a head is in the same round: LANES divides the items of a token and 32)
  while (i < tokens) {
    const int h = first + w / LANES, p = (w % LANES) * 8, n = i;
    const unsigned wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
    w += WRITE_THREADS;
    settle();
    if (i < tokens) {
      lo = *reinterpret_cast<const uint4*>(row_at());
      hi = *reinterpret_cast<const uint4*>(row_at() + HALF);
    }
    float a[8], c[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[2 * j] = __uint_as_float(wl[j] << 16);
      a[2 * j + 1] = __uint_as_float(wl[j] & 0xffff0000u);
      c[2 * j] = __uint_as_float(wh[j] << 16);
      c[2 * j + 1] = __uint_as_float(wh[j] & 0xffff0000u);
    }
    if (queries) {
      if (inv_freq) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = a[j], v = c[j], co = cf[(2 * n) * HALF + p + j], si = cf[(2 * n + 1) * HALF + p + j];
          a[j] = u * co - v * si;
          c[j] = u * si + v * co;
        }
      }
      __nv_bfloat16* o = q_out + (size_t)(t0 + n) * q_stride + (size_t)h * D + p;
      *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(a[4], a[5]), pack_bf16(a[6], a[7]));
      *reinterpret_cast<uint4*>(o + HALF) = make_uint4(pack_bf16(c[0], c[1]), pack_bf16(c[2], c[3]), pack_bf16(c[4], c[5]), pack_bf16(c[6], c[7]));
      continue;
    }
    const int slot = slots ? slots[t0 + n] : -1;
    if (slot < 0 || (slot >> page_log2) >= num_pages) continue;
    const int which = h >= nh + nkv, kvh = h - nh - which * nkv, place = slot & (P - 1);
    unsigned char* block = pages + ((size_t)(slot >> page_log2) * nkv + kvh) * r.page_bytes();
    // a NaN (or infinity) shows in the sum of x * 0; turned, it is in both halves
    float bad0 = 0.f, bad1 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { bad0 = fmaf(a[j], 0.f, bad0); bad1 = fmaf(c[j], 0.f, bad1); }
    const bool turned = inv_freq && !which, one = turned || D == 64;
    const bool nan0 = bad0 != 0.f || (one && bad1 != 0.f), nan1 = bad1 != 0.f || (one && bad0 != 0.f);
    if (turned) {
      double x[8], y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double u = widen(a[j]), v = widen(c[j]), co = cs[n][0][p + j], si = cs[n][1][p + j];
        x[j] = u * co - v * si;
        y[j] = u * si + v * co;
      }
      store_head<D, BITS, double>(x, y, nan0, nan1, p, block, r, which, place);
    } else {
      store_head<D, BITS, float>(a, c, nan0, nan1, p, block, r, which, place);
    }
  }
}

// ---------------------------------------------------------------- read
// Eight neighbouring channels (of one group) of a token.
template <int BITS>
__device__ __forceinline__ void unpack8(const unsigned char* codes, unsigned pair, float up, float* y) {       // times `up`, a power of two
  const float s = __uint_as_float(pair << 16) * up, o = __uint_as_float(pair & 0xffff0000u) * up;
  if (BITS == 4) {
    const unsigned w = *reinterpret_cast<const unsigned*>(codes);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fmaf(s, (float)((w >> (4 * i)) & 15u), o);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(codes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = fmaf(s, (float)((w.x >> (8 * i)) & 255u), o);
      y[4 + i] = fmaf(s, (float)((w.y >> (8 * i)) & 255u), o);
    }
  }
}
__device__ __forceinline__ void store8(float* p, const float* y) {
  reinterpret_cast<float4*>(p)[0] = make_float4(y[0], y[1], y[2], y[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(y[4], y[5], y[6], y[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* y) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}
__device__ __forceinline__ void store8(__half* p, const float* y) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_half(y[0], y[1]), pack_half(y[2], y[3]), pack_half(y[4], y[5]), pack_half(y[6], y[7]));
}

// One page of one sequence: the codes of kv heads z, z + nz, ... become keys and values; the tokens from `real` on, and all
// of a page that was given back, become zeros.  UP: times ups[which * nkv + kv head].
template <typename TO, int BITS, bool UP>
__device__ __forceinline__ void unpack_page(const unsigned char* pages, int page, int num_pages, int real, TO* k_out, TO* v_out, int nkv, int d,
                                            int page_size, const float* ups) {
  const PackedRows r(BITS, d, page_size);
  const int per_row = d >> 3, units = 2 * page_size * per_row;
  if (page < 0 || page >= num_pages) { page = 0; real = 0; }
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const int row = u / per_row, c = (u - row * per_row) << 3, which = row >= page_size, place = row - which * page_size;
    const unsigned char* block = pages + ((size_t)page * nkv + blockIdx.z) * r.page_bytes();
    const int codes = row * r.row() + c * BITS / 8, pair = r.pairs(which, place) + (c / r.group) * 4;
    TO* o = (which ? v_out : k_out) + ((size_t)blockIdx.z * page_size + place) * d + c;
#pragma unroll 4
    for (int h = blockIdx.z; h < nkv; h += gridDim.z) {
      float y[8];
      unpack8<BITS>(block + codes, *reinterpret_cast<const unsigned*>(block + pair), UP ? ups[which * nkv + h] : 1.f, y);
      if (place >= real) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.f;
      }
      store8(o, y);
      block += (size_t)gridDim.z * r.page_bytes();
      o += (size_t)gridDim.z * page_size * d;
    }
  }
}

// A value that is no number goes over to its token's key: 0 times it would be a NaN in rows that do not see it, where a key's score is replaced
// (heads of 64 or 128 channels; all of the head is NaN in rows that do).  Behind unpack_page, by a call of its own (inlined, it takes registers).
__device__ __forceinline__ bool no_number(unsigned pair) { return (pair & 0x7f80u) == 0x7f80u; }          // the scale: of a group with an infinity or a NaN
template <int BITS>
__device__ __noinline__ void bad_values(const unsigned char* pages, int page, int real, __half* k_out, __half* v_out, int nkv, int d, int page_size) {
  const PackedRows r(BITS, d, page_size);
  __syncthreads();
  for (int h = blockIdx.z; h < nkv; h += gridDim.z)
    for (int u = threadIdx.x; u < min(real, page_size) * (d >> 3); u += blockDim.x) {
      const int place = u / (d >> 3), c = (u - place * (d >> 3)) << 3;
      const unsigned* values = reinterpret_cast<const unsigned*>(pages + ((size_t)page * nkv + h) * r.page_bytes() + r.pairs(1, place));
      if (!no_number(values[0]) && !no_number(values[r.groups() - 1])) continue;
      const size_t at = ((size_t)h * page_size + place) * d + c;
      *reinterpret_cast<uint4*>(k_out + at) = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      *reinterpret_cast<uint4*>(v_out + at) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// grid (pages of the longest sequence, B, nz): page j of sequence b becomes page first_page[b] + j of the results.  Bound by the results' bytes
// where there are many: 8000 tokens of 8 heads of 128 in 15.5 us from 4 bits (2.7 TB/s), 14.5 from 8 (3.5 TB/s); 2048 in 6.3 us.
template <typename TO, int BITS>
__global__ void __launch_bounds__(256)
packed_read_kernel(const unsigned char* __restrict__ pages, int num_pages, const int* __restrict__ tables, int bt_stride,
                   const int* __restrict__ lens, const int* __restrict__ first_page, TO* __restrict__ k_out, TO* __restrict__ v_out,
                   int out_pages, int nkv, int d, int page_size) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, j = blockIdx.x, len = lens[b];
  if (j * page_size >= len) return;
  const int to = first_page[b] + j;
  if (to < 0 || to >= out_pages) return;
  const size_t at = (size_t)to * nkv * page_size * d;
  unpack_page<TO, BITS, false>(pages, tables[(size_t)b * bt_stride + j], num_pages, len - j * page_size, k_out + at, v_out + at, nkv, d, page_size, nullptr);
}

// What the prompt kernels need of a packed layer's portions (sequences that bring `least` tokens or more), in one launch (without pages: the
// tiles alone): their
// pages as keys and values in half precision, one sequence behind the other; block tables of those pages; and the portions cut into tiles
// of query rows, those that attend to most keys first (up to UNFOLD_SORTED tiles; more stay in the order of the sequences).
// Pages behind the window of a portion's first token are left out (-1 in the table).
//
// Half precision has three bits more than bfloat16, so that a portion's result is as near as a single token's (0.17 % of 64 bits, the result's
// own rounding, where keys, values and weights in bfloat16 leave 0.31 to 0.37), and five bits of exponent fewer: a row of q, and the keys and the
// values of each kv head, are brought to a largest value of 2^12 to 2^13 by a power of two.  packed_loud_kernel finds how large the portions'
// keys and values are from their pages' scales and offsets, LOUD_BLOCKS partial maxima each; q's rows are made in the prompt kernels.
#define UNFOLD_SORTED 1024
#define UNFOLD_SEQS 1024          // most sequences of a step
#define UNFOLD_HEADS 1024         // most kv heads
#define LOUD_BLOCKS 128
struct UnfoldTiles { int height, count; int *seq, *q0; };
struct UnfoldArgs {
  const unsigned char* pages;
  int num_pages;
  const int *tables, *cu_q_lens, *context_lens;
  int bt_stride, B, least, nkv, d, page_size, window, out_pages;
  int* out_tables;                 // [B, bt_stride]
  UnfoldTiles tiles[2];            // height 0: none
  float* loud;                     // [LOUD_BLOCKS, 2, nkv]: the largest keys and values; [LOUD_BLOCKS]: whether some value is no number
  float* kv_unit;                  // [2, nkv]: what the halves are multiples of
};
__device__ __forceinline__ int unfold_keys(const UnfoldArgs& a, int b, int* q_len) {
  *q_len = a.cu_q_lens[b + 1] - a.cu_q_lens[b];
  if (*q_len < a.least) *q_len = 0;
  return *q_len ? (int)min((long long)a.context_lens[b], (long long)a.bt_stride * a.page_size) : 0;
}
__device__ __forceinline__ int unfold_skip(const UnfoldArgs& a, int ctx, int q_len) {          // pages nobody sees
  return a.window > 0 ? max(0, ctx - q_len - a.window + 1) / a.page_size : 0;
}

// By one block.  first[b] = tiles before sequence b; a tile finds its sequence by search and its place by counting the tiles
// that attend to more keys.
__device__ __noinline__ void list_tiles(const UnfoldArgs& a) {
  __shared__ int keys_s[UNFOLD_SORTED], first_s[UNFOLD_SEQS + 1], ctx_s[UNFOLD_SEQS], len_s[UNFOLD_SEQS];
  for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
    int n;
    ctx_s[b] = unfold_keys(a, b, &n);
    len_s[b] = n;
  }
  for (int l = 0; l < 2; ++l) {
    const UnfoldTiles t = a.tiles[l];
    if (!t.height) continue;
    __syncthreads();
    if (threadIdx.x < 32) {                            // tiles before each sequence: a warp's scan, 32 at a time
      int base = 0;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + threadIdx.x, n = b < a.B ? (len_s[b] + t.height - 1) / t.height : 0;
        int v = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if ((int)threadIdx.x >= o) v += u;
        }
        if (b < a.B) first_s[b] = base + v - n;
        base += __shfl_sync(0xffffffffu, v, 31);
      }
      if (threadIdx.x == 0) first_s[a.B] = base;
    }
    __syncthreads();
    const int made = first_s[a.B];
    auto tile = [&](int i, int* seq, int* q0) {        // (a count beyond what the portions make repeats the first tile)
      if (i >= made) i = 0;
      int lo = 0, hi = a.B - 1;                        // the last sequence whose tiles start at i or before
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (first_s[m] <= i) lo = m; else hi = m - 1;
      }
      *seq = lo;
      *q0 = (i - first_s[lo]) * t.height;
      return ctx_s[lo] - len_s[lo] + min(len_s[lo], *q0 + t.height);
    };
    const bool sorted = t.count <= UNFOLD_SORTED;
    int seq, q0;
    for (int i = threadIdx.x; i < t.count; i += blockDim.x) {
      const int keys = tile(i, &seq, &q0);
      if (sorted) keys_s[i] = keys;
      else { t.seq[i] = seq; t.q0[i] = q0; }
    }
    if (!sorted) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < t.count; i += blockDim.x) {
      const int mine = keys_s[i];
      int rank = 0;
#pragma unroll 8
      for (int k = 0; k < t.count; ++k) rank += keys_s[k] > mine || (keys_s[k] == mine && k < i);
      tile(i, &seq, &q0);
      t.seq[rank] = seq;
      t.q0[rank] = q0;
    }
  }
}

// The exponent of kv head v % nkv's keys (v < nkv) or values, by a warp.
__device__ __forceinline__ int loud_exponent(const UnfoldArgs& a, int v) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < LOUD_BLOCKS / 32; ++i) big = fmaxf(big, a.loud[(size_t)(i * 32 + (threadIdx.x & 31)) * 2 * a.nkv + v]);
  return half_exponent(warp_max(big));
}

// grid LOUD_BLOCKS.  The 2 nkv kinds (keys, then values, of each kv head) are cut into chunks of LOUD_KINDS, and a warp looks at one chunk of the pages
// whose number (page - first page in sight + LOUD_APART times the sequence) it has modulo the warps of that chunk: a page or two each, whose loads are
// all under way at once.  4 us for 2048 tokens of 8 heads, 5 for four sequences of 2900.
#define LOUD_KINDS 16
#define LOUD_APART 267            // (sequences begin at different warps)
template <int BITS>
__global__ void __launch_bounds__(256) packed_loud_kernel(UnfoldArgs a) {
  __shared__ unsigned big_s[2 * UNFOLD_HEADS];       // (sizes, which compare as whole numbers do)
  pdl_wait();
  pdl_trigger();                                     // not before: what packed_unfold_kernel reads ahead of its wait is all older than this kernel
  const int lane = threadIdx.x & 31, w = blockIdx.x * 8 + (threadIdx.x >> 5), kinds = 2 * a.nkv;
  const int P = a.page_size, groups_log2 = a.d >> 7, entries_log2 = 31 - __clz(P) + groups_log2;     // pairs of a page and kind: a power of two
  const PackedRows r(BITS, a.d, P);
  const int page_bytes = r.page_bytes(), values = r.pairs(1, 0) - r.pairs(0, 0);
  for (int v = threadIdx.x; v < kinds; v += 256) big_s[v] = 0u;
  __syncthreads();
  const int chunks = (kinds + LOUD_KINDS - 1) / LOUD_KINDS, slots = LOUD_BLOCKS * 8 / chunks, v0 = w % chunks * LOUD_KINDS, slot = w / chunks;
  bool bad = false;                                  // some value is no number
  unsigned top[LOUD_KINDS];
#pragma unroll
  for (int u = 0; u < LOUD_KINDS; ++u) top[u] = 0u;
  if (slot < slots) {
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int ctx = 0, j = 0, count = 0;
      if (b0 + lane < a.B) {
        int q_len;
        ctx = unfold_keys(a, b0 + lane, &q_len);
        count = (ctx + P - 1) / P;
        j = unfold_skip(a, ctx, q_len) + ((slot - (b0 + lane) * LOUD_APART) % slots + slots) % slots;
      }
      for (unsigned m = __ballot_sync(0xffffffffu, j < count); m; m &= m - 1) {
        const int src = __ffs(m) - 1, held = __shfl_sync(0xffffffffu, ctx, src), end = __shfl_sync(0xffffffffu, count, src);
        const int* row = a.tables + (size_t)(b0 + src) * a.bt_stride;
        for (int j0 = __shfl_sync(0xffffffffu, j, src); j0 < end; j0 += 32 * slots) {
          const int mine = j0 + lane * slots;
          const int id = mine < end ? row[mine] : -1;
          const int n = min(32, (end - j0 + slots - 1) / slots) << entries_log2;                     // pairs of those pages
          for (int x0 = 0; x0 < n; x0 += 32) {
            const int x = x0 + lane, k = min(x >> entries_log2, 31), e = x & ((1 << entries_log2) - 1);
            const int page = __shfl_sync(0xffffffffu, id, k);
            // (places behind the last token hold whatever was there)
            const bool there = x < n && page >= 0 && page < a.num_pages && (j0 + k * slots) * P + (e >> groups_log2) < held;
            const unsigned char* p = a.pages + (size_t)(there ? page : 0) * a.nkv * page_bytes + r.pairs(0, 0) + (size_t)e * 4;
            unsigned pair[LOUD_KINDS];
#pragma unroll
            for (int u = 0; u < LOUD_KINDS; ++u) {
              const int v = v0 + u;
              pair[u] = there && v < kinds ? *reinterpret_cast<const unsigned*>(p + (v < a.nkv ? (size_t)v * page_bytes : (size_t)(v - a.nkv) * page_bytes + values)) : 0u;
            }
#pragma unroll
            for (int u = 0; u < LOUD_KINDS; ++u) {
              const float s = __uint_as_float(pair[u] << 16), o = __uint_as_float(pair[u] & 0xffff0000u);
              const float g = fmaxf(fabsf(o), fabsf(fmaf(s, (float)((1 << BITS) - 1), o)));
              if (g < INFINITY) top[u] = max(top[u], __float_as_uint(g));
              else bad = bad || v0 + u >= a.nkv;
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < LOUD_KINDS; ++u) {
    const unsigned most = __reduce_max_sync(0xffffffffu, top[u]);
    if (lane == 0 && v0 + u < kinds && slot < slots) atomicMax(&big_s[v0 + u], most);
  }
  bad = __syncthreads_or(bad);
  for (int v = threadIdx.x; v < kinds; v += 256) a.loud[(size_t)blockIdx.x * kinds + v] = __uint_as_float(big_s[v]);
  if (threadIdx.x == 0) a.loud[(size_t)LOUD_BLOCKS * kinds + blockIdx.x] = bad ? 1.f : 0.f;
}

// Ahead of its wait it reads nothing that packed_loud_kernel writes (with the lists alone it has another kernel ahead, and waits at once).
// 10 us for 2048 tokens of 8 heads of 128 in 4 bits, 25 for 11600 in 8 (71 MB, 2.8 TB/s); five blocks a multiprocessor, since with the 62 registers it
// would take otherwise it has four, and those take 27.
template <int BITS>
__global__ void __launch_bounds__(256, 5) packed_unfold_kernel(UnfoldArgs a, __half* __restrict__ k_out, __half* __restrict__ v_out) {
  __shared__ int red[8];
  __shared__ float ups[2 * UNFOLD_HEADS];
  pdl_trigger();
  if (!k_out) pdl_wait();
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {                             // a block of its own, among the first
    if (blockIdx.y == 0 && blockIdx.z == 0) {
      list_tiles(a);
      pdl_wait();
      if (k_out)
        for (int v = threadIdx.x >> 5; v < 2 * a.nkv; v += 8) {
          const int e = loud_exponent(a, v);
          if (lane == 0) a.kv_unit[v] = two_to(-e);
        }
    }
    return;
  }
  const int b = blockIdx.y, j = blockIdx.x - 1;
  int q_len;
  const int ctx = unfold_keys(a, b, &q_len);
  const int skip = unfold_skip(a, ctx, q_len), P = a.page_size;
  if (j * P >= ctx || j < skip) {                    // nothing to read back
    if (j * P < ctx && threadIdx.x == 0 && blockIdx.z == 0) a.out_tables[(size_t)b * a.bt_stride + j] = -1;
    return;
  }
  const int page = a.tables[(size_t)b * a.bt_stride + j];
  // pages of the sequences before this one
  int before = 0;
  for (int i = threadIdx.x; i < b; i += blockDim.x) {
    int n;
    const int c = unfold_keys(a, i, &n);
    before += (c + P - 1) / P - unfold_skip(a, c, n);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) red[threadIdx.x >> 5] = before;
  pdl_wait();
  // this block's heads (blockIdx.z, blockIdx.z + gridDim.z, ...), keys and values
  for (int i = threadIdx.x >> 5; (int)blockIdx.z + (i >> 1) * (int)gridDim.z < a.nkv; i += 8) {
    const int v = (i & 1) * a.nkv + blockIdx.z + (i >> 1) * gridDim.z, e = loud_exponent(a, v);
    if (lane == 0) ups[v] = two_to(e);
  }
  bool bad = false;                                  // some value is no number
#pragma unroll
  for (int i = 0; i < LOUD_BLOCKS / 32; ++i) bad = bad || a.loud[(size_t)LOUD_BLOCKS * 2 * a.nkv + i * 32 + lane] != 0.f;
  bad = __any_sync(0xffffffffu, bad);
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += red[w];
  const int to = before + j - skip;
  const bool seen = to < a.out_pages;
  if (threadIdx.x == 0 && blockIdx.z == 0) a.out_tables[(size_t)b * a.bt_stride + j] = seen ? to : -1;
  if (seen) {
    const size_t at = (size_t)to * a.nkv * P * a.d;
    unpack_page<__half, BITS, true>(a.pages, page, a.num_pages, ctx - j * P, k_out + at, v_out + at, a.nkv, a.d, P, ups);
    if (bad && page >= 0 && page < a.num_pages) bad_values<BITS>(a.pages, page, ctx - j * P, k_out + at, v_out + at, a.nkv, a.d, P);
  }
}

static int check_packed(const char* who, const void* pages, int num_pages, int nkv, int d, int page_size, int bits) {
  GG_REQUIRE(packed_sizes_ok(bits, d, page_size), "%s: a packed cache has 4 or 8 bits, heads of 16 to 256 channels in sixteens and pages of a power of two "
             "of 4 to 256 tokens (got %d bits, head size %d, pages of %d)", who, bits, d, page_size);
  GG_REQUIRE(nkv > 0 && num_pages >= 0, "%s: bad sizes nkv=%d pages=%d", who, nkv, num_pages);
  GG_REQUIRE(((size_t)pages % 16) == 0, "%s: the pages must start on 16 bytes", who);
  return GG_OK;
}

// early: positions, slots and inv_freq are read before the kernel ahead has finished
extern "C" int gg_packed_write(const void* qkv, long long row_stride, int act_dtype, const int* positions, const int* slots,
                               const double* inv_freq, float mag, void* pages, int num_pages, void* q_out, long long q_stride, int T,
                               int nh, int nkv, int d, int rot, int page_size, int bits, int interleaved, int early, cudaStream_t stream) {
  int rc = check_packed("packed_write", pages, num_pages, nkv, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(T >= 0 && nh >= 0, "packed_write: bad sizes T=%d nh=%d", T, nh);
  GG_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0, "packed_write: rotary width %d must be even and <= head size %d", rot, d);
  GG_REQUIRE(rot == 0 || (inv_freq && positions), "packed_write: a rotation without frequencies or positions");
  if (T == 0) return GG_OK;
  if (act_dtype == GG_BF16 && (d == 64 || d == 128) && (rot == 0 || (rot == d && !interleaved)) && ((size_t)qkv % 16) == 0 &&
      row_stride % 8 == 0 && ((size_t)q_out % 16) == 0 && q_stride % 8 == 0) {
#define WRITE_VEC_T(D, BITS, TOK) gg_launch(packed_write_vec_kernel<D, BITS, TOK>, dim3((T + TOK - 1) / TOK, q_out ? 2 : 1), dim3(WRITE_THREADS), 0, \
                                            stream, (const __nv_bfloat16*)qkv, row_stride, positions, slots, rot ? inv_freq : nullptr, mag, \
                                            (unsigned char*)pages, num_pages, (__nv_bfloat16*)q_out, q_stride, T, nh, nkv, \
                                            31 - __builtin_clz(page_size), early)
    // tokens a block: us for 1 / 2 / 4 at 200, 512 and 1024 tokens of 32 + 2 x 8 heads of 128: 4.3 5.0 7.7, 8.4 6.6 8.9, 16.3 11.8 9.6
#define WRITE_VEC(D, BITS) do { if (T >= 888) WRITE_VEC_T(D, BITS, 4); else if (T >= 296) WRITE_VEC_T(D, BITS, 2); else WRITE_VEC_T(D, BITS, 1); } while (0)
    if (d == 64) { if (bits == 4) WRITE_VEC(64, 4); else WRITE_VEC(64, 8); }
    else { if (bits == 4) WRITE_VEC(128, 4); else WRITE_VEC(128, 8); }
    return gg_check_launch("packed_write");
  }
  const dim3 grid(T, (nh + 2 * nkv + PACK_WARPS - 1) / PACK_WARPS), block(PACK_WARPS * 32);
  GG_REQUIRE(grid.y <= 65535, "packed_write: too many heads");
  const size_t smem = (size_t)(rot + PACK_WARPS * d) * sizeof(double);
  if (act_dtype == GG_F32)
    gg_launch(packed_write_kernel<float>, grid, block, smem, stream, (const float*)qkv, row_stride, positions, slots, inv_freq, mag,
              (unsigned char*)pages, num_pages, (float*)q_out, q_stride, nh, nkv, d, rot, page_size, bits, interleaved, early);
  else if (act_dtype == GG_BF16)
    gg_launch(packed_write_kernel<__nv_bfloat16>, grid, block, smem, stream, (const __nv_bfloat16*)qkv, row_stride, positions, slots,
              inv_freq, mag, (unsigned char*)pages, num_pages, (__nv_bfloat16*)q_out, q_stride, nh, nkv, d, rot, page_size, bits, interleaved, early);
  else
    return gg_fail(GG_ERR_INVALID, "packed_write: unknown dtype %d", act_dtype);
  return gg_check_launch("packed_write");
}

// Blocks of a page: its kv heads are spread until the launch has a few blocks for every multiprocessor.
static int head_blocks(long long pages, int nkv) {
  int z = 1;
  while (z < nkv && z < 64 && pages * z < 1200) z *= 2;
  return z < nkv ? z : nkv;
}

extern "C" int gg_packed_read(const void* pages, int num_pages, const int* tables, int bt_stride, const int* lens, const int* first_page,
                              void* k_out, void* v_out, int out_dtype, int out_pages, int B, int most_pages, int nkv, int d, int page_size,
                              int bits, cudaStream_t stream) {
  int rc = check_packed("packed_read", pages, num_pages, nkv, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(B >= 0 && B <= 65535 && most_pages >= 0 && most_pages <= bt_stride, "packed_read: bad sizes B=%d pages=%d of %d", B, most_pages, bt_stride);
  GG_REQUIRE(((size_t)k_out % 16) == 0 && ((size_t)v_out % 16) == 0, "packed_read: the outputs must start on 16 bytes");
  GG_REQUIRE(out_dtype == GG_F32 || out_dtype == GG_BF16, "packed_read: unknown dtype %d", out_dtype);
  if (B == 0 || most_pages == 0) return GG_OK;
  const dim3 grid(most_pages, B, head_blocks(out_pages, nkv)), block(256);
#define READ_LAUNCH(TO, BITS) gg_launch(packed_read_kernel<TO, BITS>, grid, block, 0, stream, (const unsigned char*)pages, num_pages, tables, \
                                        bt_stride, lens, first_page, (TO*)k_out, (TO*)v_out, out_pages, nkv, d, page_size)
  if (out_dtype == GG_F32) { if (bits == 4) READ_LAUNCH(float, 4); else READ_LAUNCH(float, 8); }
  else { if (bits == 4) READ_LAUNCH(__nv_bfloat16, 4); else READ_LAUNCH(__nv_bfloat16, 8); }
  return gg_check_launch("packed_read");
}

// Floats that gg_packed_unfold works in: what the keys and values are multiples of [2, nkv] first, then its own.
extern "C" int gg_packed_unfold_floats(int nkv) { return 2 * nkv + LOUD_BLOCKS * (2 * nkv + 1); }

// k_out, v_out (half precision, with `floats`) null: the lists alone.
extern "C" int gg_packed_unfold(const void* pages, int num_pages, const int* tables, int bt_stride, const int* cu_q_lens,
                                const int* context_lens, int B, void* k_out, void* v_out, int out_pages, int most_pages,
                                int* out_tables, float* floats, int height0, int count0, int* seq0, int* q00, int height1, int count1,
                                int* seq1, int* q01, int least, int nkv, int d, int page_size, int bits, int window, cudaStream_t stream) {
  int rc = check_packed("packed_unfold", pages, num_pages, nkv, d, page_size, bits);
  if (rc) return rc;
  GG_REQUIRE(B > 0 && B <= UNFOLD_SEQS && most_pages >= 0 && most_pages <= bt_stride && window >= 0 && height0 >= 0 && height1 >= 0,
             "packed_unfold: bad sizes B=%d pages=%d of %d window=%d", B, most_pages, bt_stride, window);
  GG_REQUIRE(((size_t)k_out % 16) == 0 && ((size_t)v_out % 16) == 0, "packed_unfold: the outputs must start on 16 bytes");
  GG_REQUIRE(k_out ? v_out && out_tables && floats && nkv <= UNFOLD_HEADS && (d == 64 || d == 128) : most_pages == 0,
             "packed_unfold: missing outputs, %d kv heads or head size %d", nkv, d);
  UnfoldArgs a = {};
  a.pages = (const unsigned char*)pages; a.num_pages = num_pages; a.tables = tables; a.cu_q_lens = cu_q_lens; a.context_lens = context_lens;
  a.bt_stride = bt_stride; a.B = B; a.least = least > 1 ? least : 1; a.nkv = nkv; a.d = d; a.page_size = page_size; a.window = window; a.out_pages = out_pages;
  a.out_tables = out_tables; a.kv_unit = floats; a.loud = floats + 2 * nkv;
  a.tiles[0] = {height0, count0, seq0, q00};
  a.tiles[1] = {height1, count1, seq1, q01};
  if (k_out) {                                       // directly ahead: see packed_unfold_kernel
    if (bits == 4) gg_launch(packed_loud_kernel<4>, dim3(LOUD_BLOCKS), dim3(256), 0, stream, a);
    else gg_launch(packed_loud_kernel<8>, dim3(LOUD_BLOCKS), dim3(256), 0, stream, a);
    rc = gg_check_launch("packed_loud");
    if (rc) return rc;
  }
  const dim3 grid(most_pages + 1, most_pages ? B : 1, most_pages ? head_blocks(out_pages, nkv) : 1), block(256);
  if (bits == 4) gg_launch(packed_unfold_kernel<4>, grid, block, 0, stream, a, (__half*)k_out, (__half*)v_out);
  else gg_launch(packed_unfold_kernel<8>, grid, block, 0, stream, a, (__half*)k_out, (__half*)v_out);
  return gg_check_launch("packed_unfold");
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

// Single tokens on the general kernel.  part_o float[n * nh * splits * d], part_ml float[n * nh * splits * 2].
extern "C" int gg_packed_decode(const void* q, long long q_stride, int act_dtype, const void* pages, int num_pages, const int* tables,
                                int bt_stride, int B, const int* cu_q_lens, const int* context_lens, const int* seqs, int n, int splits,
                                float* part_o, float* part_ml, void* out, int nh, int nkv, int d, int page_size, int bits, int window,
                                float scale, float softcap, const float* sink, const float* slopes, float temp_coef, float temp_every,
                                cudaStream_t stream) {
  int rc = check_packed("packed_decode", pages, num_pages, nkv, d, page_size, bits);
  if (!rc) rc = check_heads("packed_decode", nh, nkv, bt_stride, window);
  if (rc) return rc;
  GG_REQUIRE(n >= 0 && B >= 0 && (seqs || n <= B) && splits >= 1 && splits <= 65535, "packed_decode: bad n %d of %d or splits %d", n, B, splits);
  if (n == 0) return GG_OK;
  AttnArgs a = packed_args(q, q_stride, pages, num_pages, tables, bt_stride, cu_q_lens, context_lens, out, nh, nkv, d, page_size, bits, window,
                           scale, softcap, sink, slopes, temp_coef, temp_every);
  a.num_seqs = B; a.dec_seqs = seqs; a.num_splits = splits; a.part_o = part_o; a.part_ml = part_ml;
  rc = attn_decode_general(a, act_dtype, n, stream);
  return rc ? rc : attn_merge_launch(a, act_dtype, n, stream);
}

// Prompt portions on the general kernel: tiles of 16 rows (packed_unfold lists them).
extern "C" int gg_packed_prefill(const void* q, long long q_stride, int act_dtype, const void* pages, int num_pages, const int* tables,
                                 int bt_stride, const int* cu_q_lens, const int* context_lens, const int* tile_seq, const int* tile_q0, int tiles,
                                 void* out, int nh, int nkv, int d, int page_size, int bits, int window, float scale, float softcap,
                                 const float* sink, const float* slopes, float temp_coef, float temp_every, cudaStream_t stream) {
  int rc = check_packed("packed_prefill", pages, num_pages, nkv, d, page_size, bits);
  if (!rc) rc = check_heads("packed_prefill", nh, nkv, bt_stride, window);
  if (rc) return rc;
  GG_REQUIRE(tiles >= 0 && cu_q_lens && context_lens && (tiles == 0 || (tile_seq && tile_q0)), "packed_prefill: bad lists of %d tiles", tiles);
  AttnArgs a = packed_args(q, q_stride, pages, num_pages, tables, bt_stride, cu_q_lens, context_lens, out, nh, nkv, d, page_size, bits, window,
                           scale, softcap, sink, slopes, temp_coef, temp_every);
  a.tile_seq = tile_seq; a.tile_q0 = tile_q0;
  return attn_prefill_general(a, act_dtype, tiles, stream);
}
