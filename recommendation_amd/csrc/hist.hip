// A user's event history as a paged cache of keys and values: rows appended (mi_hist_write), read back
// (mi_hist_read) and attended by new tokens or candidates (mi_hist_attn).  The reference holds no histories; its
// nearest analogue is the list of recommended and clicked colours that every request carries and the model pools
// (recommendation/code/r_model.py:68-80).
//
// Cache: kv [n_pages][heads][2][page_size][dim] (0 keys, 1 values) in f32, bf16 or e4m3; an e4m3 row stands for
// code * 2^(exps - 127), one exponent byte per row, exps [n_pages][heads][2][page_size].  A power of two as the row's
// scale costs no accuracy that a floating 8-bit code does not lose anyway, and makes scaling exact: a row is rounded
// once, and every program that knows the rule gets the same codes.
#include "common.h"

namespace {

typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

template <int DT>
struct Elem;
template <>
struct Elem<MI_DT_F32> {
  static constexpr int BYTES = 4;
};
template <>
struct Elem<MI_DT_BF16> {
  static constexpr int BYTES = 2;
};
template <>
struct Elem<MI_DT_E4M3> {
  static constexpr int BYTES = 1;
};

__device__ __forceinline__ float pow2_bits(unsigned int e) { return __uint_as_float(e << 23); }

__device__ __forceinline__ void report(int32_t* err, int bit) {
  if (err) atomicOr(err, bit);
}

// ------------------------------------------------------------------------------------------------ rows: write, read
struct RowArgs {
  char* kv;
  uint8_t* exps;
  int64_t n_pages;
  int H, page_shift;
  const int32_t* table;
  int64_t ld_table;
  int width;                // pages a table row has room for
  const int32_t* lengths;
  int64_t n_seqs;
  const int64_t* offsets;   // [n_seqs + 1], or NULL: `each` rows per sequence
  int64_t each;
  int64_t n_rows;
  const char* k;            // inputs of a write, outputs of a read
  const char* v;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  int32_t* err;
};

// Number of the sorted offsets[0..n) that are <= i, by the whole wave: 64 of them a step.
__device__ __forceinline__ int64_t wave_upper_bound(const int64_t* __restrict__ offsets, int64_t n, int64_t i, int lane) {
  int64_t lo = 0, size = n;
  while (size > 0) {
    const int64_t step = (size + 63) >> 6;
    const int64_t at = lo + lane * step;
    const bool le = lane * step < size && offsets[at] <= i;
    const int got = __popcll(__ballot(le));
    if (step == 1) return lo + got;
    if (got == 0) return lo;
    // the count ends behind entry (got - 1) * step, at most step - 1 entries further
    lo += (got - 1) * step + 1;
    size = (size - ((got - 1) * step + 1) < step - 1) ? size - ((got - 1) * step + 1) : step - 1;
  }
  return lo;
}

// Where row i of the call lives: false if no sequence owns it.  [b0, b1]: the sequences the wave's rows can belong to.
struct Place {
  int64_t page;  // -1: the row has no place (in front of position 0, or a bad page)
  int slot;
};
__device__ __forceinline__ bool find_place(const RowArgs& p, int64_t i, int64_t b0, int64_t b1, Place* out) {
  int64_t b, last;
  if (p.offsets) {
    while (b0 < b1) {  // the last b with offsets[b] <= i
      const int64_t mid = (b0 + b1 + 1) >> 1;
      if (p.offsets[mid] <= i) b0 = mid; else b1 = mid - 1;
    }
    b = b0;
    if (b < 0 || b >= p.n_seqs) return false;
    last = p.offsets[b + 1];
  } else {
    b = (int64_t) ((uint32_t) i / (uint32_t) p.each);
    last = (b + 1) * p.each;
  }
  const int64_t len = p.lengths[b];
  const int64_t pos = len - (last - i);
  out->page = -1;
  out->slot = 0;
  if (pos < 0 || pos >= len) return true;
  const int64_t pi = pos >> p.page_shift;
  if (pi >= p.width) {
    report(p.err, MI_IDERR_RANGE);
    return true;
  }
  const int64_t page = p.table[b * p.ld_table + pi];
  if (page < 0 || page >= p.n_pages) {
    report(p.err, MI_IDERR_RANGE);
    return true;
  }
  out->page = page;
  out->slot = (int) (pos & ((1 << p.page_shift) - 1));
  return true;
}

struct Eight {
  float x[8];
};
template <int DT>
__device__ __forceinline__ Eight load8(const char* p);
template <>
__device__ __forceinline__ Eight load8<MI_DT_F32>(const char* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
template <>
__device__ __forceinline__ Eight load8<MI_DT_BF16>(const char* p) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  Eight r;
  const unsigned int w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.x[2 * i] = __uint_as_float(w[i] << 16);
    r.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return r;
}
__device__ __forceinline__ unsigned int pack_bf16(float a, float b) {
  bf2v p;
  p[0] = (__bf16) a;
  p[1] = (__bf16) b;
  return __builtin_bit_cast(unsigned int, p);
}
template <int DT>
__device__ __forceinline__ void store8(char* p, const Eight& e);
template <>
__device__ __forceinline__ void store8<MI_DT_F32>(char* p, const Eight& e) {
  reinterpret_cast<float4*>(p)[0] = make_float4(e.x[0], e.x[1], e.x[2], e.x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(e.x[4], e.x[5], e.x[6], e.x[7]);
}
template <>
__device__ __forceinline__ void store8<MI_DT_BF16>(char* p, const Eight& e) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(e.x[0], e.x[1]), pack_bf16(e.x[2], e.x[3]),
                                            pack_bf16(e.x[4], e.x[5]), pack_bf16(e.x[6], e.x[7]));
}

// Quantisation of a row x: a = max finite |x|, e the smallest exponent with a * 2^-e <= 448 (the largest e4m3 value),
// at least -126 so that 2^e and 2^-e are normal f32; codes = e4m3(x * 2^-e) to nearest even.  +-inf and NaN become
// NaN (e4m3 has no infinity, and a clamped one would look like data).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // false for NaN too
}
__device__ __forceinline__ unsigned int row_exponent(float top) {  // e + 127
  const unsigned int u = __float_as_uint(top);
  int biased = (int) (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // top <= 1.75 * 2^k fits 448 * 2^(k-8)
  return biased < 1 ? 1u : (unsigned int) biased;
}
__device__ __forceinline__ uint2 quantise8(const Eight& e, unsigned int exponent) {
  const float inv = pow2_bits(254u - exponent);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = e.x[i] * inv;
    if (!(fabsf(e.x[i]) < INFINITY)) y[i] = NAN;
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return make_uint2((unsigned int) lo, (unsigned int) hi);
}
__device__ __forceinline__ Eight dequantise8(uint2 c, unsigned int exponent) {
  const float s = pow2_bits(exponent);
  Eight r;
  const unsigned int w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf2v lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, false);  // exact: 4 significant bits
    const bf2v hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, true);
    r.x[4 * i + 0] = (float) lo[0] * s;
    r.x[4 * i + 1] = (float) lo[1] * s;
    r.x[4 * i + 2] = (float) hi[0] * s;
    r.x[4 * i + 3] = (float) hi[1] * s;
  }
  return r;
}

// D / 8 lanes per cache row; a row is (token, K or V, head), tokens slowest.  UNROLL rows per lane group are requested
// together.  READ: the cache is the source, k and v the destination.
constexpr int ROW_UNROLL = 4;

template <int CT, int IT, int D, bool READ>
__global__ __launch_bounds__(256) void hist_rows_kernel(RowArgs p) {
  constexpr int LPR = D / 8, GROUPS = 64 / LPR, PER_WAVE = GROUPS * ROW_UNROLL;
  constexpr int CE = Elem<CT>::BYTES, IE = Elem<IT>::BYTES;
  const int lane = threadIdx.x & 63;
  const unsigned int per_token = 2u * (unsigned int) p.H;
  const unsigned int total = (unsigned int) p.n_rows * per_token;  // checked on the host
  const unsigned int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const unsigned int r0 = wave * PER_WAVE;
  if (r0 >= total) return;
  const unsigned int r1 = r0 + PER_WAVE - 1 < total ? r0 + PER_WAVE - 1 : total - 1;
  int64_t b0 = 0, b1 = 0;
  if (p.offsets) {
    b0 = wave_upper_bound(p.offsets, p.n_seqs + 1, r0 / per_token, lane) - 1;
    b1 = wave_upper_bound(p.offsets, p.n_seqs + 1, r1 / per_token, lane) - 1;
  }
  const int c = lane % LPR;
  int64_t tok[ROW_UNROLL];
  int part[ROW_UNROLL], head[ROW_UNROLL];
  bool live[ROW_UNROLL];
  Place at[ROW_UNROLL];
  Eight x[ROW_UNROLL];
#pragma unroll
  for (int u = 0; u < ROW_UNROLL; ++u) {
    const unsigned int r = r0 + u * GROUPS + lane / LPR;
    live[u] = r < total;
    const unsigned int rr = live[u] ? r : r0;
    tok[u] = rr / per_token;
    const unsigned int rem = rr - (unsigned int) tok[u] * per_token;
    part[u] = rem >= (unsigned int) p.H ? 1 : 0;
    head[u] = (int) rem - part[u] * p.H;
    if (!READ) {
      const char* src = part[u] ? p.v + (tok[u] * p.v_row + head[u] * p.v_head + c * 8) * IE
                                : p.k + (tok[u] * p.k_row + head[u] * p.k_head + c * 8) * IE;
      x[u] = load8<IT>(src);
    }
  }
#pragma unroll
  for (int u = 0; u < ROW_UNROLL; ++u) {
    // lanes past the end repeat the wave's first row, which must not be reported twice: harmless, the bit is the same
    live[u] &= find_place(p, tok[u], b0, b1, &at[u]);
  }
#pragma unroll
  for (int u = 0; u < ROW_UNROLL; ++u) {
    const int64_t row = (((at[u].page * p.H + head[u]) * 2 + part[u]) << p.page_shift) + at[u].slot;
    if (READ) {
      Eight y = Eight{{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
      if (live[u] && at[u].page >= 0) {
        const char* src = p.kv + (row * D + c * 8) * CE;
        if (CT == MI_DT_E4M3) y = dequantise8(*reinterpret_cast<const uint2*>(src), p.exps[row]);
        else y = load8<CT == MI_DT_E4M3 ? MI_DT_F32 : CT>(src);
      }
      if (live[u]) {
        char* dst = const_cast<char*>(part[u] ? p.v + (tok[u] * p.v_row + head[u] * p.v_head + c * 8) * IE
                                              : p.k + (tok[u] * p.k_row + head[u] * p.k_head + c * 8) * IE);
        store8<IT>(dst, y);
      }
    } else {
      float top = 0.f;
      if (CT == MI_DT_E4M3) {  // all lanes take part in the exchange
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_abs(x[u].x[i]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
      }
      if (live[u] && at[u].page >= 0) {
        char* dst = p.kv + (row * D + c * 8) * CE;
        if (CT == MI_DT_E4M3) {
          const unsigned int e = row_exponent(top);
          *reinterpret_cast<uint2*>(dst) = quantise8(x[u], e);
          if (c == 0) p.exps[row] = (uint8_t) e;
        } else {
          store8<CT == MI_DT_E4M3 ? MI_DT_F32 : CT>(dst, x[u]);
        }
      }
    }
  }
}

template <int CT, int IT, bool READ>
int launch_rows(const RowArgs& p, int dim, hipStream_t s) {
  const int64_t rows = p.n_rows * 2 * p.H;
  const int per_block = 4 * (64 / (dim / 8)) * ROW_UNROLL;
  const dim3 grid((unsigned int) mi_cdiv(rows, per_block));
  switch (dim) {
    case 32: hist_rows_kernel<CT, IT, 32, READ><<<grid, 256, 0, s>>>(p); break;
    case 64: hist_rows_kernel<CT, IT, 64, READ><<<grid, 256, 0, s>>>(p); break;
    case 128: hist_rows_kernel<CT, IT, 128, READ><<<grid, 256, 0, s>>>(p); break;
    default: hist_rows_kernel<CT, IT, 256, READ><<<grid, 256, 0, s>>>(p); break;
  }
  MI_LAUNCH_CHECK();
  return MI_OK;
}

// ------------------------------------------------------------------------------------------------ attention
struct AttnArgs {
  const char* kv;
  const uint8_t* exps;
  int64_t n_pages;
  int H, page_shift;
  const char* q;
  int64_t q_seq, q_tok, q_head;  // strides in elements
  char* out;
  int64_t o_seq, o_tok, o_head;
  int G, rows, n_rt;             // query heads per cache head; n_q * G query rows per cache head, in tiles of 16
  const int32_t* table;
  int64_t ld_table;
  int width;
  const int32_t* lengths;
  int64_t n_seqs;
  float scale;                   // of the scores, times log2(e)
  int32_t* err;
};

// One wave's running state for 16 query rows of one cache head: o = sum_j 2^(s_j - m) v_j, l = sum_j 2^(s_j - m).
//
// Both products are matrix instructions whose operands come straight from memory.  Scores are formed transposed,
// S^T = K Q^T (rows: 16 cached positions; columns: query rows): lane (g = lane / 16, c = lane % 16) then holds the
// scores of query row c for positions 4g .. 4g+3 of a tile, which is what the second product, O^T = V^T P^T, wants as
// its right operand if its reduction index is read as "positions 4g..4g+3 of tile 0, then of tile 1".  Its left
// operand takes output channels j of 16 lanes' 16-byte pieces of a V row, whatever those channels are called.  So no
// score, probability or value crosses lanes; only the row maximum and sum do (over the four g).
template <int DT, int D>
struct Wave {
  static constexpr bool F32 = DT == MI_DT_F32;
  static constexpr int E = Elem<DT>::BYTES;
  static constexpr int QE = F32 ? 4 : 2;                    // query / output element
  // K: a lane fetches KB bytes of its position's row per load, the four g of a position KB * 4 contiguous bytes
  static constexpr int KB = D * E >= 64 ? 16 : D * E / 4;
  static constexpr int KL = D * E / 4 / KB;
  static constexpr int KN = KB / E;                         // channels per lane and load
  // V: a lane fetches VE channels of each of its 4 positions per piece
  static constexpr int VB = D * E / 16 > 16 ? 16 : D * E / 16;
  static constexpr int VE = VB / E;
  static constexpr int VH = D / 16 / VE;
  static constexpr int CHUNK = 32;                          // positions per step, two tiles
  static constexpr int NS = D / 32;                         // 32-channel steps of the score product (8 / 16 bit)

  f4v o[VH][VE];
  float m, l;
  bf8v qf[F32 ? 1 : NS];
  f4v qv[F32 ? KL : 1];

  // channel of element 0 of this lane's query fragment of step s
  static __device__ __forceinline__ int q_channel(int s, int g) {
    if (DT == MI_DT_E4M3 && KN == 16) return (s >> 1) * 64 + g * 16 + (s & 1) * 8;
    return s * 32 + g * 8;
  }

  __device__ __forceinline__ void init(const char* q_row, bool live, int g) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < VE; ++j) o[h][j] = f4v{0.f, 0.f, 0.f, 0.f};
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < KL; ++s) {
        const f4v x = *reinterpret_cast<const f4v*>(q_row + (s * 16 + g * 4) * 4);
        qv[s] = live ? x : f4v{0.f, 0.f, 0.f, 0.f};
      }
    } else {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const uint4 x = *reinterpret_cast<const uint4*>(q_row + q_channel(s, g) * 2);
        qf[s] = __builtin_bit_cast(bf8v, live ? x : make_uint4(0, 0, 0, 0));
      }
    }
  }

  struct Fetched {
    unsigned int k[2][KL][KB / 4];
    unsigned int v[2][4][VH][VB < 4 ? 1 : VB / 4];
    unsigned int ek[2], ev[2];
  };

  template <int BYTES>
  static __device__ __forceinline__ void fetch(unsigned int* dst, const char* src) {
    if constexpr (BYTES == 16) {
      const uint4 x = *reinterpret_cast<const uint4*>(src);
      dst[0] = x.x; dst[1] = x.y; dst[2] = x.z; dst[3] = x.w;
    } else if constexpr (BYTES == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(src);
      dst[0] = x.x; dst[1] = x.y;
    } else if constexpr (BYTES == 4) {
      dst[0] = *reinterpret_cast<const unsigned int*>(src);
    } else {
      dst[0] = *reinterpret_cast<const unsigned short*>(src);
    }
  }

  // rows: index of the tile's first K row in the cache (V lies page_size rows behind)
  __device__ __forceinline__ void request(Fetched& f, const AttnArgs& p, const int64_t (&rows)[2], int g, int c) {
    const int page = 1 << p.page_shift;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* kb = p.kv + rows[t] * (D * E);
#pragma unroll
      for (int s = 0; s < KL; ++s) fetch<KB>(f.k[t][s], kb + c * (D * E) + s * (KB * 4) + g * KB);
      if (DT == MI_DT_E4M3) f.ek[t] = *reinterpret_cast<const unsigned int*>(p.exps + rows[t] + 4 * g);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* vb = p.kv + (rows[t] + page) * (D * E);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int h = 0; h < VH; ++h)
          fetch<VB>(f.v[t][r][h], vb + (4 * g + r) * (D * E) + h * (VB * 16) + c * VB);
      if (DT == MI_DT_E4M3) f.ev[t] = *reinterpret_cast<const unsigned int*>(p.exps + rows[t] + page + 4 * g);
    }
  }

  static __device__ __forceinline__ bf8v widen(unsigned int lo, unsigned int hi) {  // 8 e4m3 codes, exactly
    uint4 w;
    w.x = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w.y = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w.z = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w.w = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return __builtin_bit_cast(bf8v, w);
  }

  // scores, softmax step and weighted sum of one chunk; valid[t]: live positions of tile t (16: all)
  __device__ __forceinline__ void step(Fetched& f, const AttnArgs& p, const int (&valid)[2], int g, int c) {
    f4v s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f4v acc = f4v{0.f, 0.f, 0.f, 0.f};
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < KL; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.k[t][k][i]), qv[k][i], acc, 0, 0, 0);
      } else if constexpr (DT == MI_DT_BF16) {
#pragma unroll
        for (int k = 0; k < KL; ++k) {
          const uint4 w = make_uint4(f.k[t][k][0], f.k[t][k][1], f.k[t][k][2], f.k[t][k][3]);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, w), qf[k], acc, 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KL; ++k)
#pragma unroll
          for (int u = 0; u < KB / 8; ++u)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(f.k[t][k][2 * u], f.k[t][k][2 * u + 1]),
                                                          qf[k * (KB / 8) + u], acc, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = acc[r] * p.scale;
        if (DT == MI_DT_E4M3) x *= pow2_bits((f.ek[t] >> (8 * r)) & 255u);
        s[t][r] = x;
      }
    }
    if (valid[0] < 16 || valid[1] < 16) {  // the same in every lane: what lies behind the history is never used
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * g + r >= valid[t]) {
            s[t][r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
              for (int i = 0; i < (VB < 4 ? 1 : VB / 4); ++i) f.v[t][r][h][i] = 0;
          }
    }
    float top = m;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;  // a row with no finite score yet: all weights are 0
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= alpha;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < VE; ++j) o[h][j] *= alpha;
    float w[8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = __builtin_amdgcn_exp2f(s[t][r] - base);
        // 8- and 16-bit caches: the weights enter the product as bf16 (off by half a step, 2^-8 of the weight at most, as the output's own
        // rounding is), and the sum they are divided by is that of the rounded weights
        w[4 * t + r] = F32 ? x : (float) (__bf16) x;
        l += w[4 * t + r];
      }
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int j = 0; j < VE; ++j)
              o[h][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.v[t][r][h][j]), w[4 * t + r], o[h][j], 0, 0, 0);
    } else {
      if (DT == MI_DT_E4M3) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = pow2_bits((f.ev[t] >> (8 * r)) & 255u);
            w[4 * t + r] *= 4 * g + r < valid[t] ? e : 0.f;  // a dead position's exponent is anything
          }
      }
      uint4 pw;
      pw.x = pack_bf16(w[0], w[1]);
      pw.y = pack_bf16(w[2], w[3]);
      pw.z = pack_bf16(w[4], w[5]);
      pw.w = pack_bf16(w[6], w[7]);
      const bf8v pf = __builtin_bit_cast(bf8v, pw);
#pragma unroll
      for (int h = 0; h < VH; ++h) {
        if constexpr (DT == MI_DT_BF16) {
#pragma unroll
          for (int j = 0; j < VE; j += 2) {
            uint4 a, b;  // channels j and j + 1 of the lane's eight positions
            unsigned int* pa = &a.x;
            unsigned int* pb = &b.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned int x = f.v[k >> 1][2 * (k & 1)][h][j / 2], y = f.v[k >> 1][2 * (k & 1) + 1][h][j / 2];
              pa[k] = __builtin_amdgcn_perm(y, x, 0x05040100u);
              pb[k] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            }
            o[h][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), pf, o[h][j], 0, 0, 0);
            o[h][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, b), pf, o[h][j + 1], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int j = 0; j < VE; j += 2) {
            uint4 a, b;
            unsigned int* pa = &a.x;
            unsigned int* pb = &b.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned int x = f.v[k >> 1][2 * (k & 1)][h][j / 4], y = f.v[k >> 1][2 * (k & 1) + 1][h][j / 4];
              // bytes: channel j of both positions, then channel j + 1 of both
              const unsigned int z = __builtin_amdgcn_perm(y, x, (j & 2) ? 0x07030602u : 0x05010400u);
              pa[k] = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(z, 1.0f, false));
              pb[k] = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(z, 1.0f, true));
            }
            o[h][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), pf, o[h][j], 0, 0, 0);
            o[h][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, b), pf, o[h][j + 1], 0, 0, 0);
          }
        }
      }
    }
  }

  // lane (g, c) holds channels h * (D / VH) + (4 g + r) * VE + j of query row c: contiguous in (r, j)
  __device__ __forceinline__ void store(char* out_row, bool live, int g) {
    float sum = l + __shfl_xor(l, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (!live) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      char* dst = out_row + (h * (D / VH) + 4 * g * VE) * QE;
      float x[4 * VE];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; ++j) x[r * VE + j] = o[h][j][r] * inv;
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4 * VE; i += 4)
          *reinterpret_cast<float4*>(dst + i * 4) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * VE; i += 8)
          *reinterpret_cast<uint4*>(dst + i * 2) = make_uint4(pack_bf16(x[i], x[i + 1]), pack_bf16(x[i + 2], x[i + 3]),
                                                             pack_bf16(x[i + 4], x[i + 5]), pack_bf16(x[i + 6], x[i + 7]));
      }
    }
  }
};

// One wave per (sequence, cache head, tile of 16 query rows).
template <int DT, int D>
__global__ __launch_bounds__(256) void hist_attn_kernel(AttnArgs p) {
  typedef Wave<DT, D> W;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int64_t seg = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t pair = seg / p.n_rt;
  const int rt = (int) (seg - pair * p.n_rt);
  const int64_t b = pair / p.H;
  const int head = (int) (pair - b * p.H);
  if (b >= p.n_seqs) return;
  const int64_t room = (int64_t) p.width << p.page_shift;
  int64_t len = p.lengths[b];
  if (len > room) {
    if (lane == 0) report(p.err, MI_IDERR_RANGE);
    len = room;
  }
  const int row = rt * 16 + c;
  const bool live = row < p.rows;
  const int tok = live ? row / p.G : 0, qh = head * p.G + (live ? row % p.G : 0);
  W w;
  w.init(p.q + (b * p.q_seq + tok * p.q_tok + qh * p.q_head) * W::QE, live, g);
  const int32_t* table = p.table + b * p.ld_table;
  for (int64_t pos = 0; pos < len; pos += W::CHUNK) {
    int64_t rows[2];
    int valid[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t first = pos + 16 * t;
      int64_t page = first < len ? table[first >> p.page_shift] : 0;
      valid[t] = first >= len ? 0 : (len - first < 16 ? (int) (len - first) : 16);
      if (page < 0 || page >= p.n_pages) {
        if (lane == 0) report(p.err, MI_IDERR_RANGE);
        page = 0;
        valid[t] = 0;
      }
      rows[t] = (((page * p.H + head) * 2) << p.page_shift) + (first & ((1 << p.page_shift) - 1));
    }
    typename W::Fetched f;
    w.request(f, p, rows, g, c);
    w.step(f, p, valid, g, c);
  }
  w.store(p.out + (b * p.o_seq + tok * p.o_tok + qh * p.o_head) * W::QE, live, g);
}

template <int DT>
int launch_attn(const AttnArgs& p, int dim, hipStream_t s) {
  const dim3 grid((unsigned int) mi_cdiv(p.n_seqs * p.H * p.n_rt, 4));
  switch (dim) {
    case 32: hist_attn_kernel<DT, 32><<<grid, 256, 0, s>>>(p); break;
    case 64: hist_attn_kernel<DT, 64><<<grid, 256, 0, s>>>(p); break;
    case 128: hist_attn_kernel<DT, 128><<<grid, 256, 0, s>>>(p); break;
    default: hist_attn_kernel<DT, 256><<<grid, 256, 0, s>>>(p); break;
  }
  MI_LAUNCH_CHECK();
  return MI_OK;
}

// ------------------------------------------------------------------------------------------------ host checks
int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return (1 << s) == x ? s : -1;
}

int check_cache(const mi_hist_cache* c, const char* who) {
  MI_REQUIRE(c && c->kv, "%s: null cache", who);
  MI_REQUIRE(c->dtype == MI_DT_F32 || c->dtype == MI_DT_BF16 || c->dtype == MI_DT_E4M3, "%s: cache dtype %d", who, c->dtype);
  MI_REQUIRE((c->exps != nullptr) == (c->dtype == MI_DT_E4M3), "%s: exps go with e4m3 caches, and only with them", who);
  MI_REQUIRE(c->dim == 32 || c->dim == 64 || c->dim == 128 || c->dim == 256, "%s: dim %d is not 32, 64, 128 or 256", who, c->dim);
  MI_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && log2_of(c->page_size) > 0,
             "%s: page_size %d is not a power of two from 16 to 1024", who, c->page_size);
  MI_REQUIRE(c->n_heads >= 1 && c->n_heads <= 1024, "%s: n_heads %d outside 1..1024", who, c->n_heads);
  MI_REQUIRE(c->n_pages >= 1 && c->n_pages <= INT32_MAX, "%s: n_pages %lld outside 1..2^31-1", who, (long long) c->n_pages);
  MI_REQUIRE(((uintptr_t) c->kv & 15) == 0 && ((uintptr_t) c->exps & 15) == 0, "%s: the cache must be 16-byte aligned", who);
  return MI_OK;
}

int check_table(const int32_t* table, int64_t ld, int width, const int32_t* lengths, int64_t n_seqs, const char* who) {
  MI_REQUIRE(table && lengths, "%s: null page table or lengths", who);
  MI_REQUIRE(n_seqs >= 0 && n_seqs <= INT32_MAX, "%s: n_seqs %lld", who, (long long) n_seqs);
  MI_REQUIRE(width >= 1 && (ld >= width || n_seqs <= 1), "%s: page table width %d with row stride %lld", who, width, (long long) ld);
  return MI_OK;
}

// 16-byte accesses: base and strides whole multiples of 16 bytes
bool aligned16(const void* p, int elem, int64_t a, int64_t b, int64_t c = 0) {
  return (((uintptr_t) p | (uintptr_t) (a * elem) | (uintptr_t) (b * elem) | (uintptr_t) (c * elem)) & 15) == 0;
}

int rows_call(const char* who, bool read, const mi_hist_cache* cache, const void* k, const void* v, int dtype, int64_t k_row,
              int64_t k_head, int64_t v_row, int64_t v_head, int64_t n_rows, const int64_t* offsets, int64_t n_seqs,
              const int32_t* table, int64_t ld_table, int width, const int32_t* lengths, int32_t* err, void* stream) {
  if (int rc = check_cache(cache, who)) return rc;
  MI_REQUIRE(dtype == MI_DT_F32 || dtype == MI_DT_BF16, "%s: rows are f32 or bf16, not %d", who, dtype);
  MI_REQUIRE(n_rows >= 0, "%s: n_rows %lld", who, (long long) n_rows);
  if (n_rows == 0 || n_seqs == 0) return MI_OK;
  if (int rc = check_table(table, ld_table, width, lengths, n_seqs, who)) return rc;
  MI_REQUIRE(k && v, "%s: null rows", who);
  MI_REQUIRE(aligned16(k, dtype == MI_DT_F32 ? 4 : 2, k_row, k_head) && aligned16(v, dtype == MI_DT_F32 ? 4 : 2, v_row, v_head),
             "%s: rows must start on 16-byte boundaries", who);
  MI_REQUIRE(offsets || n_rows % n_seqs == 0, "%s: %lld rows do not divide among %lld sequences", who, (long long) n_rows,
             (long long) n_seqs);
  if (n_rows * 2 * cache->n_heads > (int64_t) INT32_MAX) {
    mi_set_error("%s: %lld rows of %d heads in one call (at most 2^31-1 rows of K and V)", who, (long long) n_rows, cache->n_heads);
    return MI_ERR_UNSUPPORTED;
  }
  RowArgs p = {};
  p.kv = (char*) cache->kv;
  p.exps = (uint8_t*) cache->exps;
  p.n_pages = cache->n_pages;
  p.H = cache->n_heads;
  p.page_shift = log2_of(cache->page_size);
  p.table = table;
  p.ld_table = ld_table;
  p.width = width;
  p.lengths = lengths;
  p.n_seqs = n_seqs;
  p.offsets = offsets;
  p.each = offsets ? 0 : n_rows / n_seqs;
  p.n_rows = n_rows;
  p.k = (const char*) k;
  p.v = (const char*) v;
  p.k_row = k_row;
  p.k_head = k_head;
  p.v_row = v_row;
  p.v_head = v_head;
  p.err = err;
  hipStream_t s = (hipStream_t) stream;
  const bool f32 = dtype == MI_DT_F32;
  if (read) {
    switch (cache->dtype) {
      case MI_DT_F32:
        return f32 ? launch_rows<MI_DT_F32, MI_DT_F32, true>(p, cache->dim, s) : launch_rows<MI_DT_F32, MI_DT_BF16, true>(p, cache->dim, s);
      case MI_DT_BF16:
        return f32 ? launch_rows<MI_DT_BF16, MI_DT_F32, true>(p, cache->dim, s) : launch_rows<MI_DT_BF16, MI_DT_BF16, true>(p, cache->dim, s);
      default:
        return f32 ? launch_rows<MI_DT_E4M3, MI_DT_F32, true>(p, cache->dim, s) : launch_rows<MI_DT_E4M3, MI_DT_BF16, true>(p, cache->dim, s);
    }
  }
  switch (cache->dtype) {
    case MI_DT_F32:
      return f32 ? launch_rows<MI_DT_F32, MI_DT_F32, false>(p, cache->dim, s) : launch_rows<MI_DT_F32, MI_DT_BF16, false>(p, cache->dim, s);
    case MI_DT_BF16:
      return f32 ? launch_rows<MI_DT_BF16, MI_DT_F32, false>(p, cache->dim, s) : launch_rows<MI_DT_BF16, MI_DT_BF16, false>(p, cache->dim, s);
    default:
      return f32 ? launch_rows<MI_DT_E4M3, MI_DT_F32, false>(p, cache->dim, s) : launch_rows<MI_DT_E4M3, MI_DT_BF16, false>(p, cache->dim, s);
  }
}

}  // namespace

extern "C" int mi_hist_write(const mi_hist_cache* cache, const void* k, const void* v, int dtype, int64_t k_row, int64_t k_head,
                             int64_t v_row, int64_t v_head, int64_t n_rows, const int64_t* offsets, int64_t n_seqs,
                             const int32_t* page_table, int64_t ld_table, int table_width, const int32_t* lengths,
                             int32_t* err, void* stream) {
  return rows_call("mi_hist_write", false, cache, k, v, dtype, k_row, k_head, v_row, v_head, n_rows, offsets, n_seqs,
                   page_table, ld_table, table_width, lengths, err, stream);
}

extern "C" int mi_hist_read(const mi_hist_cache* cache, void* k, void* v, int dtype, int64_t k_row, int64_t k_head,
                            int64_t v_row, int64_t v_head, int64_t n_rows, const int64_t* offsets, int64_t n_seqs,
                            const int32_t* page_table, int64_t ld_table, int table_width, const int32_t* lengths,
                            int32_t* err, void* stream) {
  return rows_call("mi_hist_read", true, cache, k, v, dtype, k_row, k_head, v_row, v_head, n_rows, offsets, n_seqs,
                   page_table, ld_table, table_width, lengths, err, stream);
}

extern "C" size_t mi_hist_attn_workspace_bytes(const mi_hist_cache* cache, int64_t n_seqs, int n_queries, int q_heads,
                                               int table_width) {
  (void) cache;
  (void) n_seqs;
  (void) n_queries;
  (void) q_heads;
  (void) table_width;
  return 0;
}

extern "C" int mi_hist_attn(const mi_hist_cache* cache, const void* q, int64_t q_seq, int64_t q_tok, int64_t q_head, int q_heads,
                            int n_queries, int64_t n_seqs, const int32_t* page_table, int64_t ld_table, int table_width,
                            const int32_t* lengths, float scale, void* out, int64_t out_seq, int64_t out_tok, int64_t out_head,
                            void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  (void) workspace;
  (void) workspace_bytes;
  if (int rc = check_cache(cache, "mi_hist_attn")) return rc;
  MI_REQUIRE(n_queries >= 0 && q_heads >= 1 && q_heads % cache->n_heads == 0,
             "mi_hist_attn: %d queries of %d heads over a cache of %d heads", n_queries, q_heads, cache->n_heads);
  if (n_seqs == 0 || n_queries == 0) return MI_OK;
  if (int rc = check_table(page_table, ld_table, table_width, lengths, n_seqs, "mi_hist_attn")) return rc;
  MI_REQUIRE(q && out, "mi_hist_attn: null q or out");
  const int qe = cache->dtype == MI_DT_F32 ? 4 : 2;
  MI_REQUIRE(aligned16(q, qe, q_seq, q_tok, q_head) && aligned16(out, qe, out_seq, out_tok, out_head),
             "mi_hist_attn: the rows of q and out must start on 16-byte boundaries");
  AttnArgs p = {};
  p.kv = (const char*) cache->kv;
  p.exps = (const uint8_t*) cache->exps;
  p.n_pages = cache->n_pages;
  p.H = cache->n_heads;
  p.page_shift = log2_of(cache->page_size);
  p.q = (const char*) q;
  p.q_seq = q_seq;
  p.q_tok = q_tok;
  p.q_head = q_head;
  p.out = (char*) out;
  p.o_seq = out_seq;
  p.o_tok = out_tok;
  p.o_head = out_head;
  p.G = q_heads / cache->n_heads;
  const int64_t rows = (int64_t) n_queries * p.G;
  MI_REQUIRE(rows <= 65536, "mi_hist_attn: %lld query rows per cache head (at most 65536)", (long long) rows);
  p.rows = (int) rows;
  p.n_rt = (int) mi_cdiv(rows, 16);
  p.table = page_table;
  p.ld_table = ld_table;
  p.width = table_width;
  p.lengths = lengths;
  p.n_seqs = n_seqs;
  p.scale = scale * 1.44269504088896340736f;
  p.err = err;
  if (n_seqs * p.H * p.n_rt > (int64_t) INT32_MAX) {
    mi_set_error("mi_hist_attn: %lld sequences x %d heads x %d row tiles in one call", (long long) n_seqs, p.H, p.n_rt);
    return MI_ERR_UNSUPPORTED;
  }
  hipStream_t s = (hipStream_t) stream;
  switch (cache->dtype) {
    case MI_DT_F32: return launch_attn<MI_DT_F32>(p, cache->dim, s);
    case MI_DT_BF16: return launch_attn<MI_DT_BF16>(p, cache->dim, s);
    default: return launch_attn<MI_DT_E4M3>(p, cache->dim, s);
  }
}
