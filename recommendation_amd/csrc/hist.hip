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
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef unsigned int u2v __attribute__((ext_vector_type(2)));

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

// over the lanes l, l ^ 16, l ^ 32, l ^ 48: the swaps leave both halves of a pair in both results
__device__ __forceinline__ float max_over_g(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Read-only memory at a wave-uniform address, through the scalar cache (the compiler cannot know that nothing in the
// launch writes it, and a vector load in its place would have to wait for every load in flight).
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
  return *(const __attribute__((address_space(4))) T*) (p);
}

// Loads and stores past the caches (STREAM) or through them.  More than the last-level cache holds gains from going past
// it, less loses what an earlier launch left there (measured at each launch below).
constexpr int64_t LAST_LEVEL_BYTES = 256ll << 20;
template <bool STREAM, typename T>
__device__ __forceinline__ T load_of(const T* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool STREAM, typename T>
__device__ __forceinline__ void store_of(T* p, T x) {
  if constexpr (STREAM) __builtin_nontemporal_store(x, p);
  else *p = x;
}

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

// Where row i of the call lives: index of its K row of head 0 in the cache, or one of the two below.  [b0, b1]: the
// sequences it can belong to.
constexpr int64_t NOWHERE = -1;  // in front of position 0, or a bad page
constexpr int64_t UNOWNED = -2;  // no sequence's row
__device__ __forceinline__ int64_t find_place(const RowArgs& p, int64_t i, int64_t b0, int64_t b1) {
  int64_t b, last;
  if (p.offsets) {
    while (b0 < b1) {  // the last b with offsets[b] <= i
      const int64_t mid = (b0 + b1 + 1) >> 1;
      if (p.offsets[mid] <= i) b0 = mid; else b1 = mid - 1;
    }
    b = b0;
    if (b < 0 || b >= p.n_seqs) return UNOWNED;
    last = p.offsets[b + 1];
  } else {
    b = (int64_t) ((uint32_t) i / (uint32_t) p.each);
    last = (b + 1) * p.each;
  }
  const int64_t len = p.lengths[b];
  const int64_t pos = len - (last - i);
  if (pos < 0 || pos >= len) return NOWHERE;
  const int64_t pi = pos >> p.page_shift;
  const int64_t page = pi < p.width ? p.table[b * p.ld_table + pi] : -1;
  if (page < 0 || page >= p.n_pages) {
    report(p.err, MI_IDERR_RANGE);
    return NOWHERE;
  }
  return ((page * p.H * 2) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

struct Eight {
  float x[8];
};
// Eight values of a row as they lie in memory.  A lane's eight are channels 8c .. 8c+7, or with SPLIT 4c .. 4c+3 of each
// half of the row: where a side holds f32, 16 bytes a lane then make whole lines of a row with every instruction.
template <int DT>
struct Raw8 {
  unsigned int w[Elem<DT>::BYTES * 2];
};
template <int WORDS, bool STREAM>
__device__ __forceinline__ void load_words(unsigned int* w, const char* p) {
  if constexpr (WORDS >= 4) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const u4v a = load_of<STREAM>(reinterpret_cast<const u4v*>(p) + i / 4);
      w[i] = a[0]; w[i + 1] = a[1]; w[i + 2] = a[2]; w[i + 3] = a[3];
    }
  } else if constexpr (WORDS == 2) {
    const u2v a = load_of<STREAM>(reinterpret_cast<const u2v*>(p));
    w[0] = a[0]; w[1] = a[1];
  } else {
    w[0] = load_of<STREAM>(reinterpret_cast<const unsigned int*>(p));
  }
}
template <int WORDS, bool STREAM>
__device__ __forceinline__ void store_words(char* p, const unsigned int* w) {
  if constexpr (WORDS >= 4) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) store_of<STREAM>(reinterpret_cast<u4v*>(p) + i / 4, u4v{w[i], w[i + 1], w[i + 2], w[i + 3]});
  } else if constexpr (WORDS == 2) {
    store_of<STREAM>(reinterpret_cast<u2v*>(p), u2v{w[0], w[1]});
  } else {
    store_of<STREAM>(reinterpret_cast<unsigned int*>(p), w[0]);
  }
}
template <int DT, int D, bool SPLIT, bool STREAM>
__device__ __forceinline__ Raw8<DT> load8(const char* row, int c) {
  constexpr int E = Elem<DT>::BYTES;
  Raw8<DT> r;
  if constexpr (SPLIT) {
    load_words<E, STREAM>(r.w, row + c * 4 * E);
    load_words<E, STREAM>(r.w + E, row + (D / 2 + c * 4) * E);
  } else {
    load_words<2 * E, STREAM>(r.w, row + c * 8 * E);
  }
  return r;
}
template <int DT, int D, bool SPLIT, bool STREAM>
__device__ __forceinline__ void store8(char* row, int c, const Raw8<DT>& r) {
  constexpr int E = Elem<DT>::BYTES;
  if constexpr (SPLIT) {
    store_words<E, STREAM>(row + c * 4 * E, r.w);
    store_words<E, STREAM>(row + (D / 2 + c * 4) * E, r.w + E);
  } else {
    store_words<2 * E, STREAM>(row + c * 8 * E, r.w);
  }
}
template <int DT>
__device__ __forceinline__ Eight widen8(const Raw8<DT>& a) {
  Eight r;
#pragma unroll
  for (int i = 0; i < (DT == MI_DT_F32 ? 8 : 4); ++i) {
    if constexpr (DT == MI_DT_F32) {
      r.x[i] = __uint_as_float(a.w[i]);
    } else if constexpr (DT == MI_DT_BF16) {
      r.x[2 * i] = __uint_as_float(a.w[i] << 16);
      r.x[2 * i + 1] = __uint_as_float(a.w[i] & 0xffff0000u);
    } else {  // exact: 4 significant bits
      const bf2v c = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a.w[i / 2], 1.0f, true)
                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a.w[i / 2], 1.0f, false);
      r.x[2 * i] = (float) c[0];
      r.x[2 * i + 1] = (float) c[1];
    }
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
__device__ __forceinline__ Raw8<DT> round8(const Eight& e) {  // f32, bf16
  Raw8<DT> r;
#pragma unroll
  for (int i = 0; i < Elem<DT>::BYTES * 2; ++i)
    r.w[i] = DT == MI_DT_F32 ? __float_as_uint(e.x[i]) : pack_bf16(e.x[(2 * i) & 7], e.x[(2 * i + 1) & 7]);
  return r;
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
__device__ __forceinline__ Raw8<MI_DT_E4M3> quantise8(const Eight& e, unsigned int exponent) {
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
  return Raw8<MI_DT_E4M3>{{(unsigned int) lo, (unsigned int) hi}};
}
// A wave moves `tokens` (a power of two, up to 64) consecutive rows of the call.  Lane i first finds the place of token
// i: the chain of dependent loads (sequence, length, page) is walked once for all of them.  Then D / 8 lanes move one
// (token, K or V, head) row, tokens fastest, ROW_BATCH of them requested together.  READ: the cache is the source and
// k, v the destination.
constexpr int ROW_BATCH = 4;

template <int CT, int IT, int D, bool READ, bool STREAM>
__global__ __launch_bounds__(256) void hist_rows_kernel(RowArgs p, int token_shift) {
  constexpr int LPR = D / 8, GROUPS = 64 / LPR;
  constexpr int CE = Elem<CT>::BYTES, IE = Elem<IT>::BYTES;
  constexpr int FROM = READ ? CT : IT;
  constexpr bool SPLIT = CT == MI_DT_F32 || IT == MI_DT_F32;
  const int lane = threadIdx.x & 63, c = lane % LPR;
  const int64_t wave = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t0 = wave << token_shift;
  if (t0 >= p.n_rows) return;
  const int n_tok = p.n_rows - t0 < (1 << token_shift) ? (int) (p.n_rows - t0) : 1 << token_shift;
  const int n_move = (2 * p.H) << token_shift;  // rows to move, those of tokens >= n_tok among them

  struct Row {
    bool live;
    int token, part, head;
  };
  auto row_of = [&](int i) {
    const int r = i * GROUPS + lane / LPR;
    Row x;
    x.token = r & ((1 << token_shift) - 1);
    const int hp = r >> token_shift;
    x.live = r < n_move && x.token < n_tok;
    x.part = hp >= p.H ? 1 : 0;
    x.head = hp - x.part * p.H;
    return x;
  };
  auto io = [&](const Row& x) {
    return const_cast<char*>(x.part ? p.v + ((t0 + x.token) * p.v_row + x.head * p.v_head) * IE
                                    : p.k + ((t0 + x.token) * p.k_row + x.head * p.k_head) * IE);
  };
  Raw8<FROM> raw[ROW_BATCH];
  auto load_inputs = [&](int i0) {
#pragma unroll
    for (int u = 0; u < ROW_BATCH; ++u) {
      const Row x = row_of(i0 + u);
      if (x.live) raw[u] = load8<FROM, D, SPLIT, STREAM>(io(x), c);
      else raw[u] = Raw8<FROM>{};
    }
  };
  if (!READ) load_inputs(0);  // they depend on nothing

  int64_t b0 = 0, b1 = 0;
  if (p.offsets) {
    b0 = wave_upper_bound(p.offsets, p.n_seqs + 1, t0, lane) - 1;
    b1 = n_tok > 1 ? wave_upper_bound(p.offsets, p.n_seqs + 1, t0 + n_tok - 1, lane) - 1 : b0;
  }
  // lanes without a token repeat the last one's search
  const int64_t mine = find_place(p, t0 + (lane < n_tok ? lane : n_tok - 1), b0, b1);

  const int n_iter = (n_move + GROUPS - 1) / GROUPS;
  for (int i0 = 0; i0 < n_iter; i0 += ROW_BATCH) {
    int64_t at[ROW_BATCH];
    unsigned int exponent[ROW_BATCH];
    if (!READ && i0) load_inputs(i0);
#pragma unroll
    for (int u = 0; u < ROW_BATCH; ++u) {
      const Row x = row_of(i0 + u);
      const int64_t base = __shfl(mine, x.token, 64);
      at[u] = !x.live ? UNOWNED : base < 0 ? base : base + ((int64_t) (x.head * 2 + x.part) << p.page_shift);
      exponent[u] = 0;
      if (READ) {
        raw[u] = Raw8<FROM>{};
        if (at[u] >= 0) {
          raw[u] = load8<FROM, D, SPLIT, STREAM>(p.kv + at[u] * D * CE, c);
          if (CT == MI_DT_E4M3) exponent[u] = p.exps[at[u]];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < ROW_BATCH; ++u) {
      Eight y = widen8<FROM>(raw[u]);
      if constexpr (READ) {
        if (CT == MI_DT_E4M3) {
          const float s = pow2_bits(exponent[u]);
#pragma unroll
          for (int e = 0; e < 8; ++e) y.x[e] *= s;
        }
        if (at[u] != UNOWNED) store8<IT, D, SPLIT, STREAM>(io(row_of(i0 + u)), c, round8<IT>(y));
      } else {
        float top = 0.f;
        if (CT == MI_DT_E4M3) {  // every lane takes part in the exchange
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_abs(y.x[e]));
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        }
        if (at[u] >= 0) {
          char* dst = p.kv + at[u] * D * CE;
          if constexpr (CT == MI_DT_E4M3) {
            const unsigned int e = row_exponent(top);
            store8<CT, D, SPLIT, false>(dst, c, quantise8(y, e));
            if (c == 0) p.exps[at[u]] = (uint8_t) e;
          } else {
            store8<CT, D, SPLIT, false>(dst, c, round8<CT>(y));
          }
        }
      }
    }
  }
}

template <int CT, int IT, bool READ>
int launch_rows(const RowArgs& p, int dim, hipStream_t s) {
  // at least the rows of one instruction; beyond that up to four tokens a wave as long as there are four waves for every
  // SIMD.  f32 rows leave a wave token by token: 8 KB at a time then (65 k rows of 8 x 128 read back from e4m3 in f32: 134 us
  // so, 152 with four tokens a wave; 250 k rows in bf16: 286 token by token, 281 with four; 65 k written from bf16: 106, 91).
  const int groups = 64 / (dim / 8);
  int shift = 0;
  while ((2 * p.H) << shift < groups && shift < 6) ++shift;
  while (shift < (READ && IT == MI_DT_F32 ? 0 : 2) && (p.n_rows >> (shift + 1)) >= 4096) ++shift;
  while (shift < 6 && (p.n_rows >> shift) > (1 << 25)) ++shift;  // a launch holds less than 2^32 threads
  const dim3 grid((unsigned int) mi_cdiv(p.n_rows, 4ll << shift));
  const bool stream = p.n_rows * 2 * p.H * dim * (Elem<CT>::BYTES + Elem<IT>::BYTES) > LAST_LEVEL_BYTES;
#define MI_HIST_ROWS(D)                                                                            \
  if (stream) hist_rows_kernel<CT, IT, D, READ, true><<<grid, 256, 0, s>>>(p, shift);              \
  else hist_rows_kernel<CT, IT, D, READ, false><<<grid, 256, 0, s>>>(p, shift)
  switch (dim) {
    case 32: MI_HIST_ROWS(32); break;
    case 64: MI_HIST_ROWS(64); break;
    case 128: MI_HIST_ROWS(128); break;
    default: MI_HIST_ROWS(256); break;
  }
#undef MI_HIST_ROWS
  MI_LAUNCH_CHECK();
  return MI_OK;
}

// ------------------------------------------------------------------------------------------------ attention
struct AttnArgs {
  const char* kv;
  const uint8_t* exps;
  int n_pages;
  int H, page_shift;
  const char* q;
  int64_t q_seq, q_tok, q_head;  // strides in elements
  char* out;
  int64_t o_seq, o_tok, o_head;
  int G, rows;                   // query heads per cache head; n_q * G query rows per cache head
  const int32_t* table;
  int64_t ld_table;
  int width;
  const int32_t* lengths;
  int64_t n_seqs;
  float scale;                   // of the scores, times log2(e)
  int32_t* err;
};

// Waves on a SIMD, asked of the compiler (registers) and counted on when the work is cut.  256 channels run one: two would fit
// in 8 bits (215-226 registers), would spill 4-25 in 16 bits and need 480 and more in f32.  Calls over long histories do not
// feel it (see Wave); calls where a workgroup has a history of up to a thousand positions and lengths differ do: 547 MB in
// bf16 171 us, the same bytes at 128 channels 114.
constexpr int split_waves(bool f32, int dim, int RT) {
  return dim == 256 ? 1 : dim == 128 ? (f32 ? 3 - RT : 4 - RT) : dim == 64 ? (f32 ? 3 : 4) - (RT - 1) : 4 - (RT - 1);
}

// One wave's running state for RT tiles of 16 query rows of one cache head: o = sum_j 2^(s_j - m) v_j, l = sum_j 2^(s_j - m).
//
// Both products are matrix instructions whose operands come straight from memory.  Scores are formed transposed,
// S^T = K Q^T (rows: 16 cached positions; columns: query rows): lane (g = lane / 16, c = lane % 16) then holds the
// scores of query row c for positions 4g .. 4g+3 of a tile, which is what the second product, O^T = V^T P^T, wants as
// its right operand if its reduction index is read as "positions 4g..4g+3 of tile 0, then of tile 1".  Its left
// operand takes output channels j of 16 lanes' 16-byte pieces of a V row, whatever those channels are called.  So no
// score, probability or value crosses lanes; only the row maximum and sum do (over the four g).
//
// What bounds it: the cache's bytes (1 to 16 query rows a head: 6.1-6.7 TB/s in calls that read 0.7-3.2 GB, at 128 and 256
// channels; 3.1-4.1 in calls that read 80-310 MB), and from two row tiles on the vector instructions (e4m3, 64 rows: two waves
// a SIMD issue them in 67 % of the cycles).
template <int DT, int D, int RT, bool STREAM>
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
  static constexpr float SLACK = 8.f;

  f4v o[RT][VH][VE];
  // l: in 8 and 16 bits a column of the second product whose "values" are all 1, so that every lane of a row holds the
  // whole sum; in f32, where that product takes four times as long, the lane's own positions until close()
  float m[RT];
  f4v l[RT];
  bf8v qf[RT][F32 ? 1 : NS];
  f4v qv[RT][F32 ? KL : 1];

  // channel of element 0 of this lane's query fragment of step s
  static __device__ __forceinline__ int q_channel(int s, int g) {
    if (DT == MI_DT_E4M3 && KN == 16) return (s >> 1) * 64 + g * 16 + (s & 1) * 8;
    return s * 32 + g * 8;
  }

  __device__ __forceinline__ void init(int t, const char* q_row, bool live, int g) {
    m[t] = -INFINITY;
    l[t] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < VE; ++j) o[t][h][j] = f4v{0.f, 0.f, 0.f, 0.f};
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < KL; ++s) {
        const f4v x = *reinterpret_cast<const f4v*>(q_row + (s * 16 + g * 4) * 4);
        qv[t][s] = live ? x : f4v{0.f, 0.f, 0.f, 0.f};
      }
    } else {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const uint4 x = *reinterpret_cast<const uint4*>(q_row + q_channel(s, g) * 2);
        qf[t][s] = __builtin_bit_cast(bf8v, live ? x : make_uint4(0, 0, 0, 0));
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
      const u4v x = load_of<STREAM>(reinterpret_cast<const u4v*>(src));
      dst[0] = x[0]; dst[1] = x[1]; dst[2] = x[2]; dst[3] = x[3];
    } else if constexpr (BYTES == 8) {
      const u2v x = load_of<STREAM>(reinterpret_cast<const u2v*>(src));
      dst[0] = x[0]; dst[1] = x[1];
    } else if constexpr (BYTES == 4) {
      dst[0] = load_of<STREAM>(reinterpret_cast<const unsigned int*>(src));
    } else {
      dst[0] = load_of<STREAM>(reinterpret_cast<const unsigned short*>(src));
    }
  }

  // What is known of a chunk ahead of its loads, all of it wave-uniform: the page ids of its two tiles ...
  struct Ahead {
    unsigned int first[2];  // position of each tile; a tile behind the end stands where the last one does
    int valid[2];           // live positions (0: behind the end)
    int32_t id[2];
  };
  // ... and, once those have arrived, the tiles' first K rows in the cache.
  struct Where {
    int64_t rows[2];
    int valid[2];
  };
  static __device__ __forceinline__ Ahead look(const AttnArgs& p, const int32_t* table, unsigned int pos, unsigned int end) {
    Ahead a;
    const unsigned int last = (end - 1) & ~15u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned int first = pos + 16 * t;
      a.valid[t] = first >= end ? 0 : (end - first < 16 ? (int) (end - first) : 16);
      a.first[t] = first < last ? first : last;
      a.id[t] = scalar_load(table + (a.first[t] >> p.page_shift));
    }
    return a;
  }
  // a tile on a bad page counts as dead and stands on page 0
  static __device__ __forceinline__ Where locate(const AttnArgs& p, const Ahead& a, int head, int lane) {
    Where w;
    bool bad = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool ok = (unsigned int) a.id[t] < (unsigned int) p.n_pages;
      bad |= !ok && a.valid[t] > 0;
      const unsigned int page = ok ? (unsigned int) a.id[t] : 0u;
      w.valid[t] = ok ? a.valid[t] : 0;
      w.rows[t] = (int64_t) ((((uint64_t) page * (unsigned int) p.H + (unsigned int) head) << (p.page_shift + 1)) +
                             (a.first[t] & ((1u << p.page_shift) - 1)));
    }
    if (bad && lane == 0) report(p.err, MI_IDERR_RANGE);
    return w;
  }
  // base uniform, 32-bit offset per lane
  static __device__ __forceinline__ void request_k(Fetched& f, const AttnArgs& p, const Where& w, int lane) {
    const unsigned int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* kb = p.kv + w.rows[t] * (D * E);
      const unsigned int most = w.valid[t] > 0 ? w.valid[t] - 1 : 0;  // behind the end the last row again
      const unsigned int row = c < most ? c : most;
#pragma unroll
      for (int s = 0; s < KL; ++s) fetch<KB>(f.k[t][s], kb + s * (KB * 4) + (row * (D * E) + g * KB));
      if (DT == MI_DT_E4M3) f.ek[t] = *reinterpret_cast<const unsigned int*>(p.exps + w.rows[t] + 4 * g);
    }
    __builtin_amdgcn_sched_barrier(0);  // the loads stay in front of the work they are to overlap
  }
  static __device__ __forceinline__ void request_v(Fetched& f, const AttnArgs& p, const Where& w, int lane) {
    const unsigned int g = lane >> 4, c = lane & 15;
    const int page_size = 1 << p.page_shift;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* vb = p.kv + (w.rows[t] + page_size) * (D * E);  // V lies page_size rows behind K
      const unsigned int most = w.valid[t] > 0 ? w.valid[t] - 1 : 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned int row = 4 * g + r < most ? 4 * g + r : most;
#pragma unroll
        for (int h = 0; h < VH; ++h) fetch<VB>(f.v[t][r][h], vb + h * (VB * 16) + (row * (D * E) + c * VB));
      }
      if (DT == MI_DT_E4M3) f.ev[t] = *reinterpret_cast<const unsigned int*>(p.exps + w.rows[t] + page_size + 4 * g);
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // All chunks pos, pos + stride, ... < end.  A chunk's page ids are requested two steps ahead, its K while the values
  // of the chunk before are summed, its V while its own scores are formed: one set of registers, and loads in flight all
  // the time.  The last chunk stands behind the loop: loads that only some steps issue would make every step wait for all.
  __device__ __forceinline__ void walk(const AttnArgs& p, const int32_t* table, unsigned int pos, unsigned int end,
                                       unsigned int stride, int head, int lane) {
    if (pos >= end) return;
    Fetched f;
    f4v s[RT][2];
    Where at = locate(p, look(p, table, pos, end), head, lane);
    request_k(f, p, at, lane);
    request_v(f, p, at, lane);
    Ahead ahead = look(p, table, pos + stride, end);
    for (; pos + stride < end; pos += stride) {
      const Where next = locate(p, ahead, head, lane);
      ahead = look(p, table, pos + 2 * stride, end);
      scores(s, f, p);
      request_k(f, p, next, lane);
      weigh(s, f, at, lane);
      request_v(f, p, next, lane);
      at = next;
    }
    scores(s, f, p);
    weigh(s, f, at, lane);
  }

  static __device__ __forceinline__ bf8v widen(unsigned int lo, unsigned int hi) {  // 8 e4m3 codes, exactly
    uint4 w;
    w.x = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w.y = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w.z = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w.w = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return __builtin_bit_cast(bf8v, w);
  }

  // scores of one chunk, times log2(e)
  __device__ __forceinline__ void scores(f4v (&s)[RT][2], const Fetched& f, const AttnArgs& p) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < RT; ++i) s[i][t] = f4v{0.f, 0.f, 0.f, 0.f};
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < KL; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < RT; ++i)
              s[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.k[t][k][e]), qv[i][k][e], s[i][t], 0, 0, 0);
      } else if constexpr (DT == MI_DT_BF16) {
#pragma unroll
        for (int k = 0; k < KL; ++k) {
          const uint4 w = make_uint4(f.k[t][k][0], f.k[t][k][1], f.k[t][k][2], f.k[t][k][3]);
#pragma unroll
          for (int i = 0; i < RT; ++i)
            s[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, w), qf[i][k], s[i][t], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KL; ++k)
#pragma unroll
          for (int u = 0; u < KB / 8; ++u) {
            const bf8v w = widen(f.k[t][k][2 * u], f.k[t][k][2 * u + 1]);
#pragma unroll
            for (int i = 0; i < RT; ++i)
              s[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, qf[i][k * (KB / 8) + u], s[i][t], 0, 0, 0);
          }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (scale first: a small power of two times it could leave the normal range)
        const float e = DT == MI_DT_E4M3 ? pow2_bits((f.ek[t] >> (8 * r)) & 255u) : 1.f;
#pragma unroll
        for (int i = 0; i < RT; ++i) s[i][t][r] = DT == MI_DT_E4M3 ? s[i][t][r] * p.scale * e : s[i][t][r] * p.scale;
      }
    }
  }

  // softmax step and weighted sum of one chunk
  __device__ __forceinline__ void weigh(f4v (&s)[RT][2], Fetched& f, const Where& at, int lane) {
    const int g = lane >> 4;
    if (at.valid[0] < 16 || at.valid[1] < 16) {  // the same in every lane: what lies behind the history is never used
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * g + r >= at.valid[t]) {
#pragma unroll
            for (int i = 0; i < RT; ++i) s[i][t][r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
              for (int e = 0; e < (VB < 4 ? 1 : VB / 4); ++e) f.v[t][r][h][e] = 0;
            if (DT == MI_DT_E4M3) f.ev[t] &= ~(255u << (8 * r));  // a dead position's exponent is anything
          }
    }
    float w[RT][8];
    bf8v pf[RT];
    const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);  // bf16
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float top = m[i];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][t][r]);
      top = max_over_g(top);
      // m is a score that the row's weights are taken against, at most SLACK below its maximum so far: most chunks
      // then leave the sums as they are, at weights of up to 2^SLACK
      if (__any(top > m[i] + SLACK)) {
        const float up = top > m[i] + SLACK ? top : m[i];
        const float alpha = up == m[i] ? 1.f : __builtin_amdgcn_exp2f(m[i] - up);
        m[i] = up;
        l[i] *= alpha;
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
          for (int j = 0; j < VE; ++j) o[i][h][j] *= alpha;
      }
      const float base = m[i] == -INFINITY ? 0.f : m[i];  // no finite score yet: all weights are 0
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[i][4 * t + r] = __builtin_amdgcn_exp2f(s[i][t][r] - base);
      // 8- and 16-bit caches: the weights enter the product as bf16 (off by half a step, 2^-8 of the weight at most, as
      // the output's own rounding is), and the sum they are divided by is that of the rounded weights.  In 8 bits they
      // then carry the value row's power of two, which changes no bit of them - but their sum does not: a row of zeros
      // has the power 2^-126 and its weight all the same.
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) l[i][0] += w[i][e];
      } else {
        u4v pw;
#pragma unroll
        for (int e = 0; e < 4; ++e) pw[e] = pack_bf16(w[i][2 * e], w[i][2 * e + 1]);
        l[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, ones), __builtin_bit_cast(bf8v, pw), l[i], 0, 0, 0);
        if constexpr (DT == MI_DT_E4M3) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            pw[e] = pack_bf16(w[i][2 * e] * pow2_bits((f.ev[e >> 1] >> (16 * (e & 1))) & 255u),
                              w[i][2 * e + 1] * pow2_bits((f.ev[e >> 1] >> (16 * (e & 1) + 8)) & 255u));
        }
        pf[i] = __builtin_bit_cast(bf8v, pw);
      }
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
#pragma unroll
              for (int i = 0; i < RT; ++i)
                o[i][h][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.v[t][r][h][j]), w[i][4 * t + r],
                                                                  o[i][h][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int j = 0; j < VE; j += 2) {
          uint4 a, b;  // channels j and j + 1 of the lane's eight positions
          unsigned int* pa = &a.x;
          unsigned int* pb = &b.x;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (DT == MI_DT_BF16) {
              const unsigned int x = f.v[k >> 1][2 * (k & 1)][h][j / 2], y = f.v[k >> 1][2 * (k & 1) + 1][h][j / 2];
              pa[k] = __builtin_amdgcn_perm(y, x, 0x05040100u);
              pb[k] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            } else {
              const unsigned int x = f.v[k >> 1][2 * (k & 1)][h][j / 4], y = f.v[k >> 1][2 * (k & 1) + 1][h][j / 4];
              // bytes: channel j of both positions, then channel j + 1 of both
              const unsigned int z = __builtin_amdgcn_perm(y, x, (j & 2) ? 0x07030602u : 0x05010400u);
              pa[k] = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(z, 1.0f, false));
              pb[k] = __builtin_bit_cast(unsigned int, (bf2v) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(z, 1.0f, true));
            }
          }
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            o[i][h][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), pf[i], o[i][h][j], 0, 0, 0);
            o[i][h][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, b), pf[i], o[i][h][j + 1], 0, 0, 0);
          }
        }
    }
  }

  // f32: the four g hold the sums of their own positions
  __device__ __forceinline__ void close() {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        l[i][0] += __shfl_xor(l[i][0], 16, 64);
        l[i][0] += __shfl_xor(l[i][0], 32, 64);
      }
    }
  }

  // lane (g, c) holds channels h * (D / VH) + (4 g + r) * VE + j of query row c: contiguous in (r, j)
  __device__ __forceinline__ void store(int t, char* out_row, int g) {
    const float inv = l[t][0] == 0.f ? 0.f : 1.f / l[t][0];
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      char* dst = out_row + (h * (D / VH) + 4 * g * VE) * QE;
      float x[4 * VE];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; ++j) x[r * VE + j] = o[t][h][j][r] * inv;
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

  // unnormalised, in f32, for the joining launch: a row's D sums as the registers hold them (channel_of), and m, l
  __device__ __forceinline__ void store_part(int t, float* part_row, float2* ml, int g) {
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < VE; ++j) *reinterpret_cast<f4v*>(part_row + (h * VE + j) * 16 + g * 4) = o[t][h][j];
    if (g == 0) *ml = make_float2(m[t], l[t][0]);
  }
  // channel of element r of the 16-byte piece `piece` of such a row
  static __device__ __forceinline__ int channel_of(int piece, int r) {
    const int i = piece >> 2, g = piece & 3;
    return (i / VE) * (D / VH) + (4 * g + r) * VE + i % VE;
  }
};

// The two halves of a pair of states, lane by lane the same rows and channels.
struct Fold {
  float a, b, m;
};
__device__ __forceinline__ Fold fold_of(float m1, float m2) {
  const float top = fmaxf(m1, m2), base = top == -INFINITY ? 0.f : top;
  return Fold{__builtin_amdgcn_exp2f(m1 - base), __builtin_amdgcn_exp2f(m2 - base), top};
}

// query row r of a cache head: token r / G, head r % G of the group
template <int QE>
__device__ __forceinline__ const char* q_row_of(const AttnArgs& p, int64_t b, int head, int row, bool live) {
  const int tok = live ? row / p.G : 0, qh = head * p.G + (live ? row % p.G : 0);
  return p.q + (b * p.q_seq + tok * p.q_tok + qh * p.q_head) * QE;
}
template <int QE>
__device__ __forceinline__ char* out_row_of(const AttnArgs& p, int64_t b, int head, int row) {
  return p.out + (b * p.o_seq + (row / p.G) * p.o_tok + (head * p.G + row % p.G) * p.o_head) * QE;
}

__device__ __forceinline__ int64_t clamped_length(const AttnArgs& p, int32_t len, bool say) {
  const int64_t room = (int64_t) p.width << p.page_shift;
  if (len > room && say) report(p.err, MI_IDERR_RANGE);
  return len > room ? room : (len < 0 ? 0 : len);
}

// Short histories: one wave per (sequence, cache head, RT tiles of 16 query rows).  Through the caches whatever the pool's
// size: the waves of further row tiles come right behind (35 rows over up to 27 positions: 123 us so, 130 past them; one row
// over up to 111: 62 and 64; three rows over 22-44: 102 and 100).
template <int DT, int D, int RT>
__global__ __launch_bounds__(256, split_waves(DT == MI_DT_F32, D, RT)) void hist_attn_short_kernel(AttnArgs p, int n_tiles) {
  typedef Wave<DT, D, RT, false> W;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const unsigned int seg = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned int pair = seg / (unsigned int) n_tiles;
  const int row0 = (int) (seg - pair * n_tiles) * 16 * RT;
  const int64_t b = pair / (unsigned int) p.H;
  const int head = (int) (pair - (unsigned int) b * p.H);
  if (b >= p.n_seqs) return;
  const int64_t len = clamped_length(p, scalar_load(p.lengths + b), lane == 0);
  W w;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = row0 + t * 16 + c;
    w.init(t, q_row_of<W::QE>(p, b, head, row, row < p.rows), row < p.rows, g);
  }
  w.walk(p, p.table + b * p.ld_table, 0, (unsigned int) len, W::CHUNK, head, lane);
  w.close();
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = row0 + t * 16 + c;
    if (row < p.rows) w.store(t, out_row_of<W::QE>(p, b, head, row), g);
  }
}

// A workgroup's walk over positions first .. end-1 of one (sequence, cache head, group of NR * 16 * RT query rows): NR row
// tiles side by side, the other waves share the positions (32 each in turn) and fold their sums in LDS, halves onto halves,
// lane by lane the same rows and channels.  Afterwards the first NR waves hold the sums.
template <typename W, int RT>
struct FoldLds {
  f4v o[2][RT * W::VH * W::VE][64];
  float2 ml[2][RT][64];
};
template <typename W, int RT>
__device__ __forceinline__ void walk_shared(W& w, FoldLds<W, RT>& lds, const AttnArgs& p, int NR, int64_t b, int head, int row0,
                                            unsigned int first, unsigned int end, int wave, int lane) {
  const int g = lane >> 4, c = lane & 15, rt = wave % NR, ci = wave / NR, CI = 4 / NR;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = row0 + t * 16 + c;
    w.init(t, q_row_of<W::QE>(p, b, head, row, row < p.rows), row < p.rows, g);
  }
  if (row0 < p.rows) w.walk(p, p.table + b * p.ld_table, first + ci * W::CHUNK, end, CI * W::CHUNK, head, lane);
  w.close();
  for (int half = CI >> 1; half > 0; half >>= 1) {
    const int slot = (ci - half) * NR + rt;  // < 2: half * NR <= 2
    if (ci >= half && ci < 2 * half) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        lds.ml[slot][t][lane] = make_float2(w.m[t], w.l[t][0]);
#pragma unroll
        for (int i = 0; i < W::VH * W::VE; ++i) lds.o[slot][t * W::VH * W::VE + i][lane] = w.o[t][i / W::VE][i % W::VE];
      }
    }
    __syncthreads();
    if (ci < half) {
      const int from = ci * NR + rt;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float2 ml = lds.ml[from][t][lane];
        const Fold k = fold_of(w.m[t], ml.x);
        w.m[t] = k.m;
        w.l[t][0] = w.l[t][0] * k.a + ml.y * k.b;
#pragma unroll
        for (int i = 0; i < W::VH * W::VE; ++i)
          w.o[t][i / W::VE][i % W::VE] = w.o[t][i / W::VE][i % W::VE] * k.a + lds.o[from][t * W::VH * W::VE + i][lane] * k.b;
      }
    }
    __syncthreads();
  }
}

// Histories of a thousand positions at most: a workgroup to every (sequence, head, group), nothing is cut or joined.
template <int DT, int D, int RT, bool STREAM>
__global__ __launch_bounds__(256, split_waves(DT == MI_DT_F32, D, RT)) void hist_attn_medium_kernel(AttnArgs p, int NR, int NG) {
  typedef Wave<DT, D, RT, STREAM> W;
  __shared__ FoldLds<W, RT> lds;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned int HG = (unsigned int) (p.H * NG), b = blockIdx.x / HG, pair = blockIdx.x - b * HG;
  const int head = (int) (pair / (unsigned int) NG), grp = (int) (pair - (unsigned int) head * NG);
  const int64_t len = clamped_length(p, scalar_load(p.lengths + b), pair == 0 && threadIdx.x == 0);
  const int row0 = (grp * NR + wave % NR) * 16 * RT;
  W w;
  walk_shared(w, lds, p, NR, b, head, row0, 0, (unsigned int) len, wave, lane);
  if (wave < NR) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = row0 + t * 16 + c;
      if (row < p.rows) w.store(t, out_row_of<W::QE>(p, b, head, row), g);
    }
  }
}

// Long histories: the call's work is cut into equal runs of units, a unit being UNIT positions of one (sequence, cache
// head, group of query rows), sequences slowest; a workgroup walks its run.  A run that begins or ends inside a
// (sequence, head, group) leaves an unnormalised part, which the joining launch adds up.  The cut goes by the lengths
// alone, so histories of any mix keep every workgroup equally busy, and the parts are always joined in the same order.
constexpr unsigned int UNIT = 128;
// Runs of up to ALIGN_RUN units begin and end with a row of work instead, where the chip can hold them all: a second row
// in a workgroup costs it a second start (lengths, pages, queries, the first positions: some 6 us), more than the uneven
// pieces do.  A unit is then that many times longer, and a run one unit.  (16 candidates each for 32 users: 38 us with
// runs that cross rows, 35-36 so.)
constexpr unsigned int ALIGN_RUN = 8;

struct SplitArgs {
  int NR;            // row tiles side by side in a workgroup: 1, 2 or 4 waves; the other waves share the positions
  int NG;            // groups of NR * 16 * RT query rows
  int blocks;        // workgroups of the split launch
  int slot_rows;     // rows of a part: those of a group, or all if there are fewer
  // Parts: [0] of a workgroup's run continues a row, [1] begins one
  float* parts;      // [2][workgroups][slot_rows][D]
  float2* part_ml;   // [2][workgroups][slot_rows]
  int4* meta;        // [workgroups] {sequence (-1: nothing to join), head * NG + group, last workgroup, 0}
};

__device__ __forceinline__ unsigned int units_of(int64_t len, unsigned int unit) {
  return len <= unit ? 1u : ((unsigned int) len + unit - 1) / unit;
}

template <int DT, int D, int RT, bool STREAM>
__global__ __launch_bounds__(256, split_waves(DT == MI_DT_F32, D, RT)) void hist_attn_split_kernel(AttnArgs p, SplitArgs a) {
  typedef Wave<DT, D, RT, STREAM> W;
  __shared__ FoldLds<W, RT> lds;
  __shared__ unsigned int wave_sum[4];
  __shared__ unsigned int found[2];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned int HG = (unsigned int) (p.H * a.NG), n_seqs = (unsigned int) p.n_seqs;

  // units in front of each thread's slice of the sequences, and all
  const unsigned int per = (n_seqs + 255) / 256;
  const unsigned int s0 = threadIdx.x * per, s1 = s0 + per < n_seqs ? s0 + per : n_seqs;
  unsigned int unit = UNIT, before, mine, total;
  auto count = [&](bool say) {
    mine = 0;
    for (unsigned int b = s0; b < s1; ++b) mine += units_of(clamped_length(p, p.lengths[b], say), unit);
    unsigned int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned int up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) before += wave_sum[i];
      total += wave_sum[i];
    }
    before += incl - mine;
    total = __builtin_amdgcn_readfirstlane(total) * HG;  // < 2^31, checked on the host
  };
  count(blockIdx.x == 0);
  unsigned int run = (total + gridDim.x - 1) / gridDim.x;
  if (run > 1 && run <= ALIGN_RUN && 2 * HG * n_seqs <= gridDim.x) {
    for (unsigned int k = run; total > gridDim.x; ++k) {  // at 2 * run at the latest they fit
      __syncthreads();  // wave_sum has been read
      unit = UNIT * k;
      count(false);
    }
    run = 1;
  }
  const unsigned int x0 = blockIdx.x * run, x1 = x0 + run < total ? x0 + run : total;
  if (x0 < total && before * HG <= x0 && x0 < (before + mine) * HG) {
    unsigned int b = s0;
    for (; b + 1 < s1; ++b) {
      const unsigned int u = units_of(clamped_length(p, p.lengths[b], false), unit);
      if (x0 < (before + u) * HG) break;
      before += u;
    }
    found[0] = b;
    found[1] = before * HG;
  }
  if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  if (x0 >= total) return;

  const int rt = wave % a.NR, ci = wave / a.NR;
  const int group_rows = a.NR * 16 * RT;
  unsigned int b = __builtin_amdgcn_readfirstlane(found[0]);
  unsigned int start = __builtin_amdgcn_readfirstlane(found[1]);
  unsigned int x = x0;
  while (x < x1 && b < n_seqs) {
    const int64_t len = clamped_length(p, scalar_load(p.lengths + b), false);
    const unsigned int u = units_of(len, unit);
    const unsigned int rem = x - start, pair = rem / u, ub = rem - pair * u;
    if (pair >= HG) break;  // lengths that change under the launch give nonsense, but no access out of bounds
    const int head = (int) (pair / (unsigned int) a.NG), grp = (int) (pair - (unsigned int) head * a.NG);
    const unsigned int ue = ub + (x1 - x) < u ? ub + (x1 - x) : u;
    const int row0 = (grp * a.NR + rt) * 16 * RT;
    W w;
    walk_shared(w, lds, p, a.NR, b, head, row0, ub * unit, ue == u ? (unsigned int) len : ue * unit, wave, lane);
    if (ci == 0) {
      const bool whole = ub == 0 && ue == u;
      const int64_t part = ((int64_t) (ub == 0 ? gridDim.x : 0) + blockIdx.x) * a.slot_rows - grp * group_rows;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = row0 + t * 16 + c;
        if (row < p.rows) {
          if (whole) w.store(t, out_row_of<W::QE>(p, b, head, row), g);
          else w.store_part(t, a.parts + (part + row) * D, a.part_ml + part + row, g);
        }
      }
      if (threadIdx.x == 0 && ub == 0 && ue < u) {
        const unsigned int last = (x + u - 1) / run;
        a.meta[blockIdx.x] = make_int4((int) b, (int) pair, (int) (last < gridDim.x ? last : gridDim.x - 1), 0);
      }
    }
    x += ue - ub;
    if (ue == u && pair + 1 == HG) {
      start += u * HG;
      ++b;
    }
  }
}

// Joins the parts of the (sequence, head, group) that workgroup `owner` of the split launch began and did not finish: its
// own second part, then the first parts of the workgroups behind it, in order.  A thread takes four channels of a row and
// `runs` threads share the parts; up to eight parts are requested together, and nothing crosses threads but the runs' sums.
constexpr int JOIN_THREADS = 256;

template <int DT, int D>
__device__ __forceinline__ void join_rows(const AttnArgs& p, const SplitArgs& a, int group_rows, int wg_rows, int slice, int owner,
                                          f4v* lacc, float2* lml) {
  typedef Wave<DT, D, 1, false> W;
  constexpr int PIECES = D / 4;
  const int* meta = reinterpret_cast<const int*>(a.meta + owner);
  const int b = scalar_load(meta), pair = scalar_load(meta + 1), n = scalar_load(meta + 2) - owner + 1;
  const int head = pair / a.NG, grp = pair % a.NG;
  const int n_rows = p.rows - grp * group_rows < group_rows ? p.rows - grp * group_rows : group_rows;
  const int r0 = slice * wg_rows;
  if (r0 >= n_rows) return;
  const int t = (int) threadIdx.x, piece = t % PIECES;
  const int side = PIECES * wg_rows, runs = JOIN_THREADS / side;  // threads of a run; powers of two
  const int r = r0 + (t & (side - 1)) / PIECES, run = t / side;
  const bool live = r < n_rows;
  const int rr = live ? r : r0;
  const int per = (n + runs - 1) / runs;
  const int i0 = run * per, i1 = i0 + per < n ? i0 + per : n;
  const float* sums = a.parts + rr * D + piece * 4;
  const float2* mls = a.part_ml + rr;
  float top = -INFINITY, sum = 0.f;
  f4v acc = f4v{0.f, 0.f, 0.f, 0.f};
  for (int ib = i0; ib < i1; ib += 8) {
    float2 ml[8];
    f4v x[8];
    const int m = i1 - ib;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ml[e] = make_float2(-INFINITY, 0.f);
      x[e] = f4v{0.f, 0.f, 0.f, 0.f};
      if (e < m) {
        const unsigned int at = (unsigned int) (owner + ib + e + (ib + e == 0 ? a.blocks : 0)) * (unsigned int) a.slot_rows;
        ml[e] = mls[at];
        x[e] = *reinterpret_cast<const f4v*>(sums + (uint64_t) at * D);
      }
    }
    float up = top;
#pragma unroll
    for (int e = 0; e < 8; ++e) up = fmaxf(up, ml[e].x);
    const float base = up == -INFINITY ? 0.f : up;
    const float k = __builtin_amdgcn_exp2f(top - base);
    top = up;
    sum *= k;
    acc *= k;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < m) {
        const float w = __builtin_amdgcn_exp2f(ml[e].x - base);
        sum += ml[e].y * w;
        acc += x[e] * w;
      }
  }
  if (runs > 1) {
    __syncthreads();  // the rows before have been read
    lacc[t] = acc;
    lml[t] = make_float2(top, sum);
    __syncthreads();
    if (run == 0) {
      for (int k = 1; k < runs; ++k) {
        const float2 ml = lml[t + k * side];
        const Fold f = fold_of(top, ml.x);
        top = f.m;
        sum = sum * f.a + ml.y * f.b;
        acc = acc * f.a + lacc[t + k * side] * f.b;
      }
    }
  }
  if (live && run == 0) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    char* out = out_row_of<W::QE>(p, b, head, grp * group_rows + r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = W::channel_of(piece, e);
      if (DT == MI_DT_F32) reinterpret_cast<float*>(out)[d] = acc[e] * inv;
      else reinterpret_cast<unsigned short*>(out)[d] = mi_f2bf(acc[e] * inv);
    }
  }
}

template <int DT, int D>
__global__ __launch_bounds__(JOIN_THREADS) void hist_attn_join_kernel(AttnArgs p, SplitArgs a, int group_rows, int wg_rows,
                                                                     int slices) {
  __shared__ f4v lacc[JOIN_THREADS];
  __shared__ float2 lml[JOIN_THREADS];
  // Workgroups go to the 256 CUs in turn (the eight XCDs, and there their CUs), and the owners with something to join are
  // often every 2nd, 4th or 8th: a CU takes a stretch of owners as a whole, another one with each slice of their rows, so
  // they do not meet on a few (64 rows x 2 parts x 128 heads: 22 us in the order of the owners, 8 so).  `subs` workgroups
  // share the stretch: a workgroup costs the launch about 1 ns, whether it finds something to do or not.
  const int per_cu = (a.blocks + 255) / 256, subs = (int) gridDim.x / 256 / slices;
  const int slice = (int) blockIdx.x / (256 * subs), sub = (int) blockIdx.x / 256 % subs;
  const int first = ((int) blockIdx.x + slice * 37) % 256 * per_cu + sub;
  const int lane = (int) threadIdx.x & 63, mine = first + lane * subs;
  uint64_t todo = __ballot(sub + lane * subs < per_cu && mine < a.blocks && a.meta[mine < a.blocks ? mine : 0].x >= 0);
  for (; todo; todo &= todo - 1)
    join_rows<DT, D>(p, a, group_rows, wg_rows, slice,
                     __builtin_amdgcn_readfirstlane(first + (__ffsll((unsigned long long) todo) - 1) * subs), lacc, lml);
}

constexpr int64_t SHORT_ROOM = 256, MEDIUM_ROOM = 1024;

// How a call is run; the same on every call of the same sizes.
struct AttnPlan {
  bool short_rows, medium;
  int RT, NR, NG, blocks, slot_rows;
  size_t parts_bytes, ml_bytes, bytes;
};

AttnPlan plan_attn(int dtype, int dim, int H, int page_size, int64_t n_seqs, int64_t rows, int width) {
  AttnPlan q = {};
  const int64_t room = (int64_t) width * page_size;
  q.RT = rows > 16 && dim <= 128 ? 2 : 1;  // two tiles of 256 channels do not fit the registers
  const int64_t tiles = mi_cdiv(rows, 16 * q.RT);
  q.NR = tiles >= 3 ? 4 : (int) tiles;
  q.NG = (int) mi_cdiv(tiles, q.NR);
  q.short_rows = room <= SHORT_ROOM;
  const int64_t pairs = n_seqs * H * q.NG, most = pairs * mi_cdiv(room, UNIT);
  const int64_t resident = 256 * split_waves(dtype == MI_DT_F32, dim, q.RT);
  q.blocks = (int) (most < resident ? most : resident);
  q.medium = !q.short_rows && room <= MEDIUM_ROOM && pairs <= (1 << 23);
  if (q.medium) q.blocks = (int) pairs;
  if (!q.short_rows && !q.medium) {
    const int64_t group_rows = q.NR * 16 * q.RT;
    q.slot_rows = (int) (rows < group_rows ? rows : group_rows);
    const size_t part_rows = (size_t) q.blocks * 2 * q.slot_rows;
    q.parts_bytes = part_rows * dim * sizeof(float);
    q.ml_bytes = (part_rows * sizeof(float2) + 15) / 16 * 16;
    q.bytes = q.parts_bytes + q.ml_bytes + (size_t) q.blocks * sizeof(int4);
  }
  return q;
}

template <int DT, int D>
int launch_short(const AttnArgs& p, const AttnPlan& q, hipStream_t s) {
  const int n_tiles = (int) mi_cdiv(p.rows, 16 * q.RT);
  const dim3 grid((unsigned int) mi_cdiv(p.n_seqs * p.H * n_tiles, 4));
  if (q.RT == 2) hist_attn_short_kernel<DT, D, D <= 128 ? 2 : 1><<<grid, 256, 0, s>>>(p, n_tiles);
  else hist_attn_short_kernel<DT, D, 1><<<grid, 256, 0, s>>>(p, n_tiles);
  MI_LAUNCH_CHECK();
  return MI_OK;
}

template <int DT, int D, bool STREAM>
int launch_split(const AttnArgs& p, const AttnPlan& q, void* ws, hipStream_t s) {
  if (q.medium) {
    if (q.RT == 2) hist_attn_medium_kernel<DT, D, D <= 128 ? 2 : 1, STREAM><<<q.blocks, 256, 0, s>>>(p, q.NR, q.NG);
    else hist_attn_medium_kernel<DT, D, 1, STREAM><<<q.blocks, 256, 0, s>>>(p, q.NR, q.NG);
    MI_LAUNCH_CHECK();
    return MI_OK;
  }
  SplitArgs a = {};
  a.NR = q.NR;
  a.NG = q.NG;
  a.blocks = q.blocks;
  a.slot_rows = q.slot_rows;
  a.parts = (float*) ws;
  a.part_ml = (float2*) ((char*) ws + q.parts_bytes);
  a.meta = (int4*) ((char*) ws + q.parts_bytes + q.ml_bytes);
  if (q.RT == 2) hist_attn_split_kernel<DT, D, D <= 128 ? 2 : 1, STREAM><<<q.blocks, 256, 0, s>>>(p, a);
  else hist_attn_split_kernel<DT, D, 1, STREAM><<<q.blocks, 256, 0, s>>>(p, a);
  MI_LAUNCH_CHECK();
  // few rows can have many parts: several threads share them
  const int all = JOIN_THREADS / (D / 4), wg_rows = q.slot_rows >= 16 ? all : (all / 4 + 1) / 2;
  const int slices = (int) mi_cdiv(q.slot_rows, wg_rows), per_cu = (int) mi_cdiv(q.blocks, 256);
  const int subs = slices >= 8 ? 1 : 8 / slices < per_cu ? 8 / slices : per_cu;
  hist_attn_join_kernel<DT, D><<<256 * subs * slices, JOIN_THREADS, 0, s>>>(p, a, q.NR * 16 * q.RT, wg_rows, slices);
  MI_LAUNCH_CHECK();
  return MI_OK;
}

template <int DT, int D>
int launch_attn_dim(const AttnArgs& p, const AttnPlan& q, void* ws, hipStream_t s) {
  if (q.short_rows) return launch_short<DT, D>(p, q, s);
  // past the caches where the pool does not fit the last one (64 bf16 histories of 8-16 k: 470 us so, 523 through them; the
  // other way round a pool of 164 MB that the call before has read: 38 against 34) and no second row tile reads the same
  // positions (16 candidates each for 256 users: 203 us past the caches, 174 through them)
  const bool stream = ((int64_t) p.n_pages * p.H * 2 << p.page_shift) * D * Elem<DT>::BYTES > LAST_LEVEL_BYTES &&
                      q.NR == 1 && q.NG == 1;
  return stream ? launch_split<DT, D, true>(p, q, ws, s) : launch_split<DT, D, false>(p, q, ws, s);
}

template <int DT>
int launch_attn(const AttnArgs& p, const AttnPlan& q, int dim, void* ws, hipStream_t s) {
  switch (dim) {
    case 32: return launch_attn_dim<DT, 32>(p, q, ws, s);
    case 64: return launch_attn_dim<DT, 64>(p, q, ws, s);
    case 128: return launch_attn_dim<DT, 128>(p, q, ws, s);
    default: return launch_attn_dim<DT, 256>(p, q, ws, s);
  }
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

// A call that only reads the pages takes one row of the table for all sequences too (ld 0); in a write they would all append
// to the same pages.
int check_table(const int32_t* table, int64_t ld, int width, const int32_t* lengths, int64_t n_seqs, bool write, const char* who) {
  MI_REQUIRE(table && lengths, "%s: null page table or lengths", who);
  MI_REQUIRE(n_seqs >= 0 && n_seqs <= INT32_MAX, "%s: n_seqs %lld", who, (long long) n_seqs);
  MI_REQUIRE(width >= 1 && (ld >= width || n_seqs <= 1 || (ld == 0 && !write)), "%s: page table width %d with row stride %lld", who, width, (long long) ld);
  return MI_OK;
}

// 16-byte accesses: base and strides whole multiples of 16 bytes
bool aligned16(const void* p, int elem, int64_t a, int64_t b, int64_t c = 0) {
  return (((uintptr_t) p | (uintptr_t) (a * elem) | (uintptr_t) (b * elem) | (uintptr_t) (c * elem)) & 15) == 0;
}

// Rows of `dim` elements as a call names them, for the checks of what it writes.  Dimensions of one entry and of stride 0
// are left out and strides taken as positive, neither changes which memory the rows cover; smallest stride first.
struct RowSet {
  __int128 first;  // of the lowest element, in bytes
  int elem, dim, n_dims;
  struct { __int128 n, stride; } d[3];
  bool repeats;    // a stride of 0 over several entries

  RowSet(const void* p, int elem, int dim) : first((__int128) (uintptr_t) p), elem(elem), dim(dim), n_dims(0), repeats(false) {}
  RowSet& over(int64_t n, int64_t stride) {
    if (n <= 1) return *this;
    if (stride == 0) {
      repeats = true;
      return *this;
    }
    __int128 s = stride;
    if (s < 0) {
      first += (n - 1) * s * elem;
      s = -s;
    }
    int i = n_dims++;
    for (; i > 0 && d[i - 1].stride > s; --i) d[i] = d[i - 1];
    d[i].n = n;
    d[i].stride = s;
    return *this;
  }
  __int128 extent(int levels) const {  // elements from the first to behind the last, over the inner `levels` dimensions
    __int128 e = dim;
    for (int i = 0; i < levels; ++i) e += (d[i].n - 1) * d[i].stride;
    return e;
  }
  // No two rows share memory: every stride reaches over all that lies inside it.  (Other sets without an overlap, strides of
  // 2 and 3 rows over two entries each, do not count as apart.)
  bool apart() const {
    if (repeats) return false;
    for (int i = 0; i < n_dims; ++i)
      if (d[i].stride < extent(i)) return false;
    return true;
  }
  // May share memory: exactly so where the two differ in their start alone (or, from some dimension inwards, lie in separate
  // stretches), otherwise by their whole stretches.  `ahead`: elements from this set's first to the other's.
  bool meets(const RowSet& o) const {
    const __int128 bytes = o.first - first;
    if (bytes % elem) return first < o.first + o.extent(o.n_dims) * elem && o.first < first + extent(n_dims) * elem;
    return meets(o, n_dims, o.n_dims, bytes / elem);
  }
  bool meets(const RowSet& o, int a, int b, __int128 ahead) const {
    if (ahead >= extent(a) || -ahead >= o.extent(b)) return false;
    if (a == 0 && b == 0) return true;
    if (a == 0 || b == 0 || d[a - 1].n != o.d[b - 1].n || d[a - 1].stride != o.d[b - 1].stride) return true;
    const __int128 n = d[a - 1].n, s = d[a - 1].stride;
    if (extent(a - 1) > s || o.extent(b - 1) > s) return true;
    const __int128 t = -ahead / s;  // entries t apart come within a stride of each other, and those beside
    for (__int128 i = t - 1; i <= t + 1; ++i)
      if (i > -n && i < n && meets(o, a - 1, b - 1, ahead + i * s)) return true;
    return false;
  }
};

int rows_call(const char* who, bool read, const mi_hist_cache* cache, const void* k, const void* v, int dtype, int64_t k_row,
              int64_t k_head, int64_t v_row, int64_t v_head, int64_t n_rows, const int64_t* offsets, int64_t n_seqs,
              const int32_t* table, int64_t ld_table, int width, const int32_t* lengths, int32_t* err, void* stream) {
  if (int rc = check_cache(cache, who)) return rc;
  MI_REQUIRE(dtype == MI_DT_F32 || dtype == MI_DT_BF16, "%s: rows are f32 or bf16, not %d", who, dtype);
  MI_REQUIRE(n_rows >= 0, "%s: n_rows %lld", who, (long long) n_rows);
  if (n_rows == 0 || n_seqs == 0) return MI_OK;
  if (int rc = check_table(table, ld_table, width, lengths, n_seqs, !read, who)) return rc;
  MI_REQUIRE(k && v, "%s: null rows", who);
  MI_REQUIRE(aligned16(k, dtype == MI_DT_F32 ? 4 : 2, k_row, k_head) && aligned16(v, dtype == MI_DT_F32 ? 4 : 2, v_row, v_head),
             "%s: rows must start on 16-byte boundaries", who);
  MI_REQUIRE(offsets || n_rows % n_seqs == 0, "%s: %lld rows do not divide among %lld sequences", who, (long long) n_rows,
             (long long) n_seqs);
  if (n_rows * 2 * cache->n_heads > (int64_t) INT32_MAX) {
    mi_set_error("%s: %lld rows of %d heads in one call (at most 2^31-1 rows of K and V)", who, (long long) n_rows, cache->n_heads);
    return MI_ERR_UNSUPPORTED;
  }
  if (read) {  // rows that share memory would be written in no order
    const int e = dtype == MI_DT_F32 ? 4 : 2;
    const RowSet ks = RowSet(k, e, cache->dim).over(n_rows, k_row).over(cache->n_heads, k_head);
    const RowSet vs = RowSet(v, e, cache->dim).over(n_rows, v_row).over(cache->n_heads, v_head);
    MI_REQUIRE(ks.apart() && vs.apart() && !ks.meets(vs), "%s: the rows to be filled overlap", who);
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
  if (check_cache(cache, "mi_hist_attn_workspace_bytes") || n_seqs < 1 || n_queries < 1 || q_heads < 1 || table_width < 1 ||
      q_heads % cache->n_heads)
    return 0;
  return plan_attn(cache->dtype, cache->dim, cache->n_heads, cache->page_size, n_seqs,
                   (int64_t) n_queries * (q_heads / cache->n_heads), table_width).bytes;
}

extern "C" int mi_hist_attn(const mi_hist_cache* cache, const void* q, int64_t q_seq, int64_t q_tok, int64_t q_head, int q_heads,
                            int n_queries, int64_t n_seqs, const int32_t* page_table, int64_t ld_table, int table_width,
                            const int32_t* lengths, float scale, void* out, int64_t out_seq, int64_t out_tok, int64_t out_head,
                            void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  if (int rc = check_cache(cache, "mi_hist_attn")) return rc;
  MI_REQUIRE(n_queries >= 0 && q_heads >= 1 && q_heads % cache->n_heads == 0,
             "mi_hist_attn: %d queries of %d heads over a cache of %d heads", n_queries, q_heads, cache->n_heads);
  if (n_seqs == 0 || n_queries == 0) return MI_OK;
  if (int rc = check_table(page_table, ld_table, table_width, lengths, n_seqs, false, "mi_hist_attn")) return rc;
  MI_REQUIRE(q && out, "mi_hist_attn: null q or out");
  const int qe = cache->dtype == MI_DT_F32 ? 4 : 2;
  MI_REQUIRE(aligned16(q, qe, q_seq, q_tok, q_head) && aligned16(out, qe, out_seq, out_tok, out_head),
             "mi_hist_attn: the rows of q and out must start on 16-byte boundaries");
  AttnArgs p = {};
  p.kv = (const char*) cache->kv;
  p.exps = (const uint8_t*) cache->exps;
  p.n_pages = (int) cache->n_pages;
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
  p.table = page_table;
  p.ld_table = ld_table;
  p.width = table_width;
  p.lengths = lengths;
  p.n_seqs = n_seqs;
  p.scale = scale * 1.44269504088896340736f;
  p.err = err;
  const AttnPlan plan = plan_attn(cache->dtype, cache->dim, p.H, cache->page_size, n_seqs, rows, table_width);
  // unit numbers are 32-bit in the kernels
  const int64_t tiles = mi_cdiv(rows, 16);
  if (n_seqs * p.H > (1 << 25) / tiles ||  // waves of a launch
      mi_cdiv((int64_t) table_width * cache->page_size, UNIT) > INT32_MAX / (n_seqs * p.H * tiles)) {
    mi_set_error("mi_hist_attn: %lld sequences x %d heads x %lld row tiles over %d pages in one call", (long long) n_seqs, p.H,
                 (long long) tiles, table_width);
    return MI_ERR_UNSUPPORTED;
  }
  const RowSet outs = RowSet(out, qe, cache->dim).over(n_seqs, out_seq).over(n_queries, out_tok).over(q_heads, out_head);
  MI_REQUIRE(outs.apart(), "mi_hist_attn: the rows of out overlap");
  if (plan.bytes) {
    MI_REQUIRE(((uintptr_t) workspace & 15) == 0, "mi_hist_attn: the workspace must be 16-byte aligned");
    if (!workspace || workspace_bytes < plan.bytes) {
      mi_set_error("mi_hist_attn: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t) 0, plan.bytes);
      return MI_ERR_WORKSPACE;
    }
  }
  // a row of out that is another row of q would be written while that is still to be read
  const bool same = q == out && (n_seqs <= 1 || q_seq == out_seq) && (n_queries <= 1 || q_tok == out_tok) &&
                    (q_heads <= 1 || q_head == out_head);
  MI_REQUIRE(same || !outs.meets(RowSet(q, qe, cache->dim).over(n_seqs, q_seq).over(n_queries, q_tok).over(q_heads, q_head)),
             "mi_hist_attn: out overlaps q without being q");
  hipStream_t s = (hipStream_t) stream;
  switch (cache->dtype) {
    case MI_DT_F32: return launch_attn<MI_DT_F32>(p, plan, cache->dim, workspace, s);
    case MI_DT_BF16: return launch_attn<MI_DT_BF16>(p, plan, cache->dim, workspace, s);
    default: return launch_attn<MI_DT_E4M3>(p, plan, cache->dim, workspace, s);
  }
}
