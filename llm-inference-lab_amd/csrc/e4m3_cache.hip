// A paged cache of 8-bit keys and values: the write that turns, quantises and stores the new
// tokens' keys and values, and the reading of stored ones.  gfx950 only.
//
// A key (or value) of d numbers x is stored as d codes of e4m3 (sign, 4 bits of exponent, 3 of mantissa; largest number
// 448, subnormals in steps of 2^-9, no infinity) and one byte b = e + 127:
//   e = the smallest whole number >= -100 with max |x_i| <= 448 * 2^e,   code_i = e4m3(x_i / 2^e), ties to even,
// so x_i ~ code_i * 2^e.  A scale that is a power of two costs no rounding of its own, neither here nor where a stored
// number is read: code * 2^e is a bfloat16 number.  What is not finite becomes the code that is not a number, and the
// scale is that of the finite ones.
//
// The angles of the rotation, its products and the quantised numbers are taken in 64 bits: a position of 30,000 leaves
// a float32 angle 2^-10 of a turn, and a number next to the border between two codes (one of 16 steps in an octave) goes
// to the one that the formula says.  The vector unit takes float64 products at the float32 rate, and the pass over memory
// bounds the kernel.
#include "common.h"

constexpr int LOWEST_EXPONENT = -100;

// v to 32 bits so that a rounding to fewer bits afterwards gives what one rounding of v gives: the last bit
// is set where v lies between two float32 numbers (rounding to odd).
__device__ __forceinline__ float to_odd(double v) {
  const float f = (float)v;
  const double back = (double)f;
  if (back == v || !(fabs(v) < __builtin_huge_val())) return f;
  unsigned bits = __float_as_uint(f);
  if (fabs(back) > fabs(v)) --bits;      // towards zero ...
  return __uint_as_float(bits | 1u);     // ... and odd
}

// The byte of the scale for the largest magnitude `most` (finite, rounded to odd: no even number is crossed)
__device__ __forceinline__ int scale_byte(float most) {
  const unsigned bits = __float_as_uint(most);
  const int exponent = (int)(bits >> 23) - 127;                             // 448 = 1.75 * 2^8
  const int e = exponent - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return max(e, LOWEST_EXPONENT) + 127;
}
__device__ __forceinline__ float power_of_byte(int b) { return __uint_as_float((unsigned)b << 23); }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

// The code of x in units of the scale (inv = 2^-e)
constexpr unsigned char NO_NUMBER = 0x7f;
__device__ __forceinline__ unsigned char to_code(float x, float inv) {
  const float u = x * inv;
  return finite(x) ? (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(u, u, 0, false) : NO_NUMBER;
}

// Where the codes of a (page, kv head) lie: e4m3_key_index / e4m3_value_index below (k = key within
// the page, i = number within the head, d a multiple of 16), in the order in which the attention's operands are read.
//   keys:    [16-key block][sixteen of d][key in block][16]
//   values:  [16-key block][group of four 16-wide blocks of d][group of 4 keys][number in block][block of the group][4]
__device__ __forceinline__ size_t key_index(int k, int i, int d) {
  return ((size_t)((k >> 4) * (d >> 4) + (i >> 4)) * 16 + (k & 15)) * 16 + (i & 15);
}
__device__ __forceinline__ size_t value_index(int k, int i, int d) {
  const int group = i >> 6, wide = min(4, (d >> 4) - 4 * group);
  return (size_t)(k >> 4) * 16 * d + (size_t)group * 1024 +
         ((((k & 15) >> 2) * 16 + (i & 15)) * wide + ((i >> 4) & 3)) * 4 + (k & 3);
}

struct CacheArgs {
  const int* positions;
  const int* row_req;
  const int* table;
  int table_stride, table_width, reqs, page_size, pages;
  int nq, nkv, d;
  unsigned char* k;
  unsigned char* v;
  unsigned char* scale;      // [pages, nkv, 2, page_size]
};

// The page of row r's position, or -1 where it has none
__device__ __forceinline__ int page_of(const CacheArgs& a, int r, int* off) {
  const int pos = a.positions[r], req = a.row_req[r];
  *off = 0;
  if (pos < 0 || req < 0 || req >= a.reqs || pos / a.page_size >= a.table_width) return -1;
  *off = pos % a.page_size;
  const int page = a.table[(size_t)req * a.table_stride + pos / a.page_size];
  return page >= 0 && page < a.pages ? page : -1;
}

// N numbers of a row from an address that is aligned for it (WIDE) or not
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void load_numbers(const T* src, float (&x)[N]) {
  if constexpr (WIDE) {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec v = *(const vec*)src;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float((T)v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(src[i]);
  }
}
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void store_numbers(T* dst, const float (&x)[N]) {
  if constexpr (WIDE) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(x[i]);
    *(vec*)dst = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = from_float<T>(x[i]);
  }
}

// The four numbers of a word of codes (zeros where there is no page)
__device__ __forceinline__ void decode_four(unsigned w, float size, bool there, float* x) {
  x[0] = there ? __builtin_amdgcn_cvt_f32_fp8(w, 0) * size : 0.f;
  x[1] = there ? __builtin_amdgcn_cvt_f32_fp8(w, 1) * size : 0.f;
  x[2] = there ? __builtin_amdgcn_cvt_f32_fp8(w, 2) * size : 0.f;
  x[3] = there ? __builtin_amdgcn_cvt_f32_fp8(w, 3) * size : 0.f;
}

// Four codes in a word, in their order
__device__ __forceinline__ unsigned four_codes(const float (&x)[4], float inv) {
  return (unsigned)to_code(x[0], inv) | (unsigned)to_code(x[1], inv) << 8 | (unsigned)to_code(x[2], inv) << 16 |
         (unsigned)to_code(x[3], inv) << 24;
}

// ROWS rows a block, WAVES waves a row.  A lane has four pairs of a head (channels 4 s .. 4 s + 3 and those half a head
// further), so a wave of 64 has several heads at a time, whatever the head size.  Every lane takes the sine and cosine
// of one pair of its row (of two above heads of 128) and they are shared through LDS.  With 16 rows a block (many rows: what the
// block stores fills whole blocks of 16 keys on one die's L2) the values' codes meet in LDS: where four rows are the
// four keys of a word of the pages, the word is stored, and else its bytes.
template <typename T, int ROWS, int WAVES, bool WIDE>
__global__ __launch_bounds__(64 * ROWS * WAVES) void rope_kv_write_e4m3_kernel(const T* qkv, size_t row_stride, const float* inv_freq,
                                                                                 T* q_out, size_t q_stride, int rows, CacheArgs a) {
  __shared__ double s_turn[ROWS * WAVES][256];      // [wave][d / 2 cosines, d / 2 sines]
  __shared__ int s_page[ROWS], s_off[ROWS];
  extern __shared__ unsigned char s_codes[];        // [ROWS][nkv * d] where ROWS = 16
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = wave / WAVES, r = blockIdx.x * ROWS + slot;
  const int d = a.d, half = d >> 1, lanes = half >> 2, heads_at_once = 64 / lanes;
  const int here = lane / lanes, sub = lane - here * lanes, i0 = sub * 4;
  const bool live = r < rows;
  int off = 0;
  const int page = live ? page_of(a, r, &off) : -1;
  if (lane == 0 && wave % WAVES == 0) {
    s_page[slot] = page;
    s_off[slot] = off;
  }
  double* turn = s_turn[wave];
  if (inv_freq && live) {
    const double pos = (double)a.positions[r];
    for (int i = lane; i < half; i += 64) sincos(pos * (double)inv_freq[i], &turn[half + i], &turn[i]);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  double c[4], s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = inv_freq && live ? turn[i0 + j] : 1.0;      // (a lane past the heads: within the row of 256, not used)
    s[j] = inv_freq && live ? turn[half + i0 + j] : 0.0;
  }
  const int heads = a.nq + 2 * a.nkv;
  for (int first = (wave % WAVES) * heads_at_once; live && first < heads; first += WAVES * heads_at_once) {
    const int head = first + here;
    const bool in = here < heads_at_once && head < heads;
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.nkv;
    const T* src = qkv + (size_t)r * row_stride + (size_t)(in ? head : first) * d;
    float lo[4], hi[4], most = 0.f;
    load_numbers<T, 4, WIDE>(src + i0, lo);
    load_numbers<T, 4, WIDE>(src + i0 + half, hi);
    if (inv_freq && !is_v) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = (double)lo[j], y = (double)hi[j];
        lo[j] = to_odd(x * c[j] - y * s[j]);
        hi[j] = to_odd(y * c[j] + x * s[j]);
      }
    }
    if (in && is_q) {
      T* dst = q_out + (size_t)r * q_stride + (size_t)head * d + i0;
      store_numbers<T, 4, WIDE>(dst, lo);
      store_numbers<T, 4, WIDE>(dst + half, hi);
    }
    if (first + heads_at_once <= a.nq) continue;      // (queries only)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (finite(lo[j])) most = fmaxf(most, fabsf(lo[j]));
      if (finite(hi[j])) most = fmaxf(most, fabsf(hi[j]));
    }
    // the largest over the head's lanes: circling, every step doubles how many a lane has seen (a number seen twice
    // changes no maximum, so their count need not be a power of two)
    for (int step = 1; step < lanes; step <<= 1) {
      const int other = sub + step;
      most = fmaxf(most, __shfl(most, here * lanes + (other < lanes ? other : other - lanes), WAVE));
    }
    if (!in || is_q || page < 0) continue;
    const int byte = scale_byte(most);
    const float inv = power_of_byte(254 - byte);
    const int kvh = head - a.nq - (is_v ? a.nkv : 0);
    const size_t at = ((size_t)page * a.nkv + kvh) * a.page_size;
    const unsigned cl = four_codes(lo, inv), ch = four_codes(hi, inv);
    if (sub == 0) a.scale[2 * at + (is_v ? a.page_size : 0) + off] = (unsigned char)byte;
    if (!is_v) {
      *(unsigned*)(a.k + at * d + key_index(off, i0, d)) = cl;
      *(unsigned*)(a.k + at * d + key_index(off, i0 + half, d)) = ch;
    } else if constexpr (ROWS == 16) {
      unsigned char* dst = s_codes + ((size_t)slot * a.nkv + kvh) * d + i0;
      *(unsigned*)dst = cl;
      *(unsigned*)(dst + half) = ch;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a.v[at * d + value_index(off, i0 + j, d)] = (unsigned char)(cl >> (8 * j));
        a.v[at * d + value_index(off, i0 + half + j, d)] = (unsigned char)(ch >> (8 * j));
      }
    }
  }
  if constexpr (ROWS == 16) {
    static_assert(WAVES == 1, "a wave a row");
    __syncthreads();
    const int width = a.nkv * d;
    // lane j: whether rows j .. j + 3 are the four keys of a word
    const int j = lane & 15, jp = s_page[j], jo = s_off[j];
    bool leads = lane < 13 && jp >= 0 && (jo & 3) == 0;
#pragma unroll
    for (int t = 1; t < 4; ++t) leads = leads && s_page[min(j + t, 15)] == jp && s_off[min(j + t, 15)] == jo + t;
    const unsigned leaders = (unsigned)__ballot(leads);
    // four waves a word of keys
    unsigned left = leaders;
    for (int n = 0; left; ++n, left &= left - 1) {
      if (n != wave >> 2) continue;
      const int row = __ffs(left) - 1;
      const int to_page = s_page[row], to_off = s_off[row];
      for (int n2 = (wave & 3) * 64 + lane; n2 < width; n2 += 256) {
        const int kvh = n2 / d, m = n2 - kvh * d;      // m counts words in the order in which they lie
        const int group = m >> 6, wide = min(4, (d >> 4) - 4 * group), in_group = m & 63;
        const int i = group * 64 + (in_group % wide) * 16 + in_group / wide;
        unsigned word = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) word |= (unsigned)s_codes[((size_t)(row + t) * a.nkv + kvh) * d + i] << (8 * t);
        const size_t at = ((size_t)to_page * a.nkv + kvh) * a.page_size;
        *(unsigned*)(a.v + at * d + value_index(to_off, i, d)) = word;
      }
    }
    const unsigned covered = leaders | leaders << 1 | leaders << 2 | leaders << 3;
    if (!(covered >> slot & 1) && page >= 0)
      for (int n = lane; n < width; n += 64) {
        const int kvh = n / d, i = n - kvh * d;
        a.v[((size_t)page * a.nkv + kvh) * a.page_size * d + value_index(off, i, d)] = s_codes[(size_t)slot * width + n];
      }
  }
}

// ROWS rows a wave.  A lane takes 16 numbers of a key (16 consecutive bytes of the page) and writes them one after
// the other; of values the up to four 16-wide blocks' words of a number, each with the codes of four keys, of which a row
// takes one: all four where the wave's rows are the four keys of a word.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void read_kv_e4m3_kernel(T* k_out, T* v_out, int rows, CacheArgs a) {
  typedef unsigned uint4v __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63;
  const int r0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * ROWS;
  if (r0 >= rows) return;
  const int d = a.d, sixteens = d >> 4, groups = (sixteens + 3) >> 2, width = a.nkv * d, n_rows = min(ROWS, rows - r0);
  int page[ROWS], off[ROWS];
  bool word = ROWS == 4 && n_rows == 4;
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    page[t] = t < n_rows ? page_of(a, r0 + t, &off[t]) : -1;
    if (t >= n_rows) off[t] = 0;
    word = word && page[t] == page[0] && off[t] == (off[0] & ~3) + t;
  }
  word = word && page[0] >= 0;
  // keys
  for (int n = lane; n < a.nkv * sixteens; n += 64) {
    const int kvh = n / sixteens, six = n - kvh * sixteens;
    uint4v codes[ROWS];
    float size[ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      const size_t at = ((size_t)max(page[t], 0) * a.nkv + kvh) * a.page_size;
      codes[t] = a.pages > 0 ? *(const uint4v*)(a.k + at * d + key_index(off[t], six * 16, d)) : uint4v{0, 0, 0, 0};
      size[t] = a.pages > 0 ? power_of_byte(a.scale[2 * at + off[t]]) : 0.f;
    }
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      if (t >= n_rows) break;
      T* dst = k_out + (size_t)(r0 + t) * width + n * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) decode_four(codes[t][2 * h + j], size[t], page[t] >= 0, x + 4 * j);
        store_numbers<T, 8, true>(dst + 8 * h, x);
      }
    }
  }
  // values: a lane has four neighbouring numbers of up to four 16-wide blocks, 64 consecutive bytes of the page
  for (int n = lane; n < a.nkv * groups * 4; n += 64) {
    const int kvh = n / (groups * 4), m = n - kvh * groups * 4, group = m >> 2, c = (m & 3) * 4;
    const int wide = min(4, sixteens - 4 * group);
    unsigned codes[ROWS][4][4];      // [row][number][block of the group]
    float size[ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      const size_t at = ((size_t)max(page[t], 0) * a.nkv + kvh) * a.page_size;
      size[t] = a.pages > 0 ? power_of_byte(a.scale[2 * at + a.page_size + off[t]]) : 0.f;
      const unsigned* src = (const unsigned*)(a.v + at * d + (value_index(off[t], group * 64 + c, d) & ~(size_t)3));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (word && t > 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[t][i][j] = codes[0][i][j];
        } else if (a.pages <= 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[t][i][j] = 0;
        } else if (wide == 4) {
          const uint4v w = *(const uint4v*)(src + 4 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[t][i][j] = w[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[t][i][j] = src[i * wide + min(j, wide - 1)];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      if (t >= n_rows) break;
      T* dst = v_out + (size_t)(r0 + t) * width + (size_t)kvh * d + group * 64 + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = page[t] >= 0 ? __builtin_amdgcn_cvt_f32_fp8(codes[t][i][j] >> (8 * (off[t] & 3)), 0) * size[t] : 0.f;
        if (j < wide) store_numbers<T, 4, true>(dst + j * 16, x);
      }
    }
  }
}

extern "C" const char* llmlab_last_error() { return g_llmlab_error; }

static int check_cache(const char* what, const CacheArgs& a, int rows) {
  LLMLAB_REQUIRE(rows >= 0 && a.nq >= 0 && a.nkv > 0 && a.d >= 16 && a.d <= 256 && a.d % 16 == 0,
                 "%s: bad sizes rows=%d heads=%d kv heads=%d d=%d", what, rows, a.nq, a.nkv, a.d);
  LLMLAB_REQUIRE(a.page_size >= 16 && (a.page_size & (a.page_size - 1)) == 0,
                 "%s: page size %d is not a power of two >= 16", what, a.page_size);
  LLMLAB_REQUIRE(a.pages >= 0 && a.table_width >= 0 && a.reqs >= 0, "%s: bad block table", what);
  LLMLAB_REQUIRE(((uintptr_t)a.k % 16) == 0 && ((uintptr_t)a.v % 16) == 0, "%s: the pages are not aligned to 16 bytes", what);
  return 0;
}

extern "C" int llmlab_rope_kv_write_e4m3(const void* qkv, int dtype, int rows, size_t row_stride, int nq, int nkv, int d,
                                         const float* inv_freq, const int* positions, const int* row_req,
                                         const int* table, int table_stride, int table_width, int reqs, int page_size,
                                         int pages, void* k, void* v, void* scale, void* q_out, size_t q_stride,
                                         hipStream_t stream) {
  CacheArgs a{positions, row_req, table, table_stride, table_width, reqs, page_size, pages, nq, nkv, d,
              (unsigned char*)k, (unsigned char*)v, (unsigned char*)scale};
  const int rc = check_cache("rope_kv_write_e4m3", a, rows);
  if (rc) return rc;
  LLMLAB_REQUIRE(row_stride >= (size_t)(nq + 2 * nkv) * d && q_stride >= (size_t)nq * d, "rope_kv_write_e4m3: row strides too small");
  if (rows == 0) return 0;
  const bool wide = (uintptr_t)qkv % (dtype == DT_BF16 ? 8 : 16) == 0 && (uintptr_t)q_out % (dtype == DT_BF16 ? 8 : 16) == 0 &&
                    row_stride % 4 == 0 && q_stride % 4 == 0;
  auto launch = [&](auto kernel, int rows_a_block, int waves, size_t lds, auto* x, auto* y) {
    hipLaunchKernelGGL(kernel, dim3((rows + rows_a_block - 1) / rows_a_block), dim3(64 * rows_a_block * waves), lds, stream, x,
                       row_stride, inv_freq, y, q_stride, rows, a);
  };
  // Many rows: 16 a block where their values' codes fit beside the sines; few: as many waves a row as spread over the chip.
  const size_t codes = (size_t)16 * nkv * d;
  const bool many = rows >= 1024 && codes <= 31 * 1024;
  auto pick = [&](auto t) {
    typedef decltype(t) T;
    const T* x = (const T*)qkv;
    T* y = (T*)q_out;
    if (!wide) launch(rope_kv_write_e4m3_kernel<T, 1, 4, false>, 1, 4, 0, x, y);
    else if (many) launch(rope_kv_write_e4m3_kernel<T, 16, 1, true>, 16, 1, codes, x, y);
    else launch(rope_kv_write_e4m3_kernel<T, 1, 4, true>, 1, 4, 0, x, y);
  };
  if (dtype == DT_BF16) pick(bf16_t());
  else pick(float());
  LLMLAB_LAUNCH_CHECK("rope_kv_write_e4m3");
  return 0;
}

extern "C" int llmlab_read_kv_e4m3(const void* k, const void* v, const void* scale, int nkv, int d, int rows,
                                   const int* positions, const int* row_req, const int* table, int table_stride,
                                   int table_width, int reqs, int page_size, int pages, void* k_out, void* v_out, int dtype,
                                   hipStream_t stream) {
  CacheArgs a{positions, row_req, table, table_stride, table_width, reqs, page_size, pages, 0, nkv, d,
              (unsigned char*)k, (unsigned char*)v, (unsigned char*)scale};
  const int rc = check_cache("read_kv_e4m3", a, rows);
  if (rc) return rc;
  if (rows == 0) return 0;
  LLMLAB_REQUIRE((uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0, "read_kv_e4m3: the outputs are not aligned to 16 bytes");
  auto pick = [&](auto t) {
    typedef decltype(t) T;
    if (rows >= 4096)
      hipLaunchKernelGGL((read_kv_e4m3_kernel<T, 4>), dim3((rows + 15) / 16), dim3(256), 0, stream, (T*)k_out, (T*)v_out, rows, a);
    else
      hipLaunchKernelGGL((read_kv_e4m3_kernel<T, 1>), dim3((rows + 3) / 4), dim3(256), 0, stream, (T*)k_out, (T*)v_out, rows, a);
  };
  if (dtype == DT_BF16) pick(bf16_t());
  else pick(float());
  LLMLAB_LAUNCH_CHECK("read_kv_e4m3");
  return 0;
}
