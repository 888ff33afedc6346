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
// bounds the kernel.  8,192 rows of 28 heads of 128 over 4 (143 MB) take 37.5 us (3.8 TB/s; without the rotation 34): a row is a wave's
// chain of loads, products and stores, its next heads asked for while some are turned.
#include "common.h"

constexpr int LOWEST_EXPONENT = -100;

// v to 32 bits so that a rounding to fewer bits afterwards gives what one rounding of v gives: cut off behind 24 bits, and the last
// of them is set where anything was cut (rounding to odd).  What is finite stays finite.
__device__ __forceinline__ float to_odd(double v) {
  const unsigned low = (unsigned)__double2loint(v), cut = low & 0x1fffffffu;
  const float f = (float)__hiloint2double(__double2hiint(v), (int)((low ^ cut) | (cut ? 0x20000000u : 0u)));
  return fabsf(f) == __builtin_huge_valf() && fabs(v) < __builtin_huge_val() ? copysignf(3.40282347e38f, f) : f;
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

// Sine and cosine of an angle up to 2^31, to 2^-53: the nearest whole number k of quarter turns is taken off in two parts of pi / 2 (the
// first product is exact inside the fma), Taylor's sums of the rest, |r| <= pi / 4, to r^15 and r^16 (what is left out:
// r^17 / 17! < 5e-17), and k % 4 says which is which.
__device__ __forceinline__ void sine_cosine(double angle, double* sine, double* cosine) {
  const double k = rint(angle * 0.63661977236758134308);
  const double r = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, angle)), x = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, x, 1.0 / 6227020800.0);
  c = fma(c, x, -1.0 / 87178291200.0);
  s = fma(s, x, -1.0 / 39916800.0);
  c = fma(c, x, 1.0 / 479001600.0);
  s = fma(s, x, 1.0 / 362880.0);
  c = fma(c, x, -1.0 / 3628800.0);
  s = fma(s, x, -1.0 / 5040.0);
  c = fma(c, x, 1.0 / 40320.0);
  s = fma(s, x, 1.0 / 120.0);
  c = fma(c, x, -1.0 / 720.0);
  s = fma(s, x, -1.0 / 6.0);
  c = fma(c, x, 1.0 / 24.0);
  c = fma(c, x, -0.5);
  s = fma(s * x, r, r);
  c = fma(c, x, 1.0);
  const unsigned quarter = (unsigned)(long)k;
  const double a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  *sine = quarter & 2 ? -a : a;
  *cosine = (quarter + 1) & 2 ? -b : b;
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
template <typename T, int N>
struct Numbers {
  typedef T vec __attribute__((ext_vector_type(N)));
};
template <typename T, int N, bool WIDE>
__device__ __forceinline__ typename Numbers<T, N>::vec load_numbers(const T* src) {
  typedef typename Numbers<T, N>::vec vec;
  if constexpr (WIDE) return *(const vec*)src;
  vec v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = src[i];
  return v;
}
// PAST: written past the caches (whole lines only: of half lines each would go to memory by itself)
template <typename T, int N, bool WIDE, bool PAST = false>
__device__ __forceinline__ void store_numbers(T* dst, const float (&x)[N]) {
  if constexpr (WIDE) {
    typename Numbers<T, N>::vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(x[i]);
    if constexpr (PAST)
      __builtin_nontemporal_store(v, (decltype(v)*)dst);
    else
      *(decltype(v)*)dst = v;
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

// ROWS rows a block of WAVES waves, as many for every row.  A lane has four pairs of a head (channels 4 s .. 4 s + 3 and
// those half a head further), so a wave of 64 has several heads at a time, whatever the head size.  Every lane takes the sine and
// cosine of one pair of its row (of two above heads of 128) and they are shared through LDS.  Where a block has several
// rows the values' codes meet in LDS: where four rows are the four keys of a word of the pages, the word is stored, and else
// its bytes.
template <typename T, int ROWS, int WAVES, bool WIDE>
__global__ __launch_bounds__(64 * WAVES) void rope_kv_write_e4m3_kernel(const T* qkv, size_t row_stride, const float* inv_freq,
                                                                          T* q_out, size_t q_stride, int rows, CacheArgs a) {
  static_assert(WAVES % ROWS == 0 && (ROWS == 1 || WAVES % 4 == 0), "as many waves for every row, four for a word of keys");
  __shared__ double s_turn[WAVES][256];             // [wave][d / 2 cosines, d / 2 sines]
  __shared__ int s_page[ROWS], s_off[ROWS];
  extern __shared__ unsigned char s_codes[];        // [ROWS][nkv * d] where ROWS > 1
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int EACH = WAVES / ROWS;                // waves of a row
  const int slot = wave / EACH, r = blockIdx.x * ROWS + slot;
  const int d = a.d, half = d >> 1, lanes = half >> 2, heads_at_once = 64 / lanes;
  const int here = lane / lanes, sub = lane - here * lanes, i0 = sub * 4;
  const int heads = a.nq + 2 * a.nkv;
  const bool live = r < rows;
  // (no branch around a load: where it ends the compiler would wait for all that is on its way; past the heads the last one is read)
  typename Numbers<T, 4>::vec next_lo, next_hi;
  auto fetch = [&](int first) {
    const T* src = qkv + (size_t)min(r, rows - 1) * row_stride + (size_t)min(first + here, heads - 1) * d;
    next_lo = load_numbers<T, 4, WIDE>(src + i0);
    next_hi = load_numbers<T, 4, WIDE>(src + i0 + half);
  };
  const int step = EACH * heads_at_once;
  int first = wave % EACH * heads_at_once;
  fetch(first);
  int off = 0;
  const int page = live ? page_of(a, r, &off) : -1;
  if (lane == 0 && ROWS > 1 && wave % EACH == 0) {
    s_page[slot] = page;
    s_off[slot] = off;
  }
  double* turn = s_turn[wave];
  if (inv_freq && live) {
    const double pos = (double)a.positions[r];
    for (int i = lane; i < half; i += 64) sine_cosine(pos * (double)inv_freq[i], &turn[half + i], &turn[i]);
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
  for (; live && first < heads; first += step) {
    const int head = first + here;
    const bool in = here < heads_at_once && head < heads;
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.nkv;
    const auto raw_lo = next_lo, raw_hi = next_hi;
    fetch(first + step);
    float lo[4], hi[4], most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = to_float((T)raw_lo[j]);
      hi[j] = to_float((T)raw_hi[j]);
    }
    if (inv_freq && !is_v) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = (double)lo[j], y = (double)hi[j];
        const double p = x * c[j] - y * s[j], q = y * c[j] + x * s[j];
        lo[j] = sizeof(T) == 4 && is_q ? (float)p : to_odd(p);
        hi[j] = sizeof(T) == 4 && is_q ? (float)q : to_odd(q);
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
    } else if constexpr (ROWS > 1) {
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
  if constexpr (ROWS > 1) {
    __syncthreads();
    const int width = a.nkv * d;
    // lane j: whether rows j .. j + 3 are the four keys of a word
    const int j = lane & (ROWS - 1), jp = s_page[j], jo = s_off[j];
    bool leads = lane < ROWS - 3 && jp >= 0 && (jo & 3) == 0;
#pragma unroll
    for (int t = 1; t < 4; ++t) leads = leads && s_page[min(j + t, ROWS - 1)] == jp && s_off[min(j + t, ROWS - 1)] == jo + t;
    const unsigned leaders = (unsigned)__ballot(leads);
    // four waves a word of keys
    unsigned left = leaders;
    for (int n = 0; left; ++n, left &= left - 1) {
      if (n % (WAVES / 4) != wave >> 2) continue;
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
      for (int n = wave % EACH * 64 + lane; n < width; n += EACH * 64) {
        const int kvh = n / d, i = n - kvh * d;
        a.v[((size_t)page * a.nkv + kvh) * a.page_size * d + value_index(off, i, d)] = s_codes[(size_t)slot * width + n];
      }
  }
}

// ROWS rows a wave, 1,024 of their numbers at a time, keys and then values.  What is read and what is written both are whole lines:
// the codes are fetched 16 bytes a lane in the page's order (of four rows that are the four keys of a word: four
// neighbouring lanes have the four keys' same sixteen, 64 consecutive bytes; of values 256 bytes a group), meet in LDS row by row, and
// go out 16 bytes a lane in the rows' order, past the caches where there are many: 32,768 positions of 8 heads of 128, 67 MB read and
// 134 written, 37.9 us (5.3 TB/s; through the caches 58, so too by half lines that the L2 puts together).  A word of values holds four keys of one number; four lanes turn four such words into four numbers of one key.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void read_kv_e4m3_kernel(T* k_out, T* v_out, int rows, CacheArgs a) {
  typedef unsigned uint4v __attribute__((ext_vector_type(4)));
  constexpr int COLUMNS = 1024, EACH = 16 / sizeof(T);      // numbers a store
  __shared__ __attribute__((aligned(16))) unsigned char s_codes[4][ROWS][COLUMNS + 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = (blockIdx.x * 4 + wave) * ROWS;
  if (r0 >= rows) return;
  const int d = a.d, sixteens = d >> 4, groups = (sixteens + 3) >> 2, width = a.nkv * d;
  const int n_rows = min(ROWS, rows - r0), mine = lane & (ROWS - 1);
  // (where a row has no page, page 0 is read and zeros are written; a cache without pages is not read)
  int my_off = 0;
  const int my_page = mine < n_rows ? page_of(a, r0 + mine, &my_off) : -1;
  int page[ROWS], off[ROWS];
  bool word = ROWS == 4 && n_rows == 4;
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    page[t] = __builtin_amdgcn_readlane(my_page, t);
    off[t] = __builtin_amdgcn_readlane(my_off, t);
    word = word && page[t] == page[0] && off[t] == (off[0] & ~3) + t;
  }
  const bool any = a.pages > 0;
  unsigned char(*codes)[COLUMNS + 16] = s_codes[wave];
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // columns col0 .. col0 + count - 1 of the rows, from LDS
  auto write = [&](T* out, int col0, int count, int of_values) {
    meet();
    for (int c = lane * EACH; c < count; c += 64 * EACH) {
      const int kvh = (col0 + c) / d;
      unsigned byte[ROWS];
#pragma unroll
      for (int t = 0; t < ROWS; ++t)
        byte[t] = any ? a.scale[(((size_t)max(page[t], 0) * a.nkv + kvh) * 2 + of_values) * a.page_size + off[t]] : 0;
#pragma unroll
      for (int t = 0; t < ROWS; ++t) {
        if (t >= n_rows) break;
        float x[EACH];
#pragma unroll
        for (int i = 0; i < EACH; i += 4) decode_four(*(const unsigned*)&codes[t][c + i], power_of_byte(byte[t]), page[t] >= 0, x + i);
        store_numbers<T, EACH, true, ROWS == 4>(out + (size_t)(r0 + t) * width + col0 + c, x);
      }
    }
    meet();
  };
  for (int six0 = 0; six0 < a.nkv * sixteens; six0 += COLUMNS / 16) {
    const int count = min(COLUMNS / 16, a.nkv * sixteens - six0);
    const unsigned char* from = a.k + (size_t)max(my_page, 0) * a.nkv * a.page_size * d;
#pragma unroll
    for (int i = 0; i < COLUMNS / 16 * ROWS / 64; ++i) {
      const int n = (i * 64 + lane) / ROWS, kvh = (six0 + n) / sixteens, six = six0 + n - kvh * sixteens;
      if (n < count && any)
        *(uint4v*)&codes[mine][n * 16] = *(const uint4v*)(from + (size_t)kvh * a.page_size * d + key_index(my_off, six * 16, d));
    }
    write(k_out, six0 * 16, count * 16, 0);
  }
  for (int g0 = 0; g0 < a.nkv * groups; g0 += COLUMNS / 64) {
    const int count = min(COLUMNS / 64, a.nkv * groups - g0);
    auto column = [&](int group) { return group / groups * d + group % groups * 64; };
    const int col0 = column(g0), end = g0 + count < a.nkv * groups ? column(g0 + count) : width;
    // a unit: number c of up to four 16-wide blocks
    for (int u = lane; u < count * 16; u += 64) {
      const int kvh = (g0 + (u >> 4)) / groups, g = g0 + (u >> 4) - kvh * groups, c = u & 15, wide = min(4, sixteens - 4 * g);
      unsigned char* to = &codes[0][kvh * d + g * 64 - col0];
      auto words = [&](int t, unsigned (&w)[4]) {
        const unsigned char* at = a.v + ((size_t)max(page[t], 0) * a.nkv + kvh) * a.page_size * d;
        const unsigned* src = (const unsigned*)(at + (value_index(off[t], g * 64 + c, d) & ~(size_t)3));
        if (wide == 4) {
          const uint4v x = *(const uint4v*)src;
#pragma unroll
          for (int b = 0; b < 4; ++b) w[b] = x[b];
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b) w[b] = src[min(b, wide - 1)];
        }
      };
      if (!any) continue;
      unsigned w[4];
      if (word) {
        words(0, w);
        const unsigned pick = 0x0400u + 0x0101u * (lane & 3);      // byte (lane % 4) of two words
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int v = (int)w[b];
          const unsigned x0 = __builtin_amdgcn_update_dpp(0, v, 0x00, 0xf, 0xf, true), x1 = __builtin_amdgcn_update_dpp(0, v, 0x55, 0xf, 0xf, true),
                         x2 = __builtin_amdgcn_update_dpp(0, v, 0xaa, 0xf, 0xf, true), x3 = __builtin_amdgcn_update_dpp(0, v, 0xff, 0xf, 0xf, true);
          const unsigned low = __builtin_amdgcn_perm(x1, x0, pick), high = __builtin_amdgcn_perm(x3, x2, pick);
          if (b < wide) *(unsigned*)(to + (size_t)mine * (COLUMNS + 16) + b * 16 + (c & ~3)) = __builtin_amdgcn_perm(high, low, 0x05040100u);
        }
      } else {
#pragma unroll
        for (int t = 0; t < ROWS; ++t) {
          words(t, w);
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (b < wide) to[(size_t)t * (COLUMNS + 16) + b * 16 + c] = (unsigned char)(w[b] >> (8 * (off[t] & 3)));
        }
      }
    }
    write(v_out, col0, end - col0, 1);
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
    hipLaunchKernelGGL(kernel, dim3((rows + rows_a_block - 1) / rows_a_block), dim3(64 * waves), lds, stream, x,
                       row_stride, inv_freq, y, q_stride, rows, a);
  };
  // Many rows: eight a block, a wave each, where their values' codes fit beside the sines; few: four waves a row, so that a row's chain is
  // short and the rows spread over the chip.  us of GPU, few / many: 14 heads of 64 over 2, 1,024 rows 5.7 / 6.9, 2,048 9.0 / 7.4, 8,192
  // 25.7 / 16.7; 28 of 128 over 4 9.2 / 12.9, 14.2 / 14.5, 48.8 / 38.1; 64 of 128 over 8 14.0 / 23.2, 21.3 / 24.3, 78 / 77.  float32: 14 of 64 over 2
  // 5.8 / 6.8, 9.5 / 8.2, 25.8 / 16.8; 28 of 128 over 4 9.5 / 12.6, 14.8 / 16.2, 57.2 / 61.0 (the one kind that loses a little).  (Sixteen rows a block:
  // 2,048 rows 19.2, 8,192 37.8; four: 13.8 and 40.1; two waves a row 13.2 and 45.8; all waves of a block over its rows one
  // after the other 20.8 and 45.4.)
  constexpr int MANY = 8;
  const size_t codes = (size_t)MANY * nkv * d;
  const bool many = rows >= 2048 && codes <= 31 * 1024;
  auto pick = [&](auto t) {
    typedef decltype(t) T;
    const T* x = (const T*)qkv;
    T* y = (T*)q_out;
    if (!wide) launch(rope_kv_write_e4m3_kernel<T, 1, 4, false>, 1, 4, 0, x, y);
    else if (many) launch(rope_kv_write_e4m3_kernel<T, MANY, MANY, true>, MANY, MANY, codes, x, y);
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
  // Four rows a wave once the rows fill the chip so, whatever their width (us of GPU, one / four.  bfloat16, 8 heads of 128: 2,048 rows in order
  // 8.2 / 10.5, 8,192 14.2 / 13.9, 16,384 30.5 / 19.6, 32,768 59.1 / 37.5; in any order 10.1 / 19.3, 23.9 / 27.0, 45.9 / 38.4, 82.9 / 83.3: there
  // a lane's 16 bytes of values have four of its own, and four of four rows in order.  2 heads of 64: 8,192 6.9 / 6.9 and in any order
  // 7.7 / 9.7, 16,384 11.7 / 8.3 and 12.1 / 11.5.  float32, 8 of 128: 8,192 22.6 / 21.2 and 31.6 / 35.6, 16,384 47.4 / 33.6 and 61.9 / 51.2).
  auto pick = [&](auto t) {
    typedef decltype(t) T;
    if (rows > 8192)
      hipLaunchKernelGGL((read_kv_e4m3_kernel<T, 4>), dim3((rows + 15) / 16), dim3(256), 0, stream, (T*)k_out, (T*)v_out, rows, a);
    else
      hipLaunchKernelGGL((read_kv_e4m3_kernel<T, 1>), dim3((rows + 3) / 4), dim3(256), 0, stream, (T*)k_out, (T*)v_out, rows, a);
  };
  if (dtype == DT_BF16) pick(bf16_t());
  else pick(float());
  LLMLAB_LAUNCH_CHECK("read_kv_e4m3");
  return 0;
}
