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

// A block for every row, a wave for a head at a time.
template <typename T>
__global__ __launch_bounds__(256) void rope_kv_write_e4m3_kernel(const T* qkv, size_t row_stride, const float* inv_freq,
                                                                 T* q_out, size_t q_stride, CacheArgs a) {
  extern __shared__ double turn[];       // [d / 2] cosines, [d / 2] sines
  const int r = blockIdx.x, half = a.d >> 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (inv_freq) {
    for (int i = threadIdx.x; i < half; i += blockDim.x)
      sincos((double)a.positions[r] * (double)inv_freq[i], &turn[half + i], &turn[i]);
    __syncthreads();
  }
  int off;
  const int page = page_of(a, r, &off);
  for (int head = wave; head < a.nq + 2 * a.nkv; head += waves) {
    const T* src = qkv + (size_t)r * row_stride + (size_t)head * a.d;
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.nkv;
    if (!is_q && page < 0) continue;
    float lo[2], hi[2], most = 0.f;      // (heads of up to 256: two pairs a lane)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = lane + 64 * j;
      lo[j] = hi[j] = 0.f;
      if (i >= half) continue;
      const double x = (double)to_float(src[i]), y = (double)to_float(src[i + half]);
      if (is_v || !inv_freq) {
        lo[j] = (float)x;
        hi[j] = (float)y;
      } else {
        const double c = turn[i], s = turn[half + i];
        lo[j] = to_odd(x * c - y * s);
        hi[j] = to_odd(y * c + x * s);
      }
      if (finite(lo[j])) most = fmaxf(most, fabsf(lo[j]));
      if (finite(hi[j])) most = fmaxf(most, fabsf(hi[j]));
      if (is_q) {
        T* dst = q_out + (size_t)r * q_stride + (size_t)head * a.d;
        dst[i] = from_float<T>(lo[j]);
        dst[i + half] = from_float<T>(hi[j]);
      }
    }
    if (is_q) continue;
    const int byte = scale_byte(full_wave_max(most));
    const float inv = power_of_byte(254 - byte);
    const int kvh = head - a.nq - (is_v ? a.nkv : 0);
    const size_t at = ((size_t)page * a.nkv + kvh) * a.page_size;
    unsigned char* dst = (is_v ? a.v : a.k) + at * a.d;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = lane + 64 * j;
      if (i >= half) continue;
      dst[is_v ? value_index(off, i, a.d) : key_index(off, i, a.d)] = to_code(lo[j], inv);
      dst[is_v ? value_index(off, i + half, a.d) : key_index(off, i + half, a.d)] = to_code(hi[j], inv);
    }
    if (lane == 0) a.scale[2 * at + (is_v ? a.page_size : 0) + off] = (unsigned char)byte;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void read_kv_e4m3_kernel(T* k_out, T* v_out, CacheArgs a) {
  const int r = blockIdx.x;
  int off;
  const int page = page_of(a, r, &off);
  const int width = a.nkv * a.d;
  for (int n = threadIdx.x; n < 2 * width; n += blockDim.x) {
    const bool is_v = n >= width;
    const int j = is_v ? n - width : n, head = j / a.d, i = j - head * a.d;
    float x = 0.f;
    if (page >= 0) {
      const size_t at = ((size_t)page * a.nkv + head) * a.page_size;
      const unsigned char code = (is_v ? a.v : a.k)[at * a.d + (is_v ? value_index(off, i, a.d) : key_index(off, i, a.d))];
      x = __builtin_amdgcn_cvt_f32_fp8(code, 0) * power_of_byte(a.scale[2 * at + (is_v ? a.page_size : 0) + off]);
    }
    (is_v ? v_out : k_out)[(size_t)r * width + j] = from_float<T>(x);
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
  const size_t lds = sizeof(double) * d;
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(rope_kv_write_e4m3_kernel<bf16_t>, dim3(rows), dim3(256), lds, stream, (const bf16_t*)qkv, row_stride,
                       inv_freq, (bf16_t*)q_out, q_stride, a);
  else
    hipLaunchKernelGGL(rope_kv_write_e4m3_kernel<float>, dim3(rows), dim3(256), lds, stream, (const float*)qkv, row_stride,
                       inv_freq, (float*)q_out, q_stride, a);
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
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(read_kv_e4m3_kernel<bf16_t>, dim3(rows), dim3(256), 0, stream, (bf16_t*)k_out, (bf16_t*)v_out, a);
  else
    hipLaunchKernelGGL(read_kv_e4m3_kernel<float>, dim3(rows), dim3(256), 0, stream, (float*)k_out, (float*)v_out, a);
  LLMLAB_LAUNCH_CHECK("read_kv_e4m3");
  return 0;
}
