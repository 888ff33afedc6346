// Grouped-query attention over a paged cache of 8-bit keys and values, for one head size (HEAD_DIM is
// given on the compiler's command line).  gfx950 only.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = 2^((q_r . k_j) scale log2 e - m_r),   over the keys j that row r sees,
// k_j = 2^(e_j) code_j and v_j alike (csrc/e4m3_cache.hip has the format and the pages' order).
//
// Matrix instructions in bfloat16 (v_mfma_f32_16x16x32_bf16), everything transposed so that no data moves between lanes:
//   S^T[key, row] = K . Q^T     A = 16 keys x 32 numbers, B = queries
//   O^T[d, row]   = V^T . P^T   A = 16 numbers x 32 keys, B = probabilities
// A code is a bfloat16 number and so is a code times its scale, so nothing is lost in taking them to bfloat16 in
// registers: a key's scale goes in with the conversion (one instruction makes two numbers and multiplies them), a value's
// into its probability, in float32 behind the sum of the probabilities.  The numbers of a key are taken in the order in
// which a lane's 16 bytes hold them (lane group g of a piece of 64: numbers 16 g .. 16 g + 15, the first eight in one
// product and the others in the next), and the queries alike.  Scores, maxima, exponentials and sums are float32.
//
// float32 queries are taken as three bfloat16 parts (24 bits: nothing is lost), probabilities too, each part a
// product of its own; the keys' and values' numbers are exact.
#include <type_traits>

#include "common.h"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head sizes are multiples of 16 up to 256");

constexpr int D = HEAD_DIM;
constexpr int KP = (D + 63) / 64;        // pieces of 64 numbers of a key
constexpr int DB = D / 16;               // 16-wide blocks of a value
constexpr int VG = (DB + 3) / 4;         // groups of four of them
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float LAZY_MAX = 8.f;          // slack of the running maximum, in powers of two (see below)

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max_across_rows(float v) {      // over the four lanes that share a row
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// two codes (the low or the high half of a word) to bfloat16, times a power of two
template <bool HIGH>
__device__ __forceinline__ bf16x2 two_numbers(unsigned codes, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH);
}
__device__ __forceinline__ bf16x8 eight_numbers(unsigned a, unsigned b, float scale) {
  const bf16x2 x = two_numbers<false>(a, scale), y = two_numbers<true>(a, scale), z = two_numbers<false>(b, scale),
               w = two_numbers<true>(b, scale);
  return bf16x8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
__device__ __forceinline__ float power_of_byte(unsigned b) { return __uint_as_float(b << 23); }

struct Args {
  const void* q;               // [rows, q_stride], head h at h * D
  const unsigned char* k;      // the layer's pages
  const unsigned char* v;
  const unsigned char* scale;  // [pages, nkv, 2, page_size]
  const int* table;            // [reqs, table_stride]
  const int* q_start;          // [reqs + 1]
  const int* start_pos;        // [reqs]
  void* out;                   // [rows, out_stride]
  long q_stride, out_stride;
  int table_stride, table_width, page_shift, pages;
  int nq, nkv, window, rows;
  float scale2;                // the scores' factor times log2 e
};

template <typename T>
constexpr int parts_of() { return std::is_same<T, float>::value ? 3 : 1; }

// x as PARTS bfloat16 numbers whose sum it is (to 24 bits)
template <int PARTS>
__device__ __forceinline__ void split(float x, bf16_t (&part)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    part[i] = (bf16_t)x;
    if (i + 1 < PARTS) x -= (float)part[i];
  }
}

typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// The block's waves share 16 rows (a row: a token and a head of the group that shares a kv head) and split their keys in
// steps of 32; the waves' sums meet in LDS.
constexpr int WAVES = 4;
template <typename T>
__global__ __launch_bounds__(64 * WAVES) void attention_e4m3_kernel(Args a) {
  constexpr int PARTS = parts_of<T>();
  __shared__ float s_o[WAVES][16][D + 4];
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, kvh = blockIdx.y, G = a.nq / a.nkv;
  const int r0 = a.q_start[b], count = a.q_start[b + 1] - r0, before = a.start_pos[b];
  const int total = count * G, row0 = blockIdx.x * 16;
  if (row0 >= total || r0 < 0 || count > a.rows - r0) return;
  const int last = min(row0 + 16, total) - 1;
  const int P = 1 << a.page_shift;

  // this lane's row
  const int row = row0 + c;
  const bool valid = row < total;
  const int tok = valid ? row / G : 0, head = kvh * G + (valid ? row % G : 0), pos = before + tok;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  bf16x8 qf[PARTS][KP][2];
  const T* q = (const T*)a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)head * D;
#pragma unroll
  for (int kp = 0; kp < KP; ++kp)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int dd = kp * 64 + g * 16 + h * 8 + i;
        bf16_t part[PARTS];
        split<PARTS>(valid && dd < D ? to_float(q[dd]) : 0.f, part);
#pragma unroll
        for (int n = 0; n < PARTS; ++n) qf[n][kp][h][i] = part[n];
      }

  // the keys that some row of the tile sees, and this wave's steps among them
  const int first_pos = before + row0 / G, key_hi = before + last / G;
  const int key_lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
  const int step_lo = key_lo >> 5, steps = (key_hi >> 5) - step_lo + 1;
  const int per = (steps + WAVES - 1) / WAVES;
  const int my_lo = step_lo + wave * per, my_hi = min(my_lo + per, step_lo + steps);

  floatx4 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.f;

  for (int step = my_lo; step < my_hi; ++step) {
    const int kb = step * 32;
    floatx4 s[2];
    unsigned vw[2][DB], vs[2];      // the values' codes: a word holds the four keys 4 g .. 4 g + 3 of a number
    bool there[2];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      const int key = kb + h2 * 16, slot = key >> a.page_shift;
      const int page = slot < a.table_width && key <= key_hi && key + 15 >= key_lo ? a.table[(size_t)b * a.table_stride + slot] : -1;
      there[h2] = page >= 0 && page < a.pages;
      const size_t at = ((size_t)(there[h2] ? page : 0) * a.nkv + kvh) << a.page_shift;
      const int off = key & (P - 1);
      const unsigned char* kp = a.k + at * D + (size_t)off * D;
      const unsigned char* vp = a.v + at * D + (size_t)off * D;
      const unsigned char* sp = a.scale + 2 * at + off;
      s[h2] = floatx4{0.f, 0.f, 0.f, 0.f};
      vs[h2] = 0;
#pragma unroll
      for (int db = 0; db < DB; ++db) vw[h2][db] = 0;
      if (!there[h2]) continue;
      const float ks = power_of_byte(sp[c]);
      vs[h2] = *(const unsigned*)(sp + P + 4 * g);
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int sixteen = i * 4 + g;      // (past the last: the queries are zero there)
        const uint4v w = *(const uint4v*)(kp + (size_t)(min(sixteen, D / 16 - 1) * 16 + c) * 16);
        const bf16x8 k0 = eight_numbers(w[0], w[1], ks), k1 = eight_numbers(w[2], w[3], ks);
#pragma unroll
        for (int n = PARTS - 1; n >= 0; --n) {
          s[h2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[n][i][0], s[h2], 0, 0, 0);
          s[h2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[n][i][1], s[h2], 0, 0, 0);
        }
      }
#pragma unroll
      for (int vg = 0; vg < VG; ++vg) {
        constexpr int FULL = 4;
        const int wide = DB - 4 * vg < FULL ? DB - 4 * vg : FULL;
        const unsigned* wp = (const unsigned*)(vp + vg * 1024 + (size_t)(g * 16 + c) * wide * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (vg * 4 + j < DB) vw[h2][vg * 4 + j] = wp[j];
      }
    }
    const bool masked = !(there[0] && there[1] && kb + 31 <= first_pos && (a.window <= 0 || kb >= key_hi - a.window + 1));
    float p[8];
    float mx = NEG_INF;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = kb + (i >> 2) * 16 + g * 4 + (i & 3);
      const bool sees = there[i >> 2] && valid && j <= pos && j >= lo;
      p[i] = sees ? s[i >> 2][i & 3] * a.scale2 : NEG_INF;
      mx = fmaxf(mx, p[i]);
    }
    mx = max_across_rows(mx);
    // The maximum is raised only when a score exceeds it by more than LAZY_MAX: until then p may be as large as 2^8,
    // which float32 sums and bfloat16 probabilities hold without loss, and rescaling the sums is rare.
    const bool grow = mx > m + LAZY_MAX;
    if (__any(grow)) {
      const float m_new = grow ? mx : m, alpha = grow ? fast_exp2(m - m_new) : 1.f;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      m = m_new;
    }
    const float neg_m = m == NEG_INF ? 0.f : -m;      // (no key seen yet: every p is 2^-inf = 0)
    bf16x8 pf[PARTS];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = fast_exp2(p[i] + neg_m);
      l += p[i];
      const int j = kb + (i >> 2) * 16 + g * 4 + (i & 3);
      const bool sees = there[i >> 2] && valid && j <= pos && j >= lo;      // (the scale of another place is not used)
      const float w = sees ? p[i] * power_of_byte((vs[i >> 2] >> (8 * (i & 3))) & 255u) : 0.f;
      bf16_t part[PARTS];
      split<PARTS>(w, part);
#pragma unroll
      for (int n = 0; n < PARTS; ++n) pf[n][i] = part[n];
    }
    // Places that a row does not see may hold codes that are not numbers, which their probability of zero does not
    // keep out of the product: they become zeros, and the rows that do see them become no numbers.
    bool strange = false;
    if (masked) {
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const unsigned x = vw[h2][db] & 0x7f7f7f7fu;
          strange |= ((x + 0x01010101u) & 0x80808080u) != 0;
        }
      strange = __any(strange);
    }
    if (strange) {
      bf16x8 ind;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = kb + (i >> 2) * 16 + g * 4 + (i & 3);
        ind[i] = there[i >> 2] && valid && j <= pos && j >= lo ? (bf16_t)1.f : (bf16_t)0.f;
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        bf16x8 bad;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned shift = 8 * (i & 3);
          const bool nan = ((vw[i >> 2][db] >> shift) & 0x7fu) == 0x7fu;
          bad[i] = nan ? (bf16_t)1.f : (bf16_t)0.f;
          if (nan) vw[i >> 2][db] &= ~(0xffu << shift);
        }
        const floatx4 hits = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad, ind, floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hits[i] > 0.f) o[db][i] = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const bf16x8 vf = eight_numbers(vw[0][db], vw[1][db], 1.f);
#pragma unroll
      for (int n = PARTS - 1; n >= 0; --n) o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], o[db], 0, 0, 0);
    }
  }

  // a row's four lanes hold its keys' sums, every lane the numbers 16 db + 4 g + i of its row
  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);
  if (g == 0) {
    s_m[wave][c] = m;
    s_l[wave][c] = l;
  }
#pragma unroll
  for (int db = 0; db < DB; ++db) *(floatx4*)&s_o[wave][c][db * 16 + g * 4] = o[db];
  __syncthreads();
  for (int n = threadIdx.x; n < 16 * D; n += 64 * WAVES) {
    const int r = n / D, i = n - r * D;
    if (row0 + r >= total) continue;
    float top = NEG_INF;
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_m[w][r]);
    float sum = 0.f, weight = 0.f;
    for (int w = 0; w < WAVES; ++w) {
      // (no maximum: no key that the row sees, sums of zero, or scores that are no numbers, and sums likewise)
      const float f = s_m[w][r] == NEG_INF ? 1.f : fast_exp2(s_m[w][r] - top);
      sum += f * s_o[w][r][i];
      weight += f * s_l[w][r];
    }
    const int t = (row0 + r) / G, h = kvh * G + (row0 + r) % G;
    ((T*)a.out)[(size_t)(r0 + t) * a.out_stride + (size_t)h * D + i] = from_float<T>(weight > 0.f || weight != weight ? sum / weight : 0.f);
  }
}

extern "C" const char* llmlab_last_error() { return g_llmlab_error; }
extern "C" int llmlab_attention_head_dim() { return D; }

extern "C" int llmlab_paged_attention_e4m3(const void* q, int dtype, long q_stride, int nq, int nkv, const void* k, const void* v,
                                           const void* kv_scale, int pages, const int* table, int table_stride, int table_width,
                                           int page_size, const int* q_start, const int* start_pos, int reqs, int max_q_len,
                                           int max_ctx_len, int window, float scale, void* out, long out_stride, int rows,
                                           hipStream_t stream) {
  LLMLAB_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "attention(e4m3): %d heads, %d kv heads", nq, nkv);
  LLMLAB_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "attention(e4m3): page size %d is not a power of two >= 16",
                 page_size);
  LLMLAB_REQUIRE(q_stride >= (long)nq * D && out_stride >= (long)nq * D, "attention(e4m3): row strides too small");
  LLMLAB_REQUIRE(reqs >= 0 && reqs <= 65535, "attention(e4m3): %d requests, at most 65535 are taken", reqs);
  LLMLAB_REQUIRE(window >= 0, "attention(e4m3): negative window");
  LLMLAB_REQUIRE(scale > 0.f, "attention(e4m3): the score scale must be positive, got %g", (double)scale);
  LLMLAB_REQUIRE(((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0 && ((uintptr_t)kv_scale % 4) == 0,
                 "attention(e4m3): the pages are not aligned for vector loads");
  if (reqs == 0 || max_q_len <= 0 || rows == 0) return 0;
  Args a{q, (const unsigned char*)k, (const unsigned char*)v, (const unsigned char*)kv_scale, table, q_start, start_pos, out,
         q_stride, out_stride, table_stride, table_width, 0, pages, nq, nkv, window, rows, scale * 1.4426950408889634f};
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  const long most_rows = (long)max_q_len * (nq / nkv);
  const dim3 grid((unsigned)((most_rows + 15) / 16), nkv, reqs);
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(attention_e4m3_kernel<bf16_t>, grid, dim3(64 * WAVES), 0, stream, a);
  else
    hipLaunchKernelGGL(attention_e4m3_kernel<float>, grid, dim3(64 * WAVES), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("attention(e4m3)");
  return 0;
}
