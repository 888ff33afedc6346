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
// product and the others in the next), and the queries alike.  Scores, maxima, exponentials and sums are float32.  A probability
// times its value's scale goes into the product as bfloat16: of rows in one tile of 16 or 32 as two numbers (what is left out is 2^-16 of
// it, so that the output's own rounding is all that counts: 0.0017 off 64 bits), of more rows rounded once, as in the attention over
// bfloat16 pages (half a step, up to 2^-8 of itself: outputs 0.0022 off 64 bits).
//
// float32 queries are taken as three bfloat16 parts (24 bits: nothing is lost), probabilities too, each part a
// product of its own; the keys' and values' numbers are exact.
#include <algorithm>
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
constexpr float LARGE = 1.7014118346046923e38f;      // 2^127
constexpr float LOWEST = -3.40282347e38f;            // a row's maximum once it saw a key (minus infinity: it saw none)
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
  int last_key;                // the last that the table has room for (-1: no walk, nothing of the cache is read)
  int nq, nkv, window, rows, reqs, splits;
  int covered;                 // rows (token, head of a group) of a request that the launch has tiles for
  float scale2;                // the scores' factor times log2 e
  float* o_part;               // [rows * nq, splits, D]    (splits > 1)
  float* ml_part;              // [rows * nq, splits, 2]
};

// Four numbers of a row's output: its sums over the sum of its probabilities, zero where it saw no key.  (A row that saw keys, all with a
// score of minus infinity, has sums of zero and a maximum of LOWEST: 0 / 0 is no number.)
template <typename T>
__device__ __forceinline__ void write_output(const Args& a, int row, int head, int i, floatx4 sum, float weight, float most) {
  typedef T vec __attribute__((ext_vector_type(4)));      // (outputs begin at 16 bytes, and their rows)
  const bool any = most != NEG_INF;
  const float inv = 1.f / weight;
  vec v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = from_float<T>(!any ? 0.f : sizeof(T) == 4 ? sum[j] / weight : sum[j] * inv);
  *(vec*)((T*)a.out + (size_t)row * a.out_stride + (size_t)head * D + i) = v;
}

// The request that is the number-th by the length of its context, the longest first (at most 64 requests; every lane the same)
struct Request {
  int b, r0, count, before;
};
__device__ __forceinline__ Request longest(const Args& a, int number) {
  const int lane = threadIdx.x & 63, i = min(lane, a.reqs - 1);
  const int start = a.q_start[i], rows = a.q_start[i + 1] - start, past = a.start_pos[i], end = past + rows;
  int ahead = 0;      // requests in front of the lane's
  for (int j = 0; j < a.reqs; ++j) {
    const int other = __builtin_amdgcn_readlane(end, j);
    ahead += other > end || (other == end && j < lane);
  }
  const int b = __ffsll(__ballot(lane < a.reqs && ahead == number)) - 1;
  return Request{b, __builtin_amdgcn_readlane(start, b), __builtin_amdgcn_readlane(rows, b), __builtin_amdgcn_readlane(past, b)};
}

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

// What a step of 32 keys reads: of each of its two blocks of 16 keys the codes of the keys and values and their scales'
// bytes (a lane's key's, and those of its four values).
struct Step {
  uint4v k[2][KP];
  unsigned v[2][DB];      // a word: the four keys 4 g .. 4 g + 3 of a number
  unsigned ks[2], vs[2];
  bool there[2];
};

// The rows of one tile as a lane has them (row 16 qb + lane % 16), and what is summed for them so far.
template <int QB, int PARTS>
struct Rows {
  int lo[QB];            // the first key that the row sees (a row past the last, or in front of all keys: behind all keys)
  unsigned span[QB];     // and how many follow it
  bf16x8 q[QB][PARTS][KP][2];
  floatx4 o[QB][DB];
  float m[QB], l[QB];
};

template <typename T, int QB, int PARTS>
__device__ __forceinline__ void load_rows(const Args& a, Rows<QB, PARTS>& r, int r0, int before, int kvh, int row0, int total, int c,
                                          int g) {
  const int G = a.nq / a.nkv;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = row0 + qb * 16 + c;
    const bool valid = row < total;
    const int tok = valid ? row / G : 0, head = kvh * G + (valid ? row - tok * G : 0), pos = valid ? before + tok : -1;
    r.lo[qb] = pos < 0 ? 1 << 30 : a.window > 0 ? max(0, pos - a.window + 1) : 0;
    r.span[qb] = pos < 0 ? 0 : pos - r.lo[qb];
    const T* q = (const T*)a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)head * D;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int dd = kp * 64 + g * 16 + h * 8;
        const bool in = valid && dd < D;      // (D is a multiple of 16: eight numbers are in or out together)
        if constexpr (PARTS == 1) {
          const bf16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
          const bf16x8 x = *(const bf16x8*)(q + (in ? dd : 0));
          r.q[qb][0][kp][h] = in ? x : zero;
        } else {
          const floatx4 x = *(const floatx4*)(q + (in ? dd : 0)), y = *(const floatx4*)(q + (in ? dd + 4 : 4));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            bf16_t part[PARTS];
            split<PARTS>(in ? (i < 4 ? x[i & 3] : y[i & 3]) : 0.f, part);
#pragma unroll
            for (int n = 0; n < PARTS; ++n) r.q[qb][n][kp][h][i] = part[n];
          }
        }
      }
    r.m[qb] = NEG_INF;
    r.l[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) r.o[qb][db] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
}

// One step of 32 keys from kb on for every row of the tile.  MASKED: some row does not see some key.  P_PARTS: the bfloat16 numbers
// that a probability is taken as.  The running maximum is kept in the units of the exponent and is raised only when a score exceeds it by more than LAZY_MAX: until then p may
// be as large as 2^8, which changes no rounding (bfloat16 has float32's exponents), and rescaling the sums is rare.
template <bool MASKED, int QB, int PARTS, int P_PARTS>
__device__ __forceinline__ void add_step(const Args& a, Rows<QB, PARTS>& r, Step& f, int kb, int g) {
  floatx4 s[2][QB];
#pragma unroll
  for (int h2 = 0; h2 < 2; ++h2) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) s[h2][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
    const float ks = power_of_byte(f.ks[h2]);
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const uint4v w = f.k[h2][i];
      const bf16x8 k0 = eight_numbers(w[0], w[1], ks), k1 = eight_numbers(w[2], w[3], ks);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int n = PARTS - 1; n >= 0; --n) {
          s[h2][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, r.q[qb][n][i][0], s[h2][qb], 0, 0, 0);
          s[h2][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, r.q[qb][n][i][1], s[h2][qb], 0, 0, 0);
        }
    }
  }
  float vs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned byte = (f.vs[i >> 2] >> (8 * (i & 3))) & 255u;
    vs[i] = power_of_byte(MASKED ? min(byte, 254u) : byte);      // (finite where it may be any byte: times a probability of zero it is zero)
  }
  auto key = [&](int i) { return kb + (i >> 2) * 16 + g * 4 + (i & 3); };
  auto sees = [&](int qb, int i) { return f.there[i >> 2] && (unsigned)(key(i) - r.lo[qb]) <= r.span[qb]; };
  bf16x8 pf[QB][P_PARTS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float p[8];
    bool some = !MASKED;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool seen = !MASKED || sees(qb, i);
      some |= seen;
      p[i] = seen ? s[i >> 2][qb][i & 3] : NEG_INF;
    }
    r.m[qb] = fmaxf(r.m[qb], some ? LOWEST : NEG_INF);      // (each of the row's lanes for itself)
    float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), p[2]), fmaxf(fmaxf(p[3], p[4]), fmaxf(fmaxf(p[5], p[6]), p[7])));
    if (__any(mx * a.scale2 > r.m[qb] + LAZY_MAX)) {      // some row's maximum grew: rescale what is summed so far
      mx = max_across_rows(mx) * a.scale2;
      const bool grow = mx > r.m[qb] + LAZY_MAX;
      const float m_new = grow ? mx : r.m[qb], alpha = grow ? fast_exp2(r.m[qb] - m_new) : 1.f;
      r.l[qb] *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) r.o[qb][db] *= alpha;
      r.m[qb] = m_new;
    }
    const float neg_m = -fmaxf(r.m[qb], LOWEST);      // (no score above it yet: every p is 2^-inf = 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = fast_exp2(fmaf(p[i], a.scale2, neg_m));
    r.l[qb] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16_t part[P_PARTS];
      split<P_PARTS>(p[i] * vs[i], part);
#pragma unroll
      for (int n = 0; n < P_PARTS; ++n) pf[qb][n][i] = part[n];
    }
  }
  // Places that a row does not see may hold codes that are not numbers, which their probability of zero does not keep
  // out of the product: they become zeros, and the rows that do see them become no numbers: infinity (a product too large for
  // float32, where place and row meet) and minus infinity are added to their sums.
  if constexpr (MASKED) {
    bool strange = false;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
      for (int db = 0; db < DB; ++db) strange |= (((f.v[h2][db] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    if (__any(strange)) {
      bf16x8 up[QB], down[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          up[qb][i] = sees(qb, i) ? (bf16_t)LARGE : (bf16_t)0.f;
          down[qb][i] = -up[qb][i];
        }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        bf16x8 bad;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned shift = 8 * (i & 3);
          const bool nan = ((f.v[i >> 2][db] >> shift) & 0x7fu) == 0x7fu;
          bad[i] = nan ? (bf16_t)LARGE : (bf16_t)0.f;
          if (nan) f.v[i >> 2][db] &= ~(0xffu << shift);
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          r.o[qb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad, up[qb], r.o[qb][db], 0, 0, 0);
          r.o[qb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad, down[qb], r.o[qb][db], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const bf16x8 vf = eight_numbers(f.v[0][db], f.v[1][db], 1.f);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int n = P_PARTS - 1; n >= 0; --n) r.o[qb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[qb][n], r.o[qb][db], 0, 0, 0);
  }
}

// Few rows a request: NW waves share a tile of 16 QB rows (a row: a token and a head of the group that shares a kv head) and
// split the block's keys in steps of 32; their sums meet in LDS.  The keys of a tile are split over a.splits blocks as
// well, whose sums a kernel of its own puts together.  Bound by the reading of the codes where a request brings a token or a few: 64 requests
// of 28 heads of 128 over 4 at up to 4,096 keys (197 MB) 42 us of kernel (4.7 TB/s), 8 at 32,768 40 and 4.6 of the merge; 32 of
// 5 tokens of 40 heads over 8 at 2,500 (124 MB) 31.5 (30 with probabilities of one part).  float32 rows by their products, three a part:
// 7 of 61 tokens of 16 heads over 2 through a window of 1,000 22 us.
template <int QB, int NW>
constexpr int split_lds_floats() { return NW * 16 * QB * (D + 4) + 2 * NW * 16 * QB; }

// The waves that a SIMD is to hold: as many as fit without a spilled register (a wave more, with five to eight spilled, changed
// nothing at heads of 64 and 128).
constexpr int split_waves(int qb, int parts) {
  if (qb == 1 && parts == 1) return D <= 64 ? 4 : D <= 112 ? 3 : D <= 128 ? 2 : 1;
  return D <= (qb == 2 ? 48 : 64) ? 3 : D <= 128 ? 2 : 1;
}
template <typename T, int QB, int NW, int P_PARTS>
__global__ __launch_bounds__(64 * NW, split_waves(QB, parts_of<T>())) void attention_e4m3_split_kernel(Args a) {
  constexpr int PARTS = parts_of<T>(), TR = 16 * QB, RS = D + 4;
  __shared__ __attribute__((aligned(16))) float lds[split_lds_floats<QB, NW>()];
  float* s_m = lds + NW * TR * RS;
  float* s_l = s_m + NW * TR;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, kvh = blockIdx.y / a.splits, part = blockIdx.y % a.splits, G = a.nq / a.nkv;
  const int r0 = a.q_start[b], count = a.q_start[b + 1] - r0, before = a.start_pos[b];
  const int total = count * G, row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * TR;      // (the longest histories first)
  if (row0 >= total || r0 < 0 || count > a.rows - r0) return;
  const int last = min(row0 + TR, total) - 1;
  const int P = 1 << a.page_shift;
  Rows<QB, PARTS> r;
  load_rows<T, QB, PARTS>(a, r, r0, before, kvh, row0, total, c, g);

  // the keys that some row of the tile sees, this block's steps of 32 among them, and this wave's
  const int first_pos = before + row0 / G, key_hi = before + last / G;
  const int key_lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
  const int full_lo = a.window > 0 ? max(0, key_hi - a.window + 1) : 0;      // from here on every row sees a key before first_pos
  const int step_lo = key_lo >> 5, step_hi = (min(key_hi, a.last_key) >> 5) + 1;
  const int per = (step_hi - step_lo + a.splits - 1) / a.splits;
  const int blk_lo = step_lo + part * per, blk_hi = min(blk_lo + per, step_hi);
  const int per_wave = (max(blk_hi - blk_lo, 0) + NW - 1) / NW;
  const int my_lo = blk_lo + wave * per_wave, my_hi = min(my_lo + per_wave, blk_hi);

  // The page numbers of up to 32 steps are read ahead, a block of 16 keys a lane; the loads of the next step are in
  // flight while one is computed.  A page that is not there is read as page 0 and its keys are seen by nobody.
  for (int base = my_lo; base < my_hi; base += 32) {
    const int end = min(base + 32, my_hi);
    int page_v = -1;
    {
      const int key = base * 32 + lane * 16, slot = key >> a.page_shift;
      if (key <= key_hi && key + 15 >= key_lo && slot < a.table_width) page_v = a.table[(size_t)b * a.table_stride + slot];
      if (page_v >= a.pages) page_v = -1;
    }
    auto fetch = [&](int step, Step& f) {
      const int st = min(step, end - 1);
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const int page = __builtin_amdgcn_readlane(page_v, (st - base) * 2 + h2);
        f.there[h2] = page >= 0;
        const size_t at = ((size_t)max(page, 0) * a.nkv + kvh) << a.page_shift;
        const int off = (st * 32 + h2 * 16) & (P - 1);
        const unsigned char* kp = a.k + (at + off) * D + lane * 16;
        const unsigned char* vp = a.v + (at + off) * D;
        const unsigned char* sp = a.scale + 2 * at + off;
#pragma unroll
        for (int i = 0; i < KP; ++i)      // (a sixteen past the last: the queries are zero there)
          f.k[h2][i] = *(const uint4v*)(kp + (D % 64 == 0 ? i * 1024 : (min(i * 4 + g, D / 16 - 1) - g) * 256));
#pragma unroll
        for (int vg = 0; vg < VG; ++vg) {
          const int wide = DB - 4 * vg < 4 ? DB - 4 * vg : 4;
          const unsigned* wp = (const unsigned*)(vp + vg * 1024 + lane * wide * 4);
          if (wide == 4) {
            const uint4v w = *(const uint4v*)wp;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (vg * 4 + j < DB) f.v[h2][vg * 4 + j] = w[j];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (vg * 4 + j < DB) f.v[h2][vg * 4 + j] = wp[j];
          }
        }
        f.ks[h2] = sp[c];
        f.vs[h2] = *(const unsigned*)(sp + P + 4 * g);
      }
    };
    Step next;
    fetch(base, next);
    for (int step = base; step < end; ++step) {
      Step cur = next;
      fetch(step + 1, next);
      __builtin_amdgcn_sched_barrier(0);
      const int kb = step * 32;
      if (cur.there[0] && cur.there[1] && kb + 31 <= first_pos && kb >= full_lo)      // (rows past the last are not stored)
        add_step<false, QB, PARTS, P_PARTS>(a, r, cur, kb, g);
      else
        add_step<true, QB, PARTS, P_PARTS>(a, r, cur, kb, g);
    }
  }

  // a row's four lanes hold its keys' sums, every lane the numbers 16 db + 4 g + i of its row
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float l = r.l[qb];
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    const float m = max_across_rows(r.m[qb]);
    if (g == 0) {
      s_m[wave * TR + qb * 16 + c] = m;
      s_l[wave * TR + qb * 16 + c] = l;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) *(floatx4*)&lds[(wave * TR + qb * 16 + c) * RS + db * 16 + g * 4] = r.o[qb][db];
  }
  __syncthreads();
  const int rows = last - row0 + 1;
  for (int n = threadIdx.x; n < rows * (D / 4); n += 64 * NW) {
    const int row = n / (D / 4), i = (n - row * (D / 4)) * 4;
    float top = NEG_INF;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, s_m[w * TR + row]);
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    float weight = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      // (no maximum: no key that the row sees, and sums of zero)
      const float m = s_m[w * TR + row], f = m == NEG_INF ? 1.f : fast_exp2(m - top);
      sum += f * *(const floatx4*)&lds[(w * TR + row) * RS + i];
      weight += f * s_l[w * TR + row];
    }
    const int tok = (row0 + row) / G, head = kvh * G + (row0 + row) - tok * G;
    const size_t at = (size_t)(r0 + tok) * a.nq + head;
    if (a.splits > 1) {
      *(floatx4*)(a.o_part + (at * a.splits + part) * D + i) = sum;
      if (i == 0) {
        a.ml_part[(at * a.splits + part) * 2] = top;
        a.ml_part[(at * a.splits + part) * 2 + 1] = weight;
      }
    } else {
      write_output<T>(a, r0 + tok, head, i, sum, weight, top);
    }
  }
}

// ------------------------------------------------------------- many rows, codes staged in LDS
// Heads up to 128.  A block has RT tiles of 32 rows side by side, and P groups of waves that
// take the staged keys in turn, 32 of every 32 P; the groups' sums meet in LDS at the end.  The codes come by direct loads
// into LDS, in the cache's order, in two stages, one being multiplied while the other is on its way, one barrier a
// stage, and become bfloat16 numbers behind the read from LDS: half the bytes there and on the way.  Products by
// v_mfma_f32_32x32x16_bf16, transposed as above (lane l: row l % 32 of the tile, h = l / 32):
//   S^T[key, row] = K . Q^T: element i of the 32 keys of a step is key 8 (i / 4) + 4 h + i % 4; a lane has the numbers
//     16 (2 j + h) .. + 15 of its key, in two products, and the queries lie alike;
//   O^T[d, row] = V^T . P^T: the keys of a block of 16 in the order {4 h .. + 3, 8 + 4 h .. + 3} for half h, which is what
//     a lane holds of S^T; product i of a group of 64 numbers takes its 16-wide blocks i and 2 + i, as 8 bytes a lane
//     hold blocks 0 and 1 (lanes 0 .. 15 of a half) or 2 and 3; a last group of fewer blocks alike, by words.
// In LDS a block of 16 keys (or values) begins at a whole KB; where a head is no multiple of 64 the lanes past its end bring its last 16
// bytes again, which nobody reads.
// Every wave brings the scales of its group's keys itself, and makes float32 numbers of the values' ones in LDS.
//
// What bounds it: the vector unit beside the matrix cores.  A step of a wave, 32 keys by 32 rows at heads of 128, is 16 matrix
// instructions (512 clocks of a SIMD) and some 170 others (680 and more), 64 of them conversions; three portions of 1,000 tokens behind
// up to 3,000 keys (28 heads of 128 over 4, 121 GFLOP) take 145 to 148 us (0.82 to 0.83 PFLOP/s), 62 % of the clocks in vector and 36 % in
// matrix instructions, a sixth without a block.  A probability is one bfloat16 number: two take 192 us, one of half precision in units of
// the largest value's scale 152 to 154 and a second path where scales differ much.  Numbers made bfloat16 on the way into LDS, once for a
// block: slower (366 us, its loads through registers).  Products in 8 bits, with the queries as two parts: exact products, but sums kept to 16 bits (measured:
// 2^-16 of the sum of sizes), so not used.  float32 rows take three products a part of what they read, and as many conversions of codes as one:
// 7 requests of 700 tokens, 56 heads of 128 over 8, up to 1,400 keys 273 us (split over waves 439).
#define STAGED (HEAD_DIM <= 128)
#if STAGED
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;

// 16 bytes (a word) a lane from the cache to consecutive memory of LDS.  One statement with the m0 that the load reads:
// between two the compiler may use m0 itself.  The compiler does not see into the statements, so the five wait
// states that a load needs behind a vector instruction which wrote its scalar address (a v_readlane that brings back a
// spilled pointer, say) are in them.
__device__ __forceinline__ void load_1k(unsigned lane_offset, const unsigned char* base, unsigned to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_offset), "s"(base), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void load_words(unsigned lane_offset, const unsigned char* base, unsigned to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dword %0, %1" : : "v"(lane_offset), "s"(base), "s"(to) : "memory", "m0");
}
// A number of the block table, waited for on the spot (the compiler, which does not see it, would wait for all loads on
// their way wherever a branch with a load of its own ends)
__device__ __forceinline__ int table_entry(const int* table, int at) {
  int v;
  asm volatile("s_nop 4\n\tglobal_load_dword %0, %1, %2\n\ts_waitcnt vmcnt(0)" : "=&v"(v) : "v"(at * 4), "s"(table) : "memory");
  return v;
}

constexpr int PB = (D + 63) / 64, BLOCK = PB * 1024;             // loads of 1 KB, and bytes in LDS, of 16 keys
constexpr int FULL = D / 64, REST = D / 16 % 4;                  // groups of four 16-wide blocks of a value, and blocks of the last one
constexpr int REST_DV = (REST + 1) / 2, DV = 2 * FULL + REST_DV; // products of the last group, of all
constexpr int GROUPS = FULL + (REST > 0);

template <int RT, int P>
struct StagedSizes {
  static constexpr int NW = RT * P, KT = 32 * P;
  static constexpr int V_AT = KT / 16 * BLOCK, SCALES_AT = 2 * V_AT, STAGE = SCALES_AT + NW * 512;
  static constexpr int STAGES = 2 * STAGE, SUMS = RT * (P - 1) * DV * 4096;
  static constexpr int LDS = (STAGES > SUMS ? STAGES : SUMS) + NW * 32 * 4 * 3;
};

// The waves that a SIMD is to hold, as many as fit without a spilled register
constexpr int staged_waves(int parts, int groups) {
  if (parts > 1) return D <= 64 ? 3 : 2;
  return D <= 64 ? 4 : groups < 4 && REST != 3 ? 3 : 2;
}

template <typename T, int RT, int P>
__global__ __launch_bounds__(64 * RT * P, staged_waves(parts_of<T>(), P)) void attention_e4m3_staged_kernel(Args a, int tiles,
                                                                                                           int by_requests) {
  typedef StagedSizes<RT, P> Z;
  constexpr int PARTS = parts_of<T>();
  constexpr int NW = Z::NW, KT = Z::KT, DK = D / 16, DJ = (DK + 1) / 2;
  constexpr int PIECES = KT / 16 * PB;                           // loads of 1 KB of a stage's keys, and of its values
  constexpr int EACH = PIECES * 2 / NW;                          // ... of a wave
  constexpr int HALF = EACH > 1 ? EACH / 2 : 1;                  // ... of keys, and of values (one: keys by even waves)
  constexpr int BLOCKS = HALF > PB ? HALF / PB : 1;              // blocks of 16 that a wave's pieces belong to
  static_assert(EACH * NW == PIECES * 2 && (EACH == 1 || EACH % 2 == 0), "whole loads a wave");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Z::LDS];
  float* const own = (float*)(lds + (Z::STAGES > Z::SUMS ? Z::STAGES : Z::SUMS));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rt = wave % RT, ph = wave / RT, col = lane & 31, h = lane >> 5, odd = (lane >> 4) & 1, c = lane & 15;
  const int G = a.nq / a.nkv;
  // The tiles with the longest histories first, so that the short ones fill what those leave: by tiles, or, where what is before the
  // portions decides, by requests, those with the longest contexts first (more blocks than x takes: tiles, kv heads, requests)
  int b = blockIdx.z, kvh = blockIdx.y, rank = blockIdx.x, r0, count, before;
  if (by_requests) {
    const int per = tiles * a.nkv, number = rank / per, at = rank - number * per;
    const Request r = longest(a, number);
    b = r.b;
    r0 = r.r0;
    count = r.count;
    before = r.before;
    kvh = at % a.nkv;
    rank = at / a.nkv;
  } else {
    if (gridDim.y == 1 && gridDim.z == 1) {
      const int per = a.nkv * a.reqs, at = rank % per;
      rank /= per;
      kvh = at % a.nkv;
      b = at / a.nkv;
    }
    r0 = a.q_start[b];
    count = a.q_start[b + 1] - r0;
    before = a.start_pos[b];
  }
  const int total = count * G, block_row0 = (tiles - 1 - rank) * RT * 32;
  if (block_row0 >= total || r0 < 0 || count > a.rows - r0) return;
  const int row0 = block_row0 + rt * 32, row = row0 + col;
  const bool valid = row < total;
  const int tok = valid ? row / G : 0, head = kvh * G + (valid ? row - tok * G : 0);
  // (a key is seen if it is no further than pos - lo behind lo: one comparison; a row that sees none has its lo behind all keys)
  const int pos = valid ? before + tok : -1, lo = pos < 0 ? 1 << 30 : a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int lane_key = 4 * h - lo;
  const unsigned span = pos < 0 ? 0 : pos - lo;
  // the keys that the block's rows see; up to p_first and from full_lo on every row of the wave sees them
  const int last = min(row0 + 32, total) - 1, block_last = min(block_row0 + RT * 32, total) - 1;
  const int p_first = before + row0 / G, p_last = row0 < total ? before + last / G : -1;
  const int full_lo = a.window > 0 ? max(0, p_last - a.window + 1) : 0;
  const int key_hi = max(min(before + block_last / G, a.last_key), 0);
  const int key_lo = a.window > 0 ? min(max(0, before + block_row0 / G - a.window + 1), key_hi) : 0;
  const int tile_lo = key_lo / KT, tile_hi = key_hi / KT;
  const int block_lo = key_lo & ~15, block_hi = key_hi & ~15;

  // Of 64 tiles at a time, tile base + l in lane l: where the blocks of 16 keys are that the wave brings, counted in such
  // blocks, and where the scales of its group's two, counted in 16 bytes; negative: not there, read as page 0 and seen
  // by nobody.  Blocks that no row sees read one that some row does.
  const int* const table = a.table + (size_t)b * a.table_stride;
  const int shift = a.page_shift, page_blocks = 1 << (shift - 4);
  const int piece0 = EACH > 1 ? wave * HALF : wave >> 1;
  constexpr unsigned HERE = 0x7fffffffu;
  unsigned where[BLOCKS], scales_where[2];
  int base = tile_lo;
  auto locate = [&](int from) {
    base = from;
    auto block_at = [&](int block16, bool of_scales) {
      const int own = min(from + lane, tile_hi) * KT + block16 * 16, key = max(min(own, block_hi), block_lo), at = key >> shift;
      int page = -1;
      if (a.table_width > 0) page = table_entry(table, min(at, a.table_width - 1));
      const bool there = own <= block_hi && at < a.table_width && page >= 0 && page < a.pages;
      const unsigned row = (unsigned)(there ? page : 0) * a.nkv + kvh;
      return (row * (of_scales ? 2 : 1) * page_blocks + ((key >> 4) & (page_blocks - 1))) | (there ? 0u : ~HERE);
    };
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) where[n] = block_at(piece0 / PB + n, false);
#pragma unroll
    for (int n = 0; n < 2; ++n) scales_where[n] = block_at(ph * 2 + n, true);
  };
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const unsigned scales_from = (lane & 3) * 4 + (lane >> 2 & 1) * page_blocks * 16;      // a word of the keys' or the values' scales
  // (the result: which blocks of the wave's group are there)
  auto fetch = [&](int tile, int slot) {
    if (tile - base >= 64) locate(tile);
    const unsigned to = lds0 + slot * Z::STAGE;
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) {
      const unsigned block = (unsigned)__builtin_amdgcn_readlane((int)where[n], tile - base) & HERE;
      const size_t at = (size_t)block * (16 * D) + piece0 % PB * 1024;
#pragma unroll
      for (int i = 0; i < HALF / BLOCKS; ++i) {
        const unsigned to_piece = to + (piece0 + n * PB + i) * 1024;
        const unsigned from = D % 64 == 0 ? lane * 16 : min(lane * 16, 16 * D - 16 - (piece0 % PB + i) * 1024);
        if constexpr (EACH > 1) {
          load_1k(from, a.k + at + i * 1024, to_piece);
          load_1k(from, a.v + at + i * 1024, to_piece + Z::V_AT);
        } else {
          load_1k(from, (wave & 1 ? a.v : a.k) + at, wave & 1 ? to_piece + Z::V_AT : to_piece);
        }
      }
    }
    unsigned there = 0;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const unsigned at = (unsigned)__builtin_amdgcn_readlane((int)scales_where[n], tile - base);
      there |= at <= HERE ? 1u << n : 0u;
      load_words(scales_from, a.scale + (size_t)(at & HERE) * 16, to + Z::SCALES_AT + wave * 512 + n * 256);
    }
    return there;
  };

  // (a sixteen past the last: its keys' last one, times zero)
  bf16x8 q[PARTS][2 * DJ];
  const T* qp = (const T*)a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)head * D;
  auto in = [&](int k) { return valid && (DK % 2 == 0 || (k >> 1) * 2 + h < DK); };
  auto at = [&](int k) { return qp + min((k >> 1) * 2 + h, DK - 1) * 16 + (k & 1) * 8; };
  if constexpr (PARTS == 1) {
#pragma unroll
    for (int k = 0; k < 2 * DJ; ++k) q[0][k] = *(const bf16x8*)at(k);
    locate(tile_lo);
  } else {
    locate(tile_lo);
#pragma unroll
    for (int k = 0; k < 2 * DJ; ++k) {
      const floatx4 x = *(const floatx4*)at(k), y = *(const floatx4*)(at(k) + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bf16_t part[PARTS];
        split<PARTS>(i < 4 ? x[i & 3] : y[i & 3], part);
#pragma unroll
        for (int n = 0; n < PARTS; ++n) q[n][k][i] = part[n];
      }
    }
  }
  // (waited for here, with the table: in the loop it would be waited for, with all that is on its way, in every step)
#pragma unroll
  for (int n = 0; n < PARTS; ++n)
#pragma unroll
    for (int k = 0; k < 2 * DJ; ++k) {
      const bf16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
      q[n][k] = in(k) ? q[n][k] : zero;
      asm volatile("" : "+v"(q[n][k]));
    }
  floatx16 o[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[i][x] = 0.f;
  float m = NEG_INF, l = 0.f;
  unsigned there_next = fetch(tile_lo, 0);
  float* const own_scales = own + wave * 32;
  const int k_at = (ph * 2 + odd) * BLOCK + h * 256 + c * 16, k_last = DK % 2 == 0 ? k_at : k_at - h * 256;
  const int v_at = Z::V_AT + ph * 2 * BLOCK;
  for (int tile = tile_lo; tile <= tile_hi; ++tile) {
    // this tile's loads are in (the wave's own; behind the barrier, all), and the tile before is read by all
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    const int slot = (tile - tile_lo) & 1;
    const unsigned char* const stage = lds + slot * Z::STAGE;
    const unsigned char* const scales = stage + Z::SCALES_AT + wave * 512 + odd * 256 + c;
    uint4v kc[DJ];
#pragma unroll
    for (int j = 0; j < DJ; ++j) kc[j] = *(const uint4v*)(stage + (j + 1 < DJ ? k_at : k_last) + j * 512);
    const float ks = power_of_byte(scales[0]);
    const float own_scale = power_of_byte(min((unsigned)scales[16], 254u));      // (finite: times a probability of zero it is zero)
    own_scales[col] = own_scale;      // (both halves the same)
    const unsigned there = there_next;
    there_next = fetch(tile + 1, slot ^ 1);
    const int kb0 = tile * KT + ph * 32;
    floatx16 s;
#pragma unroll
    for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const bf16x8 k0 = eight_numbers(kc[j][0], kc[j][1], ks), k1 = eight_numbers(kc[j][2], kc[j][3], ks);
#pragma unroll
      for (int n = PARTS - 1; n >= 0; --n) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0, q[n][2 * j], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1, q[n][2 * j + 1], s, 0, 0, 0);
      }
    }
    // the values' codes travel while the maximum is found: [block of 16][group of 64][quad h or 2 + h], two blocks of 16 of d each
    typedef unsigned uint2v __attribute__((ext_vector_type(2)));
    uint2v vc[2][GROUPS][2];
#pragma unroll
    for (int block = 0; block < 2; ++block)
#pragma unroll
      for (int group = 0; group < GROUPS; ++group)
#pragma unroll
        for (int two = 0; two < 2; ++two) {
          const int wide = group < FULL ? 4 : REST;
          const unsigned char* at = stage + v_at + block * BLOCK + group * 1024 + (two * 32 + h * 16 + c) * 4 * wide;
          if (wide == 4) {
            vc[block][group][two] = *(const uint2v*)(at + odd * 8);
          } else {
            vc[block][group][two][0] = *(const unsigned*)(at + (wide == 1 ? 0 : odd * (wide == 3 ? 8 : 4)));
            vc[block][group][two][1] = wide == 3 ? *(const unsigned*)(at + (odd ? 8 : 4)) : 0u;
          }
        }
    const bool masked = !(kb0 + 31 <= p_first && kb0 >= full_lo && there == 3);
    auto sees = [&](int i) {
      return (there >> (i >> 3) & 1) != 0 && (unsigned)(kb0 + 8 * (i >> 2) + (i & 3) + lane_key) <= span;
    };
    bool some = true;
    if (masked) {
      some = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = sees(i);
        some |= seen;
        s[i] = seen ? s[i] : NEG_INF;
      }
      // (codes that are not numbers: as in add_step)
      bool strange = false;
#pragma unroll
      for (int block = 0; block < 2; ++block)
#pragma unroll
        for (int group = 0; group < GROUPS; ++group)
#pragma unroll
          for (int n = 0; n < 4; ++n)
            strange |= (((vc[block][group][n >> 1][n & 1] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
      if (__any(strange)) {
#pragma unroll
        for (int block = 0; block < 2; ++block) {
          bf16x8 up, down;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            up[i] = sees(block * 8 + i) ? (bf16_t)LARGE : (bf16_t)0.f;
            down[i] = -up[i];
          }
#pragma unroll
          for (int group = 0; group < GROUPS; ++group)
#pragma unroll
            for (int i = 0; i < (group < FULL ? 2 : REST_DV); ++i) {
              bf16x8 bad;
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const bool nan = ((vc[block][group][x >> 2][i] >> (8 * (x & 3))) & 0x7fu) == 0x7fu;
                bad[x] = nan ? (bf16_t)LARGE : (bf16_t)0.f;
                if (nan) vc[block][group][x >> 2][i] &= ~(0xffu << (8 * (x & 3)));
              }
              o[group * 2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bad, up, o[group * 2 + i], 0, 0, 0);
              o[group * 2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bad, down, o[group * 2 + i], 0, 0, 0);
            }
        }
      }
    }
    m = fmaxf(m, some ? LOWEST : NEG_INF);      // (each half of the row's lanes for itself)
    float mx[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
    for (int x = 0; x < 16; x += 2) mx[(x >> 1) & 3] = fmaxf(fmaxf(s[x], s[x + 1]), mx[(x >> 1) & 3]);
    mx[0] = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), mx[2]), mx[3]);
    if (__any(mx[0] * a.scale2 > m + LAZY_MAX)) {      // some row's maximum grew: rescale what is summed so far
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx[0]), __float_as_uint(mx[0]), false, false);
      mx[0] = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * a.scale2;
      const bool grow = mx[0] > m + LAZY_MAX;
      const float m_new = grow ? mx[0] : m, alpha = grow ? fast_exp2(m - m_new) : 1.f;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DV; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] *= alpha;
      m = m_new;
    }
    const float neg_m = -fmaxf(m, LOWEST);      // (no score above it yet: every p is 2^-inf = 0)
#pragma unroll
    for (int block = 0; block < 2; ++block) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = fast_exp2(fmaf(s[block * 8 + i], a.scale2, neg_m));
      l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      const floatx4 w0 = *(const floatx4*)(own_scales + block * 16 + 4 * h), w1 = *(const floatx4*)(own_scales + block * 16 + 8 + 4 * h);
      bf16x8 pf[PARTS];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bf16_t part[PARTS];
        split<PARTS>(p[i] * (i < 4 ? w0[i & 3] : w1[i & 3]), part);
#pragma unroll
        for (int n = 0; n < PARTS; ++n) pf[n][i] = part[n];
      }
#pragma unroll
      for (int group = 0; group < GROUPS; ++group)
#pragma unroll
        for (int i = 0; i < (group < FULL ? 2 : REST_DV); ++i) {
          const bf16x8 vf = eight_numbers(vc[block][group][0][i], vc[block][group][1][i], 1.f);
#pragma unroll
          for (int n = PARTS - 1; n >= 0; --n)
            o[group * 2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[n], o[group * 2 + i], 0, 0, 0);
        }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);      // the last loads (of a tile past the end) are in, and the stages read
  __syncthreads();
  l += __shfl_xor(l, 32, WAVE);
  m = fmaxf(m, __shfl_xor(m, 32, WAVE));

  // (the row's place worked out again: two registers less in the loop)
  int again = row0 + col;
  asm volatile("" : "+v"(again));
  const bool has_row = again < total;
  const int out_tok = has_row ? again / G : 0, out_head = kvh * G + (has_row ? again - out_tok * G : 0);
  // piece n of a row, four numbers: registers 4 (n % 4) .. + 3 of sum n / 4
  // (numbers past the head's end, of a last group of one or three 16-wide blocks: negative)
  auto place = [&](int n) {
    const int group = n >> 3, block = ((n & 3) >> 1) * (group < FULL ? 2 : REST_DV) + ((n >> 2) & 1);
    return REST % 2 == 0 || group < FULL || block < REST ? group * 64 + block * 16 + (n & 1) * 8 + h * 4 : -1;
  };
  auto piece = [&](int n) { return floatx4{o[n >> 2][4 * (n & 3)], o[n >> 2][4 * (n & 3) + 1], o[n >> 2][4 * (n & 3) + 2], o[n >> 2][4 * (n & 3) + 3]}; };
  if constexpr (P == 1) {
    if (has_row)
#pragma unroll
      for (int n = 0; n < DV * 4; ++n)
        if (place(n) >= 0) write_output<T>(a, r0 + out_tok, out_head, place(n), piece(n), l, m);
  } else {
    // group ph puts the pieces ph, ph + P, .. of its rows together; the others' it finds in LDS
    constexpr int SHARES = DV * 4 / P;
    static_assert(SHARES * P == DV * 4, "whole shares");
    floatx4* const left = (floatx4*)lds;      // [wave][share][group but the wave's own][lane]
    float* const s_m = own + NW * 32;
    float* const s_l = s_m + NW * 32;
    if (h == 0) {
      s_m[wave * 32 + col] = m;
      s_l[wave * 32 + col] = l;
    }
    floatx4 mine[SHARES];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int n = 0; n < SHARES; ++n) {
        if (p == ph) mine[n] = piece(n * P + p);
        else left[((wave * SHARES + n) * (P - 1) + (p > ph ? p - 1 : p)) * 64 + lane] = piece(n * P + p);
      }
    __syncthreads();
    float w[P], top = NEG_INF, weight = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      w[p] = s_m[(p * RT + rt) * 32 + col];
      top = fmaxf(top, w[p]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      // (no maximum: no key that the row sees, and sums of zero)
      w[p] = w[p] == NEG_INF ? 1.f : fast_exp2(w[p] - top);
      weight += w[p] * s_l[(p * RT + rt) * 32 + col];
    }
#pragma unroll
    for (int n = 0; n < SHARES; ++n) {
      floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < P; ++p)
        v += w[p] * (p == ph ? mine[n] : left[(((p * RT + rt) * SHARES + n) * (P - 1) + (ph > p ? ph - 1 : ph)) * 64 + lane]);
      const int to = place(n * P + ph);
      if (has_row && to >= 0) write_output<T>(a, r0 + out_tok, out_head, to, v, weight, top);
    }
  }
}
#endif  // STAGED

// The splits of a row put together: a wave a (row, head), four numbers a lane and, where a head leaves lanes over, several splits at a
// time.  All of up to 8 splits a group of lanes are on their way while the factors are worked out (a lane a split) and the row's request is
// found: a row that the first launch left alone (of no request, of one whose starts do not fit the rows, or behind its tiles) stays as it is.
template <typename T>
__global__ __launch_bounds__(256) void attention_e4m3_merge_kernel(Args a) {
  constexpr int LANES = D / 4, GROUPS = 64 % LANES == 0 ? 64 / LANES : 1, AT_ONCE = 8;
  const int at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = at / a.nq, head = at - row * a.nq;
  if (row >= a.rows) return;
  const int group = lane / LANES < GROUPS ? lane / LANES : 0, i = GROUPS > 1 ? lane % LANES * 4 : lane * 4;
  const float* ml = a.ml_part + (size_t)at * a.splits * 2;
  const float* o = a.o_part + (size_t)at * a.splits * D + (i < D ? i : 0);
  floatx4 x[AT_ONCE];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) x[j] = *(const floatx4*)(o + (size_t)min(s0 + j * GROUPS + group, a.splits - 1) * D);
  };
  fetch(0);
  float m[2], w[2], f[2];      // (at most 128 splits)
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int s = lane + 64 * n;
    m[n] = s < a.splits ? ml[2 * s] : NEG_INF;
    w[n] = s < a.splits ? ml[2 * s + 1] : 0.f;
  }
  int r0 = -1, end = 0;      // of the last request that begins at or before the row
  for (int base = 0; base < a.reqs; base += 64) {
    const int i = min(base + lane, a.reqs - 1), start = a.q_start[i], next = a.q_start[i + 1];
    const unsigned long long begun = __ballot(base + lane < a.reqs && start <= row);
    if (begun) {
      const int last = 63 - __clzll(begun);
      r0 = __builtin_amdgcn_readlane(start, last);
      end = __builtin_amdgcn_readlane(next, last);
    }
  }
  const int G = a.nq / a.nkv;
  if (r0 < 0 || row >= end || end > a.rows || (long)(row - r0) * G + head % G >= a.covered) return;
  const float top = full_wave_max(fmaxf(m[0], m[1]));
#pragma unroll
  for (int n = 0; n < 2; ++n) f[n] = m[n] == NEG_INF ? 1.f : fast_exp2(m[n] - top);
  const float l = full_wave_sum(f[0] * w[0] + f[1] * w[1]);
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += AT_ONCE * GROUPS) {
    if (s0 > 0) fetch(s0);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int s = s0 + j * GROUPS + group;
      const float low = __shfl(f[0], s & 63, WAVE), high = __shfl(f[1], s & 63, WAVE);
      if (s < a.splits) sum += (s < 64 ? low : high) * x[j];
    }
  }
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor(sum[j], off, WAVE);
  }
  if (GROUPS > 1 ? lane < LANES : i < D) write_output<T>(a, row, head, i, sum, l, top);
}

extern "C" const char* llmlab_last_error() { return g_llmlab_error; }
extern "C" int llmlab_attention_head_dim() { return D; }

// For measurements and tests: the number of key splits (0: by the rule) and the form of the launch (0: by the rule, else one
// of those below where it exists; + 10: its blocks by tiles, + 20: by requests)
static int g_force_splits = 0, g_force_form = 0, g_force_order = -1;
extern "C" void llmlab_debug_attention_e4m3(int splits, int form) {
  g_force_splits = splits;
  g_force_form = form % 10;
  g_force_order = form / 10 - 1;
}

constexpr int SPLIT_WAVES = 4;
// Key splits: two blocks a unit where the tiles alone leave units without one; none shorter than 8 steps of 32 keys, and none of
// up to 32 steps, where the launch that puts the splits together costs what they gain (one to 16 requests of 28 heads of 128 over 4 at 700
// to 1,000 keys 7.9 to 10.3 us of GPU in one launch, 8.1 to 10.3 in two, and the host 2.8 us less; at 1,500 11.4 and 8.4).
static int key_splits(long blocks, int visible, int num_cus) {
  const long steps = (visible + 31L) / 32, most = (steps + 7) / 8;
  if (blocks >= num_cus || steps <= 32) return 1;
  return (int)std::max(1L, std::min(std::min(2L * num_cus / blocks, most), 128L));
}

// The form of a launch at heads up to 128, of bfloat16 rows: the one whose time is the least by an estimate, rounds of blocks (`more`
// for the last one's part and for what uneven tiles leave, `least` where units have few blocks) x (a block's start and end +
// its steps of 32 keys x a step), in us as fitted to 800 launches drawn at random (1 to 64 requests of 1 to 2,048 tokens
// behind 0 to 32,768 keys, of one length and of different ones, eight head layouts, a quarter through windows), over which
// the picks lose 0.3 % (heads of 64) and 0.5 % (128) to the best of all (850 others: 0.9 %, 32 % at worst, requests of very different lengths; 500 at heads of
// 16 to 112, by the figures of 64 or 128, 0.9 %).  Up to 16 rows (32 in bfloat16: one tile; the estimate takes another form there only for
// thousands of pairs behind some 20 keys) a tile's keys are split over waves and blocks; of more rows so, too, where they are few or the
// keys many.
// us, split / 2x4 / 2x2 / 4x1, heads of 128: 35 rows of 72 (request, kv head) pairs behind 6,652 keys 47 / 68 / 89 / 165; 152
// of 72 behind 2,380 44 / 34 / 39.5 / 66; 640 of 68 behind 229 31 / 33 / 20.6 / 24.7; 10,829 of 8 and 1,547 keys 91 / 89 / 58 / 58;
// 1,304 of 40 behind 63 32 / 38 / 26 / 21.5; 6,624 of 48 behind 232 241 / 269 / 161 / 148.
//
// float32 rows likewise, without 2x4 (which no launch of 80 drawn was fastest in): fitted to 700 launches, over 600 others the
// picks lose 0.7 % to the best (39 % at worst), and gain 11 % (heads of 64) and 14 % (128) on the split form, up to 2.6 times.  us, split / 2x2 / 4x1: 1,500 tokens of 32
// heads of 128 over 8 behind 3,000 keys 315 / 239 / 276; 7 requests of 700 tokens, 56 over 8, behind 700 439 / 290 / 273; 16 of 128, 32 over 8,
// behind 100 58 / 39 / 31; 61 tokens of 16 heads over 2 through a window of 1,000 24 / 36 / 56.
enum { FORM_SPLIT = 1, FORM_2x4, FORM_2x2, FORM_4x1 };
#if STAGED
struct Form {
  int form, rows, groups;
  float blocks_a_unit, start, step, more, least;
};
template <typename T>
static int launch_form(long most_rows, long pairs, int walk, int visible, int num_cus) {
  constexpr bool F32 = parts_of<T>() > 1;
  if (most_rows <= (F32 ? 16 : 32)) return FORM_SPLIT;
  constexpr Form bf16_forms[] = {
      {FORM_SPLIT, 32, SPLIT_WAVES, D <= 64 ? 3.f : 2.f, D <= 64 ? 5.5f : 6.4f, D <= 64 ? 1.14f : 1.18f, D <= 64 ? .54f : .58f, D <= 64 ? .79f : .92f},
      {FORM_2x4, 64, 4, D <= 64 ? 2.f : 1.f, D <= 64 ? 6.f : 8.2f, D <= 64 ? .85f : 1.18f, D <= 64 ? .9f : .34f, D <= 64 ? .83f : 1.f},
      {FORM_2x2, 64, 2, D <= 64 ? 4.f : 3.f, D <= 64 ? 6.2f : 10.5f, D <= 64 ? .75f : 1.06f, D <= 64 ? .82f : .51f, .71f},
      {FORM_4x1, 128, 1, D <= 64 ? 4.f : 3.f, D <= 64 ? 6.7f : 10.4f, D <= 64 ? .63f : .97f, D <= 64 ? .95f : .72f, D <= 64 ? .71f : .8f}};
  constexpr Form f32_forms[] = {
      {FORM_SPLIT, 16, SPLIT_WAVES, D <= 64 ? 3.f : 2.f, D <= 64 ? 4.2f : 4.9f, D <= 64 ? 1.28f : 1.35f, D <= 64 ? .61f : .52f, D <= 64 ? .83f : .91f},
      {FORM_2x2, 64, 2, D <= 64 ? 3.f : 2.f, D <= 64 ? 8.4f : 10.7f, D <= 64 ? 1.27f : 1.62f, D <= 64 ? .71f : .57f, D <= 64 ? .34f : .82f},
      {FORM_4x1, 128, 1, D <= 64 ? 3.f : 2.f, D <= 64 ? 8.1f : 9.8f, D <= 64 ? 1.23f : 1.62f, D <= 64 ? .8f : .77f, D <= 64 ? .78f : .74f}};
  constexpr float MERGE = F32 ? (D <= 64 ? 2.6f : .6f) : D <= 64 ? 2.2f : 1.3f;
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < (F32 ? 3 : 4); ++i) {
    const Form& f = F32 ? f32_forms[i < 3 ? i : 0] : bf16_forms[i];
    const long tiles = (most_rows + f.rows - 1) / f.rows * pairs;
    const int splits = f.form == FORM_SPLIT ? key_splits(tiles, visible, num_cus) : 1;
    const float steps = splits > 1 ? (float)visible / (32 * f.groups * splits) : (float)walk / (32 * f.groups);
    const float rounds = (float)tiles * splits / (f.blocks_a_unit * num_cus) + f.more;
    const float time = std::max(rounds, f.least) * (f.start + std::max(steps, 1.f) * f.step) + (splits > 1 ? MERGE : 0.f);
    if (i == 0 || time < least) {
      least = time;
      best = f.form;
    }
  }
  return best;
}
#endif

template <typename T, int QB, int P_PARTS>
static int launch_split(Args a, long most_rows, int visible, float* workspace, size_t workspace_floats, int num_cus,
                        hipStream_t stream) {
  const long tiles = (most_rows + 16 * QB - 1) / (16 * QB);
  a.covered = (int)std::min(tiles * 16 * QB, 0x7fffffffL);
  a.splits = g_force_splits > 0 ? g_force_splits : key_splits(tiles * a.nkv * a.reqs, visible, num_cus);
  const size_t each = (size_t)a.rows * a.nq * (D + 2);
  a.splits = (int)std::max((size_t)1, std::min((size_t)std::min(a.splits, 65535 / a.nkv), workspace_floats / std::max(each, (size_t)1)));
  if (a.splits > 1) {
    a.o_part = workspace;
    a.ml_part = workspace + (size_t)a.rows * a.nq * a.splits * D;
  }
  hipLaunchKernelGGL((attention_e4m3_split_kernel<T, QB, SPLIT_WAVES, P_PARTS>), dim3((unsigned)tiles, a.nkv * a.splits, a.reqs),
                     dim3(64 * SPLIT_WAVES), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("attention(e4m3)");
  if (a.splits > 1) {
    hipLaunchKernelGGL(attention_e4m3_merge_kernel<T>, dim3((unsigned)(((long)a.rows * a.nq + 3) / 4)), dim3(256), 0, stream, a);
    LLMLAB_LAUNCH_CHECK("attention(e4m3, merge)");
  }
  return 0;
}

#if STAGED
// The blocks' order where what is before the portions is half of them or more: by requests, the longest contexts first (us, by tiles / by
// requests, 28 heads of 128 over 4, contexts from 4 / 9 of the longest on: 3 x 1,000 up to 4,096 160 / 149, 5 x 700 up to 8,192 368 / 320, 2 x 2,000 up to
// 4,000 195 / 165, 3 x 1,200 up to 1,800 73.7 / 70.7; prompts from their start, 5 x 1,600 87 / 98).
template <typename T, int RT, int P>
static int launch_staged(const Args& a, long most_rows, bool history, hipStream_t stream) {
  const long tiles = (most_rows + 32 * RT - 1) / (32 * RT), blocks = tiles * a.nkv * a.reqs;
  const bool along_x = blocks * 64 * RT * P <= 0xffffffffL;
  const dim3 grid = along_x ? dim3((unsigned)blocks) : dim3((unsigned)tiles, a.nkv, a.reqs);
  const int by_requests = g_force_order >= 0 && a.reqs <= 64 ? g_force_order : along_x && history && a.reqs > 1 && a.reqs <= 64;
  hipLaunchKernelGGL((attention_e4m3_staged_kernel<T, RT, P>), grid, dim3(64 * RT * P), 0, stream, a, (int)tiles, by_requests);
  LLMLAB_LAUNCH_CHECK("attention(e4m3, staged)");
  return 0;
}
#endif

extern "C" int llmlab_paged_attention_e4m3(const void* q, int dtype, long q_stride, int nq, int nkv, const void* k, const void* v,
                                           const void* kv_scale, int pages, const int* table, int table_stride, int table_width,
                                           int page_size, const int* q_start, const int* start_pos, int reqs, int max_q_len,
                                           int max_ctx_len, int window, float scale, void* out, long out_stride, int rows,
                                           float* workspace, size_t workspace_floats, int num_cus, hipStream_t stream) {
  LLMLAB_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "attention(e4m3): %d heads, %d kv heads", nq, nkv);
  LLMLAB_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "attention(e4m3): page size %d is not a power of two >= 16",
                 page_size);
  LLMLAB_REQUIRE(q_stride >= (long)nq * D && out_stride >= (long)nq * D, "attention(e4m3): row strides too small");
  LLMLAB_REQUIRE(reqs >= 0 && reqs <= 65535, "attention(e4m3): %d requests, at most 65535 are taken", reqs);
  LLMLAB_REQUIRE(window >= 0, "attention(e4m3): negative window");
  LLMLAB_REQUIRE(pages >= 0 && table_width >= 0, "attention(e4m3): %d pages, a block table of %d", pages, table_width);
  LLMLAB_REQUIRE(scale > 0.f, "attention(e4m3): the score scale must be positive, got %g", (double)scale);
  LLMLAB_REQUIRE(((uintptr_t)q % 16) == 0 && ((uintptr_t)out % 16) == 0 && q_stride % (dtype == DT_F32 ? 4 : 8) == 0 && out_stride % 8 == 0,
                 "attention(e4m3): queries and outputs are not aligned for vector loads");
  LLMLAB_REQUIRE(((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0 && ((uintptr_t)kv_scale % 4) == 0,
                 "attention(e4m3): the pages are not aligned for vector loads");
  if (reqs == 0 || max_q_len <= 0 || rows == 0) return 0;
  Args a{q, (const unsigned char*)k, (const unsigned char*)v, (const unsigned char*)kv_scale, table, q_start, start_pos, out,
         q_stride, out_stride, table_stride, table_width, 0, pages,
         pages == 0 ? -1 : (int)std::min((long)table_width * page_size, 0x7fffffffL) - 1, nq, nkv, window, rows, reqs, 1, 0,
         scale * 1.4426950408889634f, nullptr, nullptr};
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  const long most_rows = (long)std::min(max_q_len, rows) * (nq / nkv);
  const int visible = window > 0 ? (int)std::min((long)max_ctx_len, (long)window + max_q_len) : max_ctx_len;
  if (num_cus <= 0) num_cus = 256;
  const bool f32 = dtype == DT_F32;
#if STAGED
  const int middle = max_ctx_len - max_q_len / 2, walk = window > 0 ? std::min(window, middle) : middle;
  const bool history = 2L * (max_ctx_len - max_q_len) >= max_q_len;
  // (a cache without pages: nothing there to be read in the place of a missing page.  With no last key the split form walks no step and
  // the rows are zeros; the staged forms read a stage in any case.)
  const int form = pages == 0         ? (int)FORM_SPLIT
                   : g_force_form > 0 ? g_force_form
                   : f32              ? launch_form<float>(most_rows, (long)nkv * reqs, walk, visible, num_cus)
                                      : launch_form<bf16_t>(most_rows, (long)nkv * reqs, walk, visible, num_cus);
  if (form == FORM_2x4 && !f32) return launch_staged<bf16_t, 2, 4>(a, most_rows, history, stream);
  if (form == FORM_2x2)
    return f32 ? launch_staged<float, 2, 2>(a, most_rows, history, stream) : launch_staged<bf16_t, 2, 2>(a, most_rows, history, stream);
  if (form == FORM_4x1)
    return f32 ? launch_staged<float, 4, 1>(a, most_rows, history, stream) : launch_staged<bf16_t, 4, 1>(a, most_rows, history, stream);
#endif
  const auto split = [&](auto launch) { return launch(a, most_rows, visible, workspace, workspace_floats, num_cus, stream); };
  if (f32) return split(launch_split<float, 1, 3>);
  // One token or a few, a tile for all their rows: probabilities of two parts, as the reading of the codes bounds them (us, one part /
  // two: 64 tokens of 28 heads of 128 over 4 at up to 4,096 keys 41.8 / 41.8, of 14 of 64 over 2 15.3 / 15.9, of 8 of 256 over 1 29.4 /
  // 30.5; 8 of 128 at 32,768 44.6 / 44.8; one of 64 at 700 9.9 / 9.8; 32 requests of 5 tokens of 40 heads over 8 at 2,500 30.1 / 31.6).
  // More rows: one part, as products bound them (staged forms: three portions of 1,000 tokens 145 / 192).
  if (most_rows <= 16) return split(launch_split<bf16_t, 1, 2>);
  if constexpr (D <= 128) {
    return most_rows <= 32 ? split(launch_split<bf16_t, 2, 2>) : split(launch_split<bf16_t, 2, 1>);
  } else {      // (32 rows do not fit the registers)
    return split(launch_split<bf16_t, 1, 1>);
  }
}
