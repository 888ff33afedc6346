// Verification of drafted tokens against the target model's distributions, with random numbers given by
// the caller.  gfx950 only.
//
// A request brings d drafted tokens x_0 .. x_(d-1) and d + 1 rows of float32 logits; p_j is the softmax of row j over its
// temperature, q_j the drafting model's distribution of x_j (the softmax of its logits over the same temperature; without
// logits all of it on x_j).  x_j stands while u_j q_j(x_j) < p_j(x_j); at the first that falls the next token is drawn
// from max(p_j - q_j, 0), behind the last from p_d: the first token at which the running sum of these weights reaches u_d
// times the whole.  The tokens so produced are distributed as the target model's own.  Temperature 0: x_j stands
// while it is the row's argmax (ties to the smallest index), and the next token is the argmax of the row that is reached.
//
// Exponentials and sums are taken in 64 bits (the vector unit runs float64 at the float32 rate): the running sum of 150,000
// weights has a border every 1e-5 or so, and float32 sums taken in another order would cross one in every few hundred
// draws.  What is summed is summed in one fixed order.
//
// Two launches: the rows in chunks (each leaves its maximum, its place and its sum of exponentials), then blocks for the
// chunks of every request's reached row, which find that row from the chunks' sums and weigh their chunks; the last of a request
// draws.  64 requests, 578 rows of 152,064 (351 MB): the first launch takes 65 us (5.4 TB/s; by a
// polynomial of degree 12 with conversions 89), bound by its exponentials and the reading alike, the second 27: a chain of
// small steps, 10 us for one request alone (first rows, sums, weights, the count of blocks, the chunk, the place in it).
#include "common.h"

constexpr int THREADS = 256, EACH = 16, CHUNK = THREADS * EACH;
constexpr double LOG2_E = 1.44269504088896340736;
constexpr int NONE = 0x7fffffff;      // the place of a maximum that is not there

struct VerifyArgs {
  const float* logits;       // [rows, vocab]
  const float* draft;        // [rows - n, vocab] or null
  const int* drafts;         // [rows - n]
  const int* row_start;      // [n + 1]
  const float* temperature;  // [n]
  const float* uniform;      // [rows]
  int* accepted;
  int* tokens;
  size_t stride, draft_stride;
  int n, rows, vocab, chunks;
  int each;                  // chunks that a block of the second launch weighs
  // scratch
  double* sum;               // [rows + drafted, chunks]: sum of exp((z - chunk's maximum) / t)
  double* mass;              // [n, chunks]: what the chunk weighs in the draw
  float* most;               // the chunks' maxima
  int* best;                 // and the first place of each
  int* arrived;              // [n]: chunks weighed so far (the first launch clears it)
};

// 2^y for y <= 0 (minus infinity, and what is not a number, too: exactly zero) to 1.1e-12 of itself: y = n + f, |f| <= 1/2, the
// n by adding 1.5 * 2^52 (its low word then is n), the polynomial of degree 8 that meets 2^f at the nine Chebyshev points of
// [-1/2, 1/2] (zero among them), and n added to the exponent's bits.  Below 2^-1023 it is zero: f is zero there, the polynomial 1 and
// its exponent's bits all gone.  (Every step at the rate of a product: a rint, a conversion and an ldexp are slower, and the
// exponentials bound the first launch.)  1.1e-12 is enough: one of 150,000 borders between tokens lies so near a given random number once in
// six million draws.  Degree 10 (3e-16, full 64 bits) takes 100 us where this takes 94 (64 requests, five drafts each with logits, 152,064
// tokens), 61 and 57 without.
__device__ __forceinline__ double exp2_below(double y) {
  constexpr double WHOLE = 6755399441055744.0;
  y = fmax(y, -1023.0);
  const double t = y + WHOLE, f = y - (t - WHOLE);
  double p = 1.32552248786688168e-06;
  p = fma(p, f, 1.53100794022492960e-05);
  p = fma(p, f, 1.54034558524538382e-04);
  p = fma(p, f, 1.33334505680006454e-03);
  p = fma(p, f, 9.61812915940255843e-03);
  p = fma(p, f, 5.55041094120593270e-02);
  p = fma(p, f, 2.40226506958129887e-01);
  p = fma(p, f, 6.93147180545933494e-01);
  p = fma(p, f, 1.0);
  return __hiloint2double((int)((unsigned)__double2hiint(p) + ((unsigned)__double2loint(t) << 20)), __double2loint(p));
}
// A logit's weight where `most` has weight 1; rate = log2 e over the temperature
__device__ __forceinline__ double weight(float z, float most, double rate) { return exp2_below(((double)z - (double)most) * rate); }

__device__ __forceinline__ bool bounded(float v) { return fabsf(v) < __builtin_huge_valf(); }

// Sums over the wave by lane swaps and DPP, no trip through LDS: every lane has the whole (wave_sum64), or what lies up to it
// (running_sum).  All 64 lanes are active.
__device__ __forceinline__ double of_halves(unsigned high, unsigned low) { return __hiloint2double((int)high, (int)low); }
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double moved(double v) {      // zero where nothing comes from
  return of_halves(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, ROWS == 0xf),
                   __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, ROWS == 0xf));
}
__device__ __forceinline__ double wave_sum64(double v) {
  {
    const auto h = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
    const auto l = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
    v = of_halves(h[0], l[0]) + of_halves(h[1], l[1]);
  }
  {
    const auto h = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
    v = of_halves(h[0], l[0]) + of_halves(h[1], l[1]);
  }
  v += moved<0x128>(v);      // row_ror:8
  v += moved<0x124>(v);      // row_ror:4
  v += moved<0x4E>(v);       // quad_perm 2, 3, 0, 1
  return v + moved<0xB1>(v); // quad_perm 1, 0, 3, 2
}
__device__ __forceinline__ double running_sum(double v) {
  v += moved<0x111>(v);      // row_shr:1
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<0x142, 0xa>(v); // row_bcast:15 into rows 1 and 3
  return v + moved<0x143, 0xc>(v);      // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ double lane_value64(double v, int lane) {      // (the same lane for the whole wave)
  return of_halves(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, WAVE));
  return v;
}

// The thread's numbers of a chunk: places quad * 1024 + 4 * thread + 0 .. 3, in rising order; minus infinity past the row's
// end.  (What is not a number stays so: no maximum takes it, and its weight is zero.)
__device__ __forceinline__ int place(int j) { return (j >> 2) * 4 * THREADS + 4 * (int)threadIdx.x + (j & 3); }
__device__ __forceinline__ void load_chunk(const float* z, int count, float (&v)[EACH]) {
  if (((uintptr_t)z & 15) == 0 && count == CHUNK) {
#pragma unroll
    for (int q = 0; q < EACH / 4; ++q) {
      const floatx4 x = *(const floatx4*)(z + place(4 * q));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = place(j) < count ? z[place(j)] : -__builtin_huge_valf();
  }
}

// The first launch: one chunk of one row (target rows, then the drafting model's).
__global__ __launch_bounds__(THREADS) void verify_chunks_kernel(VerifyArgs a) {
  __shared__ float s_most[THREADS / 64];
  __shared__ int s_best[THREADS / 64];
  __shared__ double s_sum[THREADS / 64];
  const int chunk = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (chunk == 0 && row < a.n && threadIdx.x == 0) a.arrived[row] = 0;      // (rows >= n)
  const bool target = row < a.rows;
  const float* z = target ? a.logits + (size_t)row * a.stride : a.draft + (size_t)(row - a.rows) * a.draft_stride;
  const int first = chunk * CHUNK;
  float v[EACH];
  load_chunk(z + first, min(CHUNK, a.vocab - first), v);
  // The request of the row: as many begin at or before it, without one (drafted token j of request b is number
  // row_start[b] - b + j, so its row of the drafting model's logits too).
  int before = 0;
  for (int base = 0; base < a.n; base += 64) {
    const int i = base + lane;
    before += __popcll(__ballot(i < a.n && (target ? a.row_start[i] <= row : a.row_start[i] - i <= row - a.rows)));
  }
  const float t = before > 0 ? a.temperature[before - 1] : 0.f;
  if (!target && !(t > 0.f)) return;
  float most = -__builtin_huge_valf();
#pragma unroll
  for (int j = 0; j < EACH; ++j) most = fmaxf(most, v[j]);
  const float top = full_wave_max(most);
  int at_best = NONE;
  double sum = 0.0;
  if (!(t > 0.f)) {      // (only the argmax is asked for)
    int best = EACH;
#pragma unroll
    for (int j = EACH - 1; j >= 0; --j) best = v[j] == top ? j : best;
    at_best = wave_min(best < EACH && top > -__builtin_huge_valf() ? first + place(best) : NONE);
  } else if (bounded(top)) {
    const double rate = LOG2_E / (double)t;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += weight(v[j], top, rate);
    sum = wave_sum64(sum);
  }
  if (lane == 0) {
    s_most[wave] = top;
    s_best[wave] = at_best;
    s_sum[wave] = sum;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  float all = s_most[0];
  for (int w = 1; w < THREADS / 64; ++w) all = fmaxf(all, s_most[w]);
  int place_of = NONE;
  double total = 0.0;
  for (int w = 0; w < THREADS / 64; ++w) {
    if (s_most[w] == all) place_of = min(place_of, s_best[w]);
    if (t > 0.f && bounded(all) && bounded(s_most[w])) total += s_sum[w] * weight(s_most[w], all, LOG2_E / (double)t);
  }
  const size_t at = (size_t)row * a.chunks + chunk;
  a.most[at] = all;
  a.best[at] = place_of;
  a.sum[at] = total;
}

struct RowSum {
  float most;
  int best;
  double sum;
};
// A row's chunks put together, by one wave; every lane gets the result
__device__ __forceinline__ RowSum whole_row(const VerifyArgs& a, int row, double rate) {
  const size_t at = (size_t)row * a.chunks;
  const int lane = threadIdx.x & 63;
  float most = -__builtin_huge_valf();
  int best = NONE;
  double sum = 0.0;
  for (int c = lane; c < a.chunks; c += 64) {
    const float m = a.most[at + c];
    const int i = a.best[at + c];
    const double s = a.sum[at + c];
    if (m > most) {      // (a lane's chunks: the running sum in units of the running maximum)
      sum = bounded(most) && bounded(m) ? sum * weight(most, m, rate) + s : s;
      most = m;
      best = i;
    } else if (bounded(m) && bounded(most)) {
      sum += s * weight(m, most, rate);
    }
  }
  RowSum r;
  r.most = full_wave_max(most);
  r.best = rate == 0.0 ? wave_min(most == r.most ? best : NONE) : NONE;      // (asked for where greedy)
  r.sum = wave_sum64(bounded(most) && bounded(r.most) ? sum * weight(most, r.most, rate) : 0.0);
  return r;
}

// What the next token is drawn from
struct Source {
  int row, draft_row;        // the row, the draft's that is subtracted (-1: none)
  int without;               // the token that has no weight (a draft without logits that fell), or -1
  float most, draft_most;
  double rate, inv_sum, draft_inv_sum;
};

__device__ __forceinline__ void chunk_weights(const VerifyArgs& a, const Source& d, int first, double (&w)[EACH]) {
  const int count = min(CHUNK, a.vocab - first);
  float z[EACH];
  load_chunk(a.logits + (size_t)d.row * a.stride + first, count, z);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    w[j] = weight(z[j], d.most, d.rate) * d.inv_sum;
    if (first + place(j) == d.without) w[j] = 0.0;
  }
  if (d.draft_row < 0) return;
  load_chunk(a.draft + (size_t)d.draft_row * a.draft_stride + first, count, z);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const double q = weight(z[j], d.draft_most, d.rate) * d.draft_inv_sum;
    w[j] = w[j] > q ? w[j] - q : 0.0;
  }
}

// Of the chunks' masses (lane c of a round of 64 has chunk base + c), by one wave: the first positive one in which the running
// sum reaches u times the whole (the last positive one where roundings keep the sum short of it), and what is left there.
template <typename F>
__device__ __forceinline__ int pick_chunk(int chunks, double u, F mass, double* left) {
  const int lane = threadIdx.x & 63;
  const double first = lane < chunks ? mass(lane) : 0.0;
  double total = wave_sum64(first);
  for (int base = 64; base < chunks; base += 64) total += wave_sum64(base + lane < chunks ? mass(base + lane) : 0.0);
  if (!(total > 0.0)) return -1;
  const double target = u * total;
  double run = 0.0;
  int chunk = -1;
  for (int base = 0; base < chunks; base += 64) {
    const double m = base == 0 ? first : base + lane < chunks ? mass(base + lane) : 0.0;
    const double sum = run + running_sum(m);
    const unsigned long long positive = __ballot(m > 0.0), reached = __ballot(m > 0.0 && sum >= target);
    const unsigned long long use = reached ? reached & -reached : 0;
    const int at = use ? __ffsll(use) - 1 : positive ? 63 - __clzll(positive) : -1;
    if (at >= 0) {
      chunk = base + at;
      *left = target - (lane_value64(sum, at) - lane_value64(m, at));
    }
    if (use) break;
    run = lane_value64(sum, 63);
  }
  return chunk;
}

// The second launch: a block for every (chunk, request).
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(VerifyArgs a) {
  constexpr int WAVES = THREADS / 64;
  constexpr int AT_ONCE = 16;      // drafted tokens looked at together
  __shared__ int s_last, s_chunk, s_plain;
  __shared__ double s_sum[WAVES], s_left;
  __shared__ RowSum s_row[2 * AT_ONCE + 1];
  const int chunk = blockIdx.x * a.each, b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r0 = a.row_start[b];
  int count = a.row_start[b + 1] - r0;
  const float t = a.temperature[b];
  // (a request without a row, or starts that do not fit the rows: no token)
  if (count < 1 || r0 < b || count > a.rows - r0 || count - 1 > a.rows - a.n - (r0 - b)) count = 0;
  const bool greedy = !(t > 0.f);
  if ((greedy || count == 0) && chunk > 0) return;
  if (count == 0) {
    if (threadIdx.x == 0) {
      a.accepted[b] = 0;
      a.tokens[b] = -1;
    }
    return;
  }
  const double rate = greedy ? 0.0 : LOG2_E / (double)t;

  // Which drafted tokens stand: the first that falls, or the last row.  A wave a row of logits; then every wave, a lane a token, all alike.
  const bool with_draft = a.draft != nullptr && !greedy;
  int first = count - 1;
  RowSum p = {}, q = {};
  for (int from = 0;; from += AT_ONCE) {
    const int n = min(AT_ONCE, count - 1 - from), rows = with_draft ? 2 * n : n;
    const bool at_end = from + n == count - 1;
    const int j = from + min(lane, max(n - 1, 0));
    // (asked for before the sums)
    int x = -1;
    float zx = 0.f, dx = 0.f, u = 0.f;
    if (lane < n) {
      x = a.drafts[r0 - b + j];
      u = a.uniform[r0 + j];
      if (x >= 0 && x < a.vocab) {
        zx = a.logits[(size_t)(r0 + j) * a.stride + x];
        if (with_draft) dx = a.draft[(size_t)(r0 - b + j) * a.draft_stride + x];
      }
    }
    for (int i = wave; i < rows + (at_end ? 1 : 0); i += WAVES) {
      const int of = i == rows ? n : i < n ? i : i - n;
      const RowSum r = whole_row(a, i < n || i == rows ? r0 + from + of : a.rows + r0 - b + from + of, rate);
      if (lane == 0) s_row[i == rows ? 2 * AT_ONCE : i < n ? i : AT_ONCE + of] = r;
    }
    __syncthreads();
    bool stands = lane >= n;
    if (lane < n && x >= 0 && x < a.vocab) {
      const RowSum of_p = s_row[lane];
      if (greedy) {
        stands = x == of_p.best;
      } else {
        double qx = 1.0;
        if (with_draft) {
          const RowSum of_q = s_row[AT_ONCE + lane];
          qx = bounded(of_q.most) ? weight(dx, of_q.most, rate) / of_q.sum : __builtin_nan("");
        }
        const double px = bounded(of_p.most) ? weight(zx, of_p.most, rate) / of_p.sum : 0.0;
        stands = (double)u * qx < px;      // (false where either is not a number)
      }
    }
    const unsigned long long falls = ~__ballot(stands);
    if (falls) {
      const int at = __ffsll(falls) - 1;
      first = from + at;
      p = s_row[at];
      if (with_draft) q = s_row[AT_ONCE + at];
      break;
    }
    if (at_end) {
      p = s_row[2 * AT_ONCE];
      break;
    }
    __syncthreads();
  }

  Source d{r0 + first, -1, -1, p.most, 0.f, rate, 1.0 / p.sum, 0.0};
  bool sound = greedy ? p.best != NONE : bounded(p.most);
  if (!greedy && first < count - 1) {
    if (a.draft) {
      d.draft_row = r0 - b + first;
      d.draft_most = q.most;
      d.draft_inv_sum = 1.0 / q.sum;
      sound = sound && bounded(q.most);
    } else {
      d.without = a.drafts[r0 - b + first];
    }
  }
  if (chunk == 0 && threadIdx.x == 0) {
    a.accepted[b] = first;
    if (greedy || !sound) a.tokens[b] = sound ? p.best : -1;
  }
  if (greedy || !sound) return;

  // its chunks' weights
  double w[EACH];
  double* mass = a.mass + (size_t)b * a.chunks;
  for (int c = chunk; c < min(chunk + a.each, a.chunks); ++c) {
    double mine = 0.0;
    chunk_weights(a, d, c * CHUNK, w);
#pragma unroll
    for (int j = 0; j < EACH; ++j) mine += w[j];
    mine = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) s_sum[wave] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double total = 0.0;
      for (int i = 0; i < WAVES; ++i) total += s_sum[i];
      // (device scope: past this die's L2, and done before the count)
      __hip_atomic_store(&mass[c], total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (threadIdx.x == 0) {
    __builtin_amdgcn_s_waitcnt(0);
    s_last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;

  // the last block of the request draws
  if (wave == 0) {
    const double u = (double)a.uniform[r0 + count - 1];
    double left = 0.0;
    int at = pick_chunk(a.chunks, u, [&](int c) { return __hip_atomic_load(&mass[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }, &left);
    int plain = 0;
    if (at < 0) {      // p and q are the same, and a drafted token that neither gives weight fell: from p
      plain = 1;
      const size_t of = (size_t)d.row * a.chunks;
      at = pick_chunk(a.chunks, u, [&](int c) {
        return bounded(a.most[of + c]) ? a.sum[of + c] * weight(a.most[of + c], d.most, rate) * d.inv_sum : 0.0;
      }, &left);
    }
    if (lane == 0) {
      s_chunk = at;
      s_left = left;
      s_plain = plain;
    }
  }
  __syncthreads();
  if (s_plain) d.draft_row = d.without = -1;
  const int from = s_chunk * CHUNK;
  if (s_chunk < 0) {
    if (threadIdx.x == 0) a.tokens[b] = -1;
    return;
  }
  // The place in the chunk.  Its places in rising order are quad after quad of 1,024, in each wave after wave, thread after thread: the
  // running sum over the threads' sums of four.
  chunk_weights(a, d, from, w);
  constexpr int QUADS = EACH / 4, PARTS = QUADS * WAVES;
  __shared__ double s_part[PARTS];
  __shared__ int s_has[PARTS], s_reached[PARTS];      // the last lane with weight, the first that reaches what is left (-1: none)
  const double left = s_left;
  double four[QUADS], sum[QUADS];
#pragma unroll
  for (int k = 0; k < QUADS; ++k) {
    four[k] = (w[4 * k] + w[4 * k + 1]) + (w[4 * k + 2] + w[4 * k + 3]);
    sum[k] = running_sum(four[k]);
    const unsigned long long positive = __ballot(four[k] > 0.0);
    if (lane == 63) s_part[k * WAVES + wave] = sum[k];
    if (lane == 0) s_has[k * WAVES + wave] = positive ? 63 - __clzll(positive) : -1;
  }
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    if (i % WAVES == wave) {
      const int k = i / WAVES;
      sum[k] += before;
      const unsigned long long reached = __ballot(four[k] > 0.0 && sum[k] >= left);
      if (lane == 0) s_reached[i] = reached ? __ffsll(reached) - 1 : -1;
    }
    before += s_part[i];
  }
  __syncthreads();
  int part = -1, owner = 0;
  bool whole = false;      // roundings kept the sum short of it: the last token that has weight
  for (int i = PARTS - 1; i >= 0; --i)
    if (s_reached[i] >= 0) {
      part = i;
      owner = s_reached[i];
    }
  if (part < 0) {
    whole = true;
    for (int i = 0; i < PARTS; ++i)
      if (s_has[i] >= 0) {
        part = i;
        owner = s_has[i];
      }
  }
  if (part < 0 || part % WAVES != wave || lane != owner) return;
  int token = -1;
#pragma unroll
  for (int k = 0; k < QUADS; ++k) {
    if (k != part / WAVES) continue;
    double run = sum[k] - four[k];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!whole && token >= 0 && run >= left) break;
      if (w[4 * k + j] > 0.0) token = from + place(4 * k + j);
      run += w[4 * k + j];
    }
  }
  a.tokens[b] = token;
}

extern "C" const char* llmlab_last_error() { return g_llmlab_error; }

// Bytes of scratch of a call (8-byte aligned)
extern "C" size_t llmlab_verify_drafts_scratch(int n, int rows, int vocab, int with_draft) {
  const size_t chunks = ((size_t)vocab + CHUNK - 1) / CHUNK, all = (size_t)rows + (with_draft ? rows - n : 0);
  return all * chunks * 16 + (size_t)n * chunks * 8 + (size_t)n * 4;
}

extern "C" int llmlab_verify_drafts(const float* logits, size_t stride, const float* draft, size_t draft_stride,
                                    const int* drafts, const int* row_start, const float* temperature, const float* uniform,
                                    int n, int rows, int vocab, int* accepted, int* tokens, void* scratch,
                                    size_t scratch_bytes, int num_cus, hipStream_t stream) {
  LLMLAB_REQUIRE(n >= 0 && rows >= n && vocab > 0, "verify_drafts: bad sizes requests=%d rows=%d vocabulary=%d", n, rows, vocab);
  LLMLAB_REQUIRE(stride >= (size_t)vocab && (draft == nullptr || draft_stride >= (size_t)vocab), "verify_drafts: row strides too small");
  if (n == 0) return 0;
  const size_t all = (size_t)rows + (draft ? rows - n : 0);
  LLMLAB_REQUIRE(all <= 65535 && n <= 65535, "verify_drafts: %zu rows of logits, at most 65535 are taken", all);
  LLMLAB_REQUIRE(scratch_bytes >= llmlab_verify_drafts_scratch(n, rows, vocab, draft != nullptr) && ((uintptr_t)scratch % 8) == 0,
                 "verify_drafts: the scratch buffer is too small");
  VerifyArgs a{logits, draft, drafts, row_start, temperature, uniform, accepted, tokens, stride, draft_stride, n, rows, vocab,
               (vocab + CHUNK - 1) / CHUNK, 1, nullptr, nullptr, nullptr, nullptr, nullptr};
  char* p = (char*)scratch;
  const size_t parts = all * a.chunks;
  a.sum = (double*)p;
  a.mass = a.sum + parts;
  a.most = (float*)(a.mass + (size_t)n * a.chunks);
  a.best = (int*)(a.most + parts);
  a.arrived = a.best + parts;
  hipLaunchKernelGGL(verify_chunks_kernel, dim3(a.chunks, (unsigned)all), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(chunks)");
  // Two chunks a block once there are more blocks than the chip holds at a time, five a unit: the decision is made half as often
  // (us, one / two, with the draft's logits and without: 32 requests of 152,064 55 / 55 and 38 / 37, 48 77 / 77 and 53 / 48, 64 97 / 93 and 63 / 57).
  a.each = (long)a.chunks * n > 5L * (num_cus > 0 ? num_cus : 256) ? 2 : 1;
  hipLaunchKernelGGL(verify_draw_kernel, dim3((a.chunks + a.each - 1) / a.each, n), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(draw)");
  return 0;
}
