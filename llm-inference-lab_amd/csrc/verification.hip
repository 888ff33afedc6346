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
// Exponentials and sums are taken in 64 bits (the vector unit runs float64 at the float32 rate and the rows' reading bounds
// the pass): the running sum of 150,000 weights has a border every 1e-5 or so, and float32 sums taken in another order
// would cross one in every few hundred draws.  What is summed is summed in one fixed order.
//
// Two launches: the rows in chunks (each leaves its maximum, its place and its sum of exponentials), then a block for every
// chunk of every request's reached row, which finds that row from the chunks' sums, weighs its chunk, and is the one that
// draws if it is the last of its request.
#include "common.h"

constexpr int THREADS = 256, EACH = 16, CHUNK = THREADS * EACH;
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
  // scratch
  double* sum;               // [rows + drafted, chunks]: sum of exp((z - chunk's maximum) / t)
  double* mass;              // [n, chunks]: what the chunk weighs in the draw
  float* most;               // the chunks' maxima
  int* best;                 // and the first place of each
  int* arrived;              // [n]: chunks weighed so far (the first launch clears it)
};

// e^x for x <= 0 (minus infinity too) to about a rounding: x = n ln 2 + r, |r| <= ln 2 / 2, Taylor's sum of e^r to the
// twelfth power (what is left out: r^13 / 13! < 2e-16), times 2^n.
__device__ __forceinline__ double exp_below(double x) {
  x = fmax(x, -800.0);
  const double n = rint(x * 1.4426950408889634074);
  double r = fma(n, -0.69314718055994528623, x);
  r = fma(n, -2.3190468138462995584e-17, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

__device__ __forceinline__ bool bounded(float v) { return fabsf(v) < __builtin_huge_valf(); }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, WAVE));
  return v;
}

// The thread's numbers of a chunk: places quad * 1024 + 4 * thread + 0 .. 3, in rising order; nothing past the row's end,
// and what is not a number, is minus infinity.
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
#pragma unroll
  for (int j = 0; j < EACH; ++j) v[j] = v[j] == v[j] ? v[j] : -__builtin_huge_valf();
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
  float most = v[0];
  int best = 0;
#pragma unroll
  for (int j = 1; j < EACH; ++j)
    if (v[j] > most) {
      most = v[j];
      best = j;
    }
  const float top = full_wave_max(most);
  const int at_best = wave_min(most == top && top > -__builtin_huge_valf() ? first + place(best) : NONE);
  double sum = 0.0;
  if (t > 0.f && bounded(top)) {
    const double inv_t = 1.0 / (double)t;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += exp_below(((double)v[j] - (double)top) * inv_t);
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
    if (t > 0.f && bounded(all) && bounded(s_most[w])) total += s_sum[w] * exp_below(((double)s_most[w] - (double)all) / (double)t);
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
__device__ __forceinline__ RowSum whole_row(const VerifyArgs& a, int row, double inv_t) {
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
      sum = bounded(most) && bounded(m) ? sum * exp_below(((double)most - (double)m) * inv_t) + s : s;
      most = m;
      best = i;
    } else if (bounded(m) && bounded(most)) {
      sum += s * exp_below(((double)m - (double)most) * inv_t);
    }
  }
  RowSum r;
  r.most = full_wave_max(most);
  r.best = wave_min(most == r.most ? best : NONE);
  r.sum = wave_sum64(bounded(most) && bounded(r.most) ? sum * exp_below(((double)most - (double)r.most) * inv_t) : 0.0);
  return r;
}

// What the next token is drawn from
struct Source {
  int row, draft_row;        // the row, the draft's that is subtracted (-1: none)
  int without;               // the token that has no weight (a draft without logits that fell), or -1
  float most, draft_most;
  double inv_t, inv_sum, draft_inv_sum;
};

__device__ __forceinline__ void chunk_weights(const VerifyArgs& a, const Source& d, int first, double (&w)[EACH]) {
  const int count = min(CHUNK, a.vocab - first);
  float z[EACH];
  load_chunk(a.logits + (size_t)d.row * a.stride + first, count, z);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    w[j] = exp_below(((double)z[j] - (double)d.most) * d.inv_t) * d.inv_sum;
    if (first + place(j) == d.without) w[j] = 0.0;
  }
  if (d.draft_row < 0) return;
  load_chunk(a.draft + (size_t)d.draft_row * a.draft_stride + first, count, z);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const double q = exp_below(((double)z[j] - (double)d.draft_most) * d.inv_t) * d.draft_inv_sum;
    w[j] = w[j] > q ? w[j] - q : 0.0;
  }
}

// The running sum over the wave's lanes, one number a lane
__device__ __forceinline__ double running_sum(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double x = __shfl_up(v, off, WAVE);
    if (lane >= off) v += x;
  }
  return v;
}

// Of the chunks' masses (lane c of a round of 64 has chunk base + c), by one wave: the first positive one in which the running
// sum reaches u times the whole (the last positive one where roundings keep the sum short of it), and what is left there.
template <typename F>
__device__ __forceinline__ int pick_chunk(int chunks, double u, F mass, double* left) {
  const int lane = threadIdx.x & 63;
  double total = 0.0;
  for (int base = 0; base < chunks; base += 64) total += __shfl(running_sum(base + lane < chunks ? mass(base + lane) : 0.0), 63, WAVE);
  if (!(total > 0.0)) return -1;
  const double target = u * total;
  double run = 0.0;
  int chunk = -1;
  for (int base = 0; base < chunks; base += 64) {
    const double m = base + lane < chunks ? mass(base + lane) : 0.0;
    const double sum = run + running_sum(m);
    const unsigned long long positive = __ballot(m > 0.0), reached = __ballot(m > 0.0 && sum >= target);
    const unsigned long long use = reached ? reached & -reached : 0;
    const int at = use ? __ffsll(use) - 1 : positive ? 63 - __clzll(positive) : -1;
    if (at >= 0) {
      chunk = base + at;
      *left = target - (__shfl(sum, at, WAVE) - __shfl(m, at, WAVE));
    }
    if (use) break;
    run = __shfl(sum, 63, WAVE);
  }
  return chunk;
}

// The second launch: a block for every (chunk, request).
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(VerifyArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int s_first, s_last, s_chunk, s_wave_last[WAVES];
  __shared__ double s_sum[WAVES], s_left;
  const int chunk = blockIdx.x, b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r0 = a.row_start[b];
  int count = a.row_start[b + 1] - r0;
  // (a request without a row, or starts that do not fit the rows: no token)
  if (count < 1 || r0 < b || count > a.rows - r0 || count - 1 > a.rows - a.n - (r0 - b)) count = 0;
  const float t = a.temperature[b];
  const bool greedy = !(t > 0.f);
  if ((greedy || count == 0) && chunk > 0) return;
  const double inv_t = greedy ? 0.0 : 1.0 / (double)t;

  // which drafted tokens stand: the first that falls (or the last row)
  if (threadIdx.x == 0) s_first = max(count - 1, 0);
  __syncthreads();
  for (int j = wave; j < count - 1; j += WAVES) {
    const int x = a.drafts[r0 - b + j];
    const RowSum p = whole_row(a, r0 + j, inv_t);
    bool stands = x >= 0 && x < a.vocab;
    if (greedy) {
      stands = x == p.best;
    } else if (stands) {
      const double px = exp(((double)a.logits[(size_t)(r0 + j) * a.stride + x] - (double)p.most) * inv_t) / p.sum;
      double qx = 1.0;
      if (a.draft) {
        const RowSum q = whole_row(a, a.rows + r0 - b + j, inv_t);
        qx = exp(((double)a.draft[(size_t)(r0 - b + j) * a.draft_stride + x] - (double)q.most) * inv_t) / q.sum;
      }
      stands = (double)a.uniform[r0 + j] * qx < px;      // (false where either is not a number)
    }
    if (!stands && lane == 0) atomicMin(&s_first, j);
  }
  __syncthreads();
  const int first = s_first;
  if (count == 0) {
    if (threadIdx.x == 0) {
      a.accepted[b] = 0;
      a.tokens[b] = -1;
    }
    return;
  }

  // the row that is reached (every wave the same)
  const RowSum p = whole_row(a, r0 + first, inv_t);
  Source d{r0 + first, -1, -1, p.most, 0.f, inv_t, 1.0 / p.sum, 0.0};
  bool sound = greedy ? p.best != NONE : bounded(p.most);
  if (!greedy && first < count - 1) {
    if (a.draft) {
      const RowSum q = whole_row(a, a.rows + r0 - b + first, inv_t);
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

  // this chunk's weight
  double w[EACH], mine = 0.0;
  chunk_weights(a, d, chunk * CHUNK, w);
#pragma unroll
  for (int j = 0; j < EACH; ++j) mine += w[j];
  mine = wave_sum64(mine);
  if (lane == 0) s_sum[wave] = mine;
  __syncthreads();
  double* mass = a.mass + (size_t)b * a.chunks;
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < WAVES; ++i) total += s_sum[i];
    // (device scope: past this die's L2, and done before the count)
    __hip_atomic_store(&mass[chunk], total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    s_last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
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
        return bounded(a.most[of + c]) ? a.sum[of + c] * exp_below(((double)a.most[of + c] - (double)d.most) * inv_t) * d.inv_sum : 0.0;
      }, &left);
    }
    if (lane == 0) {
      s_chunk = at;
      s_left = left;
      s_first = plain;
    }
  }
  __syncthreads();
  if (s_first) d.draft_row = d.without = -1;
  const int from = s_chunk * CHUNK;
  if (s_chunk < 0) {
    if (threadIdx.x == 0) a.tokens[b] = -1;
    return;
  }
  // The place in the chunk.  Its places in rising order are quad after quad of 1,024, in each thread after thread: the running sum over
  // the threads' sums of four, quad by quad.
  chunk_weights(a, d, from, w);
  double run = 0.0;
  const double left = s_left;
  int last_positive = -1;
  for (int q = 0; q < EACH / 4; ++q) {
    const double four = (w[4 * q] + w[4 * q + 1]) + (w[4 * q + 2] + w[4 * q + 3]);
    const double sum = running_sum(four);
    const unsigned long long positive = __ballot(four > 0.0);
    __syncthreads();
    if (lane == 63) s_sum[wave] = sum;
    if (lane == 0) s_wave_last[wave] = positive ? 63 - __clzll(positive) : -1;
    __syncthreads();
    double before = run;
    for (int i = 0; i < wave; ++i) before += s_sum[i];
    for (int i = 0; i < WAVES; ++i) {
      run += s_sum[i];
      if (s_wave_last[i] >= 0) last_positive = q * THREADS + i * 64 + s_wave_last[i];
    }
    // the first thread whose sum reaches what is left
    const unsigned long long reached = __ballot(four > 0.0 && before + sum >= left);
    if (lane == 0) s_wave_last[wave] = reached ? __ffsll(reached) - 1 : -1;
    __syncthreads();
    int owner = -1;
    for (int i = WAVES - 1; i >= 0; --i)
      if (s_wave_last[i] >= 0) owner = i * 64 + s_wave_last[i];
    if (owner < 0) continue;
    if ((int)threadIdx.x == owner) {
      double r = before + (sum - four);
      int token = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (token >= 0 && r >= left) break;
        if (w[4 * q + j] > 0.0) token = from + place(4 * q + j);
        r += w[4 * q + j];
      }
      a.tokens[b] = token;
    }
    return;
  }
  // (roundings kept the sum short of it: the last token that has weight)
  if (last_positive >= 0 && (int)threadIdx.x == last_positive % THREADS) {
    const int q = last_positive / THREADS;
    int token = -1;
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if ((j >> 2) == q && w[j] > 0.0) token = from + place(j);
    a.tokens[b] = token;
  }
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
                                    size_t scratch_bytes, hipStream_t stream) {
  LLMLAB_REQUIRE(n >= 0 && rows >= n && vocab > 0, "verify_drafts: bad sizes requests=%d rows=%d vocabulary=%d", n, rows, vocab);
  LLMLAB_REQUIRE(stride >= (size_t)vocab && (draft == nullptr || draft_stride >= (size_t)vocab), "verify_drafts: row strides too small");
  if (n == 0) return 0;
  const size_t all = (size_t)rows + (draft ? rows - n : 0);
  LLMLAB_REQUIRE(all <= 65535 && n <= 65535, "verify_drafts: %zu rows of logits, at most 65535 are taken", all);
  LLMLAB_REQUIRE(scratch_bytes >= llmlab_verify_drafts_scratch(n, rows, vocab, draft != nullptr) && ((uintptr_t)scratch % 8) == 0,
                 "verify_drafts: the scratch buffer is too small");
  VerifyArgs a{logits, draft, drafts, row_start, temperature, uniform, accepted, tokens, stride, draft_stride, n, rows, vocab,
               (vocab + CHUNK - 1) / CHUNK, nullptr, nullptr, nullptr, nullptr, nullptr};
  char* p = (char*)scratch;
  const size_t parts = all * a.chunks;
  a.sum = (double*)p;
  a.mass = a.sum + parts;
  a.most = (float*)(a.mass + (size_t)n * a.chunks);
  a.best = (int*)(a.most + parts);
  a.arrived = a.best + parts;
  hipLaunchKernelGGL(verify_chunks_kernel, dim3(a.chunks, (unsigned)all), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(chunks)");
  hipLaunchKernelGGL(verify_draw_kernel, dim3(a.chunks, n), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(draw)");
  return 0;
}
