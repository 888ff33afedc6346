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
#include "common.h"

constexpr int CHUNK = 4096, THREADS = 256, EACH = CHUNK / THREADS;
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
  float* most;               // the chunks' maxima
  int* best;                 // and the first place of each
  double* mass;              // [n, chunks]: what the chunk weighs in the draw
  struct Decision* decision; // [n]
};

struct Decision {
  int row, draft_row;        // the row that is drawn from, the draft's that is subtracted (-1: none)
  int without;               // the token that has no weight (a draft without logits that fell), or -1
  int last;                  // the request's last row, whose random number the draw takes
  int done;                  // nothing is drawn
  double inv_t, most, inv_sum, draft_most, draft_inv_sum;
};

// The request of a row: how many begin at or before it (empty ones come before the one that holds it)
__device__ __forceinline__ int request_of_row(const VerifyArgs& a, int row) {
  int before = 0;
  for (int base = 0; base < a.n; base += 64) {
    const int i = base + (threadIdx.x & 63);
    before += __popcll(__ballot(i < a.n && a.row_start[i] <= row));
  }
  return before - 1;
}

template <typename F>
__device__ __forceinline__ double block_reduce(double v, double* red, F op) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, WAVE));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = op(v, red[w]);
  return v;
}

// One chunk of one row (target rows, then the drafting model's): its maximum, the first place of it, and the sum of its
// exponentials.  What is not a number counts as minus infinity.
__global__ __launch_bounds__(THREADS) void verify_chunks_kernel(VerifyArgs a) {
  __shared__ double red[THREADS / 64];
  __shared__ int s_best[THREADS / 64];
  const int chunk = blockIdx.x, row = blockIdx.y;
  const bool target = row < a.rows;
  // drafted token j of request b is number row_start[b] - b + j
  int b;
  if (target) {
    b = request_of_row(a, row);
  } else {
    int before = 0;
    for (int base = 0; base < a.n; base += 64) {
      const int i = base + (threadIdx.x & 63);
      before += __popcll(__ballot(i < a.n && a.row_start[i] - i <= row - a.rows));
    }
    b = before - 1;
  }
  if (b < 0) return;
  const float t = a.temperature[b];
  if (!target && !(t > 0.f)) return;
  const float* z = target ? a.logits + (size_t)row * a.stride : a.draft + (size_t)(row - a.rows) * a.draft_stride;
  const int first = chunk * CHUNK, count = min(CHUNK, a.vocab - first);
  float v[EACH];
  float most = -__builtin_huge_valf();
  int best = NONE;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = threadIdx.x + j * THREADS;
    const float x = i < count ? z[first + i] : -__builtin_huge_valf();
    v[j] = x == x ? x : -__builtin_huge_valf();
    if (v[j] > most) {
      most = v[j];
      best = first + i;
    }
  }
  const float top = (float)block_reduce((double)most, red, [](double x, double y) { return x > y ? x : y; });
  if (most != top) best = NONE;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) best = min(best, __shfl_xor(best, off, WAVE));
  if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
  double sum = 0.0;
  if (t > 0.f && top > -__builtin_huge_valf() && top < __builtin_huge_valf()) {
    const double inv_t = 1.0 / (double)t;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += exp(((double)v[j] - (double)top) * inv_t);
  }
  sum = block_reduce(sum, red, [](double x, double y) { return x + y; });
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 64; ++w) best = min(best, s_best[w]);
    const size_t at = (size_t)row * a.chunks + chunk;
    a.most[at] = top;
    a.best[at] = best;
    a.sum[at] = sum;
  }
}

struct RowSum {
  double most, sum;
  int best;
};
// A row's chunks put together, by one wave; every lane gets the result
__device__ __forceinline__ RowSum whole_row(const VerifyArgs& a, int row, double inv_t) {
  const size_t at = (size_t)row * a.chunks;
  const int lane = threadIdx.x & 63;
  float most = -__builtin_huge_valf();
  int best = NONE;
  for (int c = lane; c < a.chunks; c += 64)
    if (a.most[at + c] > most) {
      most = a.most[at + c];
      best = a.best[at + c];
    }
  const float top = wave_max(most);
  if (most != top) best = NONE;
  double sum = 0.0;
  if (top < __builtin_huge_valf() && top > -__builtin_huge_valf() && inv_t > 0.0)
    for (int c = lane; c < a.chunks; c += 64) sum += a.sum[at + c] * exp(((double)a.most[at + c] - (double)top) * inv_t);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    best = min(best, __shfl_xor(best, off, WAVE));
    sum += __shfl_xor(sum, off, WAVE);
  }
  return RowSum{(double)top, sum, best};
}

// One block a request: which drafted tokens stand, and what the next token is drawn from.
__global__ __launch_bounds__(256) void verify_decide_kernel(VerifyArgs a) {
  __shared__ int s_first;
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r0 = a.row_start[b];
  int count = a.row_start[b + 1] - r0;
  // (a request without a row, or starts that do not fit the rows: no token)
  if (count < 1 || r0 < b || count > a.rows - r0 || count - 1 > a.rows - a.n - (r0 - b)) count = 0;
  const float t = a.temperature[b];
  const bool greedy = !(t > 0.f);
  const double inv_t = greedy ? 0.0 : 1.0 / (double)t;
  if (threadIdx.x == 0) s_first = max(count - 1, 0);
  __syncthreads();
  for (int j = wave; j < count - 1; j += 4) {
    const int x = a.drafts[r0 - b + j];
    const RowSum p = whole_row(a, r0 + j, inv_t);
    bool stands = x >= 0 && x < a.vocab;
    if (greedy) {
      stands = x == p.best;
    } else if (stands) {
      const double px = exp(((double)a.logits[(size_t)(r0 + j) * a.stride + x] - p.most) * inv_t) / p.sum;
      double qx = 1.0;
      if (a.draft) {
        const RowSum q = whole_row(a, a.rows + r0 - b + j, inv_t);
        qx = exp(((double)a.draft[(size_t)(r0 - b + j) * a.draft_stride + x] - q.most) * inv_t) / q.sum;
      }
      stands = (double)a.uniform[r0 + j] * qx < px;      // (false where either is not a number)
    }
    if (!stands && lane == 0) atomicMin(&s_first, j);
  }
  __syncthreads();
  if (wave != 0) return;
  const int first = s_first;
  Decision d{r0 + first, -1, -1, r0 + count - 1, 1, inv_t, 0.0, 0.0, 0.0, 0.0};
  int token = -1;
  if (count > 0) {
    const RowSum p = whole_row(a, d.row, inv_t);
    const bool sound = p.most < __builtin_huge_val() && p.most > -__builtin_huge_val();      // (else no distribution)
    if (greedy && p.best != NONE) token = p.best;
    if (!greedy && sound) {
      d.done = 0;
      d.most = p.most;
      d.inv_sum = 1.0 / p.sum;
      if (first < count - 1) {
        if (a.draft) {
          const RowSum q = whole_row(a, a.rows + r0 - b + first, inv_t);
          d.draft_row = r0 - b + first;
          d.draft_most = q.most;
          d.draft_inv_sum = 1.0 / q.sum;
          if (!(q.most < __builtin_huge_val() && q.most > -__builtin_huge_val())) d.done = 1;
        } else {
          d.without = a.drafts[r0 - b + first];
        }
      }
    }
  }
  if (lane == 0) {
    a.accepted[b] = first;
    a.decision[b] = d;
    if (d.done) a.tokens[b] = token;
  }
}

__device__ __forceinline__ double weight(const VerifyArgs& a, const Decision& d, int i) {
  const float z = a.logits[(size_t)d.row * a.stride + i];
  double w = z == z ? exp(((double)z - d.most) * d.inv_t) * d.inv_sum : 0.0;
  if (i == d.without) w = 0.0;
  if (d.draft_row >= 0) {
    const float y = a.draft[(size_t)d.draft_row * a.draft_stride + i];
    const double q = y == y ? exp(((double)y - d.draft_most) * d.inv_t) * d.draft_inv_sum : 0.0;
    w = w > q ? w - q : 0.0;
  }
  return w;
}

// What every chunk of the row weighs in the draw
__global__ __launch_bounds__(THREADS) void verify_mass_kernel(VerifyArgs a) {
  __shared__ double red[THREADS / 64];
  const int chunk = blockIdx.x, b = blockIdx.y;
  const Decision d = a.decision[b];
  if (d.done) return;
  const int first = chunk * CHUNK, count = min(CHUNK, a.vocab - first);
  double mass = 0.0;
  for (int i = threadIdx.x; i < count; i += THREADS) mass += weight(a, d, first + i);
  mass = block_reduce(mass, red, [](double x, double y) { return x + y; });
  if (threadIdx.x == 0) a.mass[(size_t)b * a.chunks + chunk] = mass;
}

// The chunk in which the running sum reaches u times the whole, then the place in it
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double s_sum[THREADS];
  __shared__ double s_left;
  __shared__ int s_chunk, s_owner, s_plain;
  const int b = blockIdx.x;
  Decision d = a.decision[b];
  if (d.done) return;
  if (threadIdx.x == 0) {
    double* mass = a.mass + (size_t)b * a.chunks;
    double total = 0.0, run = 0.0;
    for (int c = 0; c < a.chunks; ++c) total += mass[c];
    if (!(total > 0.0)) {      // p and q are the same: a drafted token that neither gives weight fell.  From p.
      d.draft_row = d.without = -1;
      const size_t at = (size_t)d.row * a.chunks;
      for (int c = 0; c < a.chunks; ++c)
        total += mass[c] = a.sum[at + c] * exp(((double)a.most[at + c] - d.most) * d.inv_t) * d.inv_sum;
    }
    s_plain = d.draft_row < 0 && d.without < 0;
    int chunk = -1;
    if (total > 0.0) {
      const double target = (double)a.uniform[d.last] * total;
      for (int c = 0; c < a.chunks; ++c) {
        if (!(mass[c] > 0.0)) continue;
        chunk = c;
        s_left = target - run;
        if (run + mass[c] >= target) break;
        run += mass[c];
      }
    }
    s_chunk = chunk;
  }
  __syncthreads();
  const int chunk = s_chunk;
  if (s_plain) d.draft_row = d.without = -1;
  if (chunk < 0) {
    if (threadIdx.x == 0) a.tokens[b] = -1;
    return;
  }
  const int first = chunk * CHUNK, count = min(CHUNK, a.vocab - first);
  const int begin = min(count, (int)threadIdx.x * EACH), end = min(count, begin + EACH);
  double mine = 0.0;
  for (int i = begin; i < end; ++i) mine += weight(a, d, first + i);
  s_sum[threadIdx.x] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double run = 0.0, left = s_left;
    int owner = -1;
    for (int i = 0; i < THREADS; ++i) {
      if (!(s_sum[i] > 0.0)) continue;
      owner = i;
      s_left = left - run;
      if (run + s_sum[i] >= left) break;
      run += s_sum[i];
    }
    s_owner = owner;
  }
  __syncthreads();
  if ((int)threadIdx.x != s_owner) return;
  double run = 0.0;
  int token = -1;
  for (int i = begin; i < end; ++i) {
    const double w = weight(a, d, first + i);
    if (!(w > 0.0)) continue;
    token = first + i;
    run += w;
    if (run >= s_left) break;
  }
  a.tokens[b] = token;
}

extern "C" const char* llmlab_last_error() { return g_llmlab_error; }

// Bytes of scratch of a call (8-byte aligned)
extern "C" size_t llmlab_verify_drafts_scratch(int n, int rows, int vocab, int with_draft) {
  const size_t chunks = ((size_t)vocab + CHUNK - 1) / CHUNK, all = (size_t)rows + (with_draft ? rows - n : 0);
  return all * chunks * 16 + (size_t)n * chunks * 8 + (size_t)n * sizeof(Decision);
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
  p += parts * 8;
  a.mass = (double*)p;
  p += (size_t)n * a.chunks * 8;
  a.decision = (Decision*)p;
  p += (size_t)n * sizeof(Decision);
  a.most = (float*)p;
  p += parts * 4;
  a.best = (int*)p;
  hipLaunchKernelGGL(verify_chunks_kernel, dim3(a.chunks, (unsigned)all), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(chunks)");
  hipLaunchKernelGGL(verify_decide_kernel, dim3(n), dim3(256), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(decide)");
  hipLaunchKernelGGL(verify_mass_kernel, dim3(a.chunks, n), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(mass)");
  hipLaunchKernelGGL(verify_draw_kernel, dim3(n), dim3(THREADS), 0, stream, a);
  LLMLAB_LAUNCH_CHECK("verify_drafts(draw)");
  return 0;
}
