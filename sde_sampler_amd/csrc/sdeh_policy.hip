// Losses over trajectories drawn before the update: the step log-ratio of two controls, the clipped policy loss with a KL term and the
// preference loss, each with its gradient (include/sdeh.h, ABI v8).  All of them are streams over [rows, steps] or [steps, batch, dim] tensors
// with a handful of operations per element: bounded by memory, and by their launches below about 1e5 entries.
#include "sdeh_elem.hpp"

namespace sdeh {

namespace {

constexpr int kThreads = 256;

// A launch holds fewer than 2^32 threads: kernels that take one piece of work a workgroup take theirs in several launches where there are more, each told
// how many workgroups the launches before it had.
constexpr long long kMostBlocks = 0xFFFFFFFFll / kThreads;

template <typename F>
void launch_pieces(long long blocks, const F& launch) {
  for (long long first = 0; first < blocks; first += kMostBlocks) launch(first, dim3((unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks)));
}

// i = row * steps + col; by 32-bit arithmetic where i fits it (a 64-bit division takes a hundred instructions and more)
__device__ __forceinline__ void split_index(long long i, long long steps, long long& row, long long& col) {
  if ((unsigned long long)i >> 32 == 0ull && (unsigned long long)steps >> 32 == 0ull) {
    const unsigned r = (unsigned)i / (unsigned)steps;
    row = r;
    col = (unsigned)i - r * (unsigned)steps;
  } else {
    row = i / steps;
    col = i - row * steps;
  }
}

// -------------------------------------------------------------------------------------------------------------------------------------------
// step log-ratio: l = sum_d e dW - dt/2 e^2, e = u - v;   gradient g (dW - dt e)
//
// A row is one trajectory at one step, dim coordinates: 1 .. a few hundred, seldom a multiple of what a lane loads at once.  A workgroup
// therefore takes `rows` whole rows -- one contiguous stretch, loaded 16 bytes a lane whatever dim is --, puts the elements' terms into LDS and
// sums the rows from there with G lanes a row.  dt differs from row to row only where a stretch passes the end of a step; it is staged per row.
// Bounded by memory: 200 x 4096 x 196 bf16 forward 0.18 ms (0.96 GB, 5.4 TB/s), backward 0.22 ms (1.28 GB, 5.9 TB/s); 200 x 2048 x 50 fp32 54 + 52 us.
// -------------------------------------------------------------------------------------------------------------------------------------------
constexpr int kStretch = 4096;      // elements of a stretch, at most (16 KB of terms)
constexpr int kStretchRows = 1024;  // rows of a stretch, at most
constexpr int kStagedDim = 512;     // rows longer than this are summed by a workgroup each, without LDS

struct RatioArgs {
  const void* u;
  const void* v;
  const void* dw;
  const float* dt;
  const float* g;
  void* out;
  long long rows_total, batch;
  int dim, rows, group;  // rows per stretch, lanes per row
  long long first;       // workgroups of the launches before
};

template <typename T, int V, bool BACK>
__global__ __launch_bounds__(kThreads) void ratio_kernel(RatioArgs a) {
  __shared__ float term[BACK ? 1 : kStretch + kStretch / 32];
  __shared__ float row_dt[kStretchRows];
  __shared__ float row_g[BACK ? kStretchRows : 1];
  const long long r0 = (a.first + blockIdx.x) * a.rows;
  const int nr = (int)(a.rows_total - r0 < a.rows ? a.rows_total - r0 : a.rows);
  const int d = a.dim, n = nr * d;
  const long long t0 = r0 / a.batch;  // (uniform over the workgroup)
  const long long b0 = r0 - t0 * a.batch;
  for (int r = threadIdx.x; r < nr; r += kThreads) {
    const long long b = b0 + r, t = b < a.batch ? t0 : t0 + b / a.batch;
    row_dt[r] = a.dt[t];
    if (BACK) row_g[r] = a.g[r0 + r];
  }
  __syncthreads();
  const T* u = static_cast<const T*>(a.u) + r0 * d;
  const T* v = a.v == nullptr ? nullptr : static_cast<const T*>(a.v) + r0 * d;
  const T* dw = static_cast<const T*>(a.dw) + r0 * d;
  T* out = static_cast<T*>(a.out) + r0 * d;
  for (int i = threadIdx.x * V; i < n; i += kThreads * V) {
    float xu[V], xv[V], xw[V];
    const int live = n - i < V ? n - i : V;
    if (live == V) {
      load_pack<T, V>(u + i, xu);
      load_pack<T, V>(dw + i, xw);
      if (v != nullptr) load_pack<T, V>(v + i, xv);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        xu[k] = k < live ? (float)u[i + k] : 0.0f;
        xw[k] = k < live ? (float)dw[i + k] : 0.0f;
        if (v != nullptr) xv[k] = k < live ? (float)v[i + k] : 0.0f;
      }
    }
    int r = (int)((unsigned)i / (unsigned)d), c = i - r * d;
    float dt = row_dt[r], g = BACK ? row_g[r] : 0.0f;
    float y[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float e = xu[k] - (v != nullptr ? xv[k] : 0.0f);
      if (BACK) {
        y[k] = g * (xw[k] - dt * e);
      } else {
        term[i + k + ((i + k) >> 5)] = e * (xw[k] - 0.5f * dt * e);  // (one word of padding in 32: rows of 32, 64, .. words spread over the banks)
      }
      if (++c == d && k + 1 < live) {
        c = 0;
        ++r;
        dt = row_dt[r];
        if (BACK) g = row_g[r];
      }
    }
    if (BACK) {
      if (live == V) {
        store_pack<T, V>(out + i, y);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k < live) out[i + k] = static_cast<T>(y[k]);
      }
    }
  }
  if (!BACK) {
    __syncthreads();
    const int G = a.group, lane = threadIdx.x & (G - 1);
    for (int r = threadIdx.x / G; r < nr; r += kThreads / G) {
      float s = 0.0f;
      for (int j = lane; j < d; j += G) {
        const int w = r * d + j;
        s += term[w + (w >> 5)];
      }
      for (int o = G >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      if (lane == 0) static_cast<float*>(a.out)[r0 + r] = s;
    }
  }
}

// The forward pass for rows of at least V coordinates and aligned tensors.  A vector of V elements then meets at most two rows: its lane sums the part
// before the row's end and the part after it, and only these two numbers go through LDS (2 words for V elements instead of V).  All loads of a stretch
// are on their way before the first is used.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void ratio_forward_kernel(RatioArgs a, unsigned inverse) {  // inverse = ceil(2^32 / dim)
  constexpr int kTurns = 2, kVectors = kTurns * kThreads;  // (four turns of fp32 took 140 registers: 60 instead of 54 us for 200 x 2048 x 50)
  __shared__ float before[kVectors], after[kVectors];
  __shared__ float row_dt[kStretchRows + 1];
  const long long r0 = (a.first + blockIdx.x) * a.rows;
  const int nr = (int)(a.rows_total - r0 < a.rows ? a.rows_total - r0 : a.rows);
  const int d = a.dim, n = nr * d, whole = n / V;
  const T* u = static_cast<const T*>(a.u) + r0 * d;
  const T* v = static_cast<const T*>(a.v != nullptr ? a.v : a.u) + r0 * d;
  const T* dw = static_cast<const T*>(a.dw) + r0 * d;
  Raw xu[kTurns]{}, xv[kTurns]{}, xw[kTurns]{};
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const int i = t * kThreads + threadIdx.x;
    if (i < whole) {
      xu[t] = load_raw(u + i * V);
      xv[t] = load_raw(v + i * V);
      xw[t] = load_raw(dw + i * V);
    }
  }
  const long long t0 = r0 / a.batch, b0 = r0 - t0 * a.batch;  // (uniform over the workgroup)
  for (int r = threadIdx.x; r <= nr; r += kThreads) {
    const long long b = b0 + r, t = b < a.batch ? t0 : t0 + b / a.batch;
    row_dt[r] = r < nr ? 0.5f * a.dt[t] : 0.0f;
  }
  __syncthreads();
  const float keep = a.v != nullptr ? 1.0f : 0.0f;
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const int i = t * kThreads + threadIdx.x;
    if (i < whole) {
      const int r = (int)__umulhi((unsigned)(i * V), inverse), left = (r + 1) * d - i * V;  // (elements of this row from here on)
      float pu[V], pv[V], pw[V];
      unpack<T, V>(xu[t], pu);
      unpack<T, V>(xv[t], pv);
      unpack<T, V>(xw[t], pw);
      float s1 = 0.0f, s2 = 0.0f, a1 = 0.0f, a2 = 0.0f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float e = keep != 0.0f ? pu[k] - pv[k] : pu[k];
        const bool here = k < left;
        const float eh = here ? e : 0.0f, ea = here ? 0.0f : e;  // (both factors: 0 times an infinite neighbour would be NaN in this row)
        s1 = fmaf(eh, here ? pw[k] : 0.0f, s1);
        s2 = fmaf(eh, eh, s2);
        a1 = fmaf(ea, here ? 0.0f : pw[k], a1);
        a2 = fmaf(ea, ea, a2);
      }
      before[i] = fmaf(-row_dt[r], s2, s1);
      after[i] = left < V ? fmaf(-row_dt[r + 1], a2, a1) : 0.0f;
    }
  }
  __syncthreads();
  const int G = a.group, lane = threadIdx.x & (G - 1);
  for (int r = threadIdx.x / G; r < nr; r += kThreads / G) {
    const int lo = r * d, hi = lo + d, first = (lo + V - 1) / V, last = (hi - 1) / V;  // vectors that start in the row
    float s = lane == 0 && lo % V != 0 ? after[lo / V] : 0.0f;
    for (int i = first + lane; i <= last; i += G) {
      if (i < whole) {
        s += before[i];
      } else {  // (less than a vector at the end of the last stretch)
        for (int k = whole * V; k < n; ++k) {
          const float e = (float)u[k] - (keep != 0.0f ? (float)v[k] : 0.0f);
          s += e * ((float)dw[k] - row_dt[r] * e);
        }
      }
    }
    for (int o = G >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) static_cast<float*>(a.out)[r0 + r] = s;
  }
}

// rows longer than kStagedDim: a workgroup sums one, an element a lane.  100 x 2048 x 784 fp32 forward 0.35 ms (5.4 TB/s), backward 5.7 TB/s; bf16, of which
// a lane loads 2 bytes at a time, forward 0.45 ms (2.1 TB/s), backward 2.8 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void ratio_long_kernel(RatioArgs a) {
  const long long row = a.first + blockIdx.x, base = row * a.dim;
  const T* u = static_cast<const T*>(a.u) + base;
  const T* v = a.v == nullptr ? nullptr : static_cast<const T*>(a.v) + base;
  const T* dw = static_cast<const T*>(a.dw) + base;
  const float half_dt = 0.5f * a.dt[row / a.batch];
  float s = 0.0f;
  for (int i = threadIdx.x; i < a.dim; i += kThreads) {
    const float e = (float)u[i] - (v != nullptr ? (float)v[i] : 0.0f);
    s += e * ((float)dw[i] - half_dt * e);
  }
  s = block_sum<kThreads>(s);
  if (threadIdx.x == 0) static_cast<float*>(a.out)[row] = s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ratio_long_back_kernel(RatioArgs a) {
  const long long row = a.first + blockIdx.x, base = row * a.dim;
  const T* u = static_cast<const T*>(a.u) + base;
  const T* v = a.v == nullptr ? nullptr : static_cast<const T*>(a.v) + base;
  const T* dw = static_cast<const T*>(a.dw) + base;
  T* out = static_cast<T*>(a.out) + base;
  const float dt = a.dt[row / a.batch], g = a.g[row];
  for (int i = threadIdx.x; i < a.dim; i += kThreads) {
    const float e = (float)u[i] - (v != nullptr ? (float)v[i] : 0.0f);
    out[i] = static_cast<T>(g * ((float)dw[i] - dt * e));
  }
}

template <typename T, bool BACK>
int launch_ratio_t(RatioArgs a, hipStream_t stream) {
  if (a.dim > kStagedDim) {
    launch_pieces(a.rows_total, [&](long long first, dim3 grid) {
      a.first = first;
      if (BACK)
        hipLaunchKernelGGL(ratio_long_back_kernel<T>, grid, dim3(kThreads), 0, stream, a);
      else
        hipLaunchKernelGGL(ratio_long_kernel<T>, grid, dim3(kThreads), 0, stream, a);
    });
    return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
  }
  // whole rows, a multiple of eight of them: every stretch then starts at a multiple of 16 bytes
  int rows = kStretch / a.dim / 8 * 8;
  a.rows = rows > kStretchRows ? kStretchRows : rows;
  a.group = 1;
  while (a.group < 64 && a.group * 2 * a.rows <= kThreads && a.group * 2 <= a.dim) a.group *= 2;
  constexpr int V = 16 / (int)sizeof(T);
  const bool wide = aligned_to(a.u, 16) && aligned_to(a.dw, 16) && (a.v == nullptr || aligned_to(a.v, 16)) && (!BACK || aligned_to(a.out, 16));
  const bool split = wide && !BACK && a.dim >= V;
  if (split) {
    a.rows = 2 * kThreads * V / a.dim / V * V;  // (whole rows, V of them: at least V as dim <= 512)
    a.group = 1;                                // (for the vectors of a row, not its elements)
    while (a.group < 64 && a.group * 2 * a.rows <= kThreads && a.group * 2 * V <= a.dim) a.group *= 2;
  }
  launch_pieces((a.rows_total + a.rows - 1) / a.rows, [&](long long first, dim3 grid) {
    a.first = first;
    if (split)
      hipLaunchKernelGGL((ratio_forward_kernel<T, V>), grid, dim3(kThreads), 0, stream, a, (unsigned)((0x100000000ull + a.dim - 1) / a.dim));
    else if (wide)
      hipLaunchKernelGGL((ratio_kernel<T, V, BACK>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((ratio_kernel<T, 1, BACK>), grid, dim3(kThreads), 0, stream, a);
  });
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

}  // namespace

int launch_step_log_ratio(const void* u, const void* v, const void* dw, const float* dt, const float* g, long long n_steps, long long batch,
                          int dim, int dtype, void* out, hipStream_t stream) {
  RatioArgs a{u, v, dw, dt, g, out, n_steps * batch, batch, dim, 0, 0, 0};
  if (g != nullptr)
    return dtype == SDEH_F32 ? launch_ratio_t<float, true>(a, stream)
                             : dtype == SDEH_BF16 ? launch_ratio_t<bf16_t, true>(a, stream) : launch_ratio_t<f16_t, true>(a, stream);
  return dtype == SDEH_F32 ? launch_ratio_t<float, false>(a, stream)
                           : dtype == SDEH_BF16 ? launch_ratio_t<bf16_t, false>(a, stream) : launch_ratio_t<f16_t, false>(a, stream);
}

namespace {

// -------------------------------------------------------------------------------------------------------------------------------------------
// clipped policy loss
//
// One pass reads every input once, forms the entry's loss and slope and writes the gradient; what it needs beforehand is the weight of an
// entry, i.e. how many entries are valid -- a pass over the mask's bytes alone (1 of 14 to 21 bytes an entry), which leaves partial counts that
// every workgroup of the main pass adds up again.  No atomics, no last-workgroup ticket: results do not depend on the order of workgroups and
// nothing has to be cleared between calls.
// 8192 x 8191 bf16 entries with a KL term and an advantage each, 62 % valid: 17 us for the mask, 131 us for the pass -- 0.6 GB, 100 us at the rate of a
// large copy; 60 vector instructions an entry take 76 us of it --, 5 us for the result.
// -------------------------------------------------------------------------------------------------------------------------------------------
constexpr int kCountBlocks = 1024, kPolicyBlocks = 2048, kSmallThreads = 1024;

struct PolicyArgs {
  SdehPolicyLoss p;
  long long n;          // rows * steps
  double log_hi, log_lo, log_dual;     // the borders' logarithms,
  float log_hi_f, log_lo_f, log_dual_f;  // and rounded
  float hi, lo, dual, kl_coef;
  const float* grad_scale;
  float grad_factor;
  void* grad;
  float* out;
  int* row_count;       // [rows]              scratch
  long long* part_n;    // [kCountBlocks]
  double* part;         // [kPolicyBlocks][4]
  int n_count, n_part;  // workgroups of the two passes
};

__device__ __forceinline__ bool needs_counts(const PolicyArgs& a) { return a.p.mask.data != nullptr && a.p.reduction != SDEH_REDUCE_SUM; }

// non-zero bytes of m[0 .. n), the share of thread `me` of `team`
__device__ __forceinline__ int count_span(const uint8_t* m, long long n, long long stride, long long me, long long team) {
  int c = 0;
  if (stride != 1) {
    for (long long i = me; i < n; i += team) c += m[i * stride] != 0;
    return c;
  }
  const long long to_border = (16 - (reinterpret_cast<uintptr_t>(m) & 15)) & 15, head = to_border < n ? to_border : n;
  const long long packs = (n - head) / 16;
  for (long long i = me; i < head; i += team) c += m[i] != 0;
#pragma unroll 4
  for (long long i = me; i < packs; i += team) {
    const Pack<unsigned, 4> k = *reinterpret_cast<const Pack<unsigned, 4>*>(m + head + 16 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) c += __popc((((k.v[j] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | k.v[j]) & 0x80808080u);  // (bit 7 of every byte that is not 0)
  }
  for (long long i = head + 16 * packs + me; i < n; i += team) c += m[i] != 0;
  return c;
}

// What the weights divide by, this workgroup's share: valid entries (SDEH_REDUCE_STEPS) or rows that have one (SDEH_REDUCE_ROWS; the row
// counts are kept).  A wave counts a row, of more than kLongRow entries the workgroup; a dense mask of SDEH_REDUCE_STEPS is one span.
constexpr long long kLongRow = 4096;

template <int NT>
__device__ __forceinline__ void count_pass(const PolicyArgs& a) {
  const uint8_t* m = static_cast<const uint8_t*>(a.p.mask.data);
  const long long T = a.p.steps;
  long long mine = 0;
  if (a.p.reduction == SDEH_REDUCE_STEPS && a.p.mask.step_stride == 1 && a.p.mask.row_stride == T) {
    mine = count_span(m, a.n, 1, (long long)blockIdx.x * NT + threadIdx.x, (long long)gridDim.x * NT);
  } else if (T > kLongRow) {
    for (long long row = blockIdx.x; row < a.p.rows; row += gridDim.x) {
      const int c = block_sum<NT>(count_span(m + row * a.p.mask.row_stride, T, a.p.mask.step_stride, threadIdx.x, NT));
      if (threadIdx.x == 0) {
        a.row_count[row] = c;
        mine += a.p.reduction == SDEH_REDUCE_ROWS ? c != 0 : c;
      }
    }
  } else {
    const int lane = threadIdx.x & 63;
    for (long long row = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); row < a.p.rows; row += (long long)gridDim.x * (NT / 64)) {
      const int c = wave_sum(count_span(m + row * a.p.mask.row_stride, T, a.p.mask.step_stride, lane, 64));
      if (lane == 0) {
        a.row_count[row] = c;
        mine += a.p.reduction == SDEH_REDUCE_ROWS ? c != 0 : c;
      }
    }
  }
  mine = block_sum<NT>(mine);
  if (threadIdx.x == 0) a.part_n[blockIdx.x] = mine;
}

// The weight that all entries have in common.
template <int NT>
__device__ __forceinline__ double common_weight(const PolicyArgs& a, int n_count) {
  if (a.p.reduction == SDEH_REDUCE_SUM) return 1.0;
  long long n = a.p.reduction == SDEH_REDUCE_ROWS ? a.p.rows : a.n;
  if (a.p.mask.data != nullptr) {
    long long s = 0;
    for (int i = threadIdx.x; i < n_count; i += NT) s += a.part_n[i];
    n = block_sum<NT>(s);
  }
  return 1.0 / (double)(n > 0 ? n : 1);
}

// exp(x) from the hardware's 2^y (one unit in the last place; results below 2^-126 become 0).  y = x log2(e) is rounded: off by at most
// (2 + 1.3 |x|) 2^-24 of itself, and a ratio's |x| is seldom above 1.  Two instructions where the library's takes thirteen.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502f); }

struct PolicySums {
  double policy, kl;
  unsigned clipped, valid;  // (a thread meets fewer than 2^32 entries)
};

// The KL term of V entries, k = log_prob - ref: value and slope.  (What does not depend on the entry is decided outside the loops over entries here and
// below: with these decisions inside, the compiler spent more instructions on branches than on the mathematics.)
//   k3: exp(-k) - 1 + k and 1 - exp(-k).  Up to |k| = 1 from a polynomial (the difference would lose the digits that exp(-k) and 1 - k share):
//   (exp(-k) - 1 + k) / k^2 through its eight Chebyshev nodes of [-1, 1], off by less than 2e-08 of itself with these coefficients.
template <int V>
__device__ __forceinline__ void kl_terms(int kind, const float (&x)[V], const float (&q)[V], float (&kl)[V], float (&slope)[V]) {
  if (kind == SDEH_KL_3) {
    bool far = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float k = x[j] - q[j];
      float s = -2.80628024e-06f;
      s = fmaf(k, s, 2.53585131e-05f);
      s = fmaf(k, s, -0.000198381022f);
      s = fmaf(k, s, 0.00138853968f);
      s = fmaf(k, s, -0.00833333936f);
      s = fmaf(k, s, 0.041666735f);
      s = fmaf(k, s, -0.166666672f);
      s = fmaf(k, s, 0.5f);
      kl[j] = k * k * s;
      slope[j] = k - kl[j];
      far |= !(fabsf(k) <= 1.0f);
    }
    if (far) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float k = x[j] - q[j], e = fast_exp(-k), far_kl = (e - 1.0f) + k, far_slope = 1.0f - e;
        const bool near = fabsf(k) <= 1.0f;
        kl[j] = near ? kl[j] : far_kl;
        slope[j] = near ? slope[j] : far_slope;
      }
    }
  } else if (kind == SDEH_KL_2) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      slope[j] = x[j] - q[j];
      kl[j] = 0.5f * slope[j] * slope[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      kl[j] = x[j] - q[j];
      slope[j] = 1.0f;
    }
  }
}

// V entries from their values: adds to `sums`, returns the gradients (without the loss's own scale).  MASKED: `ok` has a bit for each valid entry.
//
// Which side of a border the ratio lies on has to be right to the last bit of delta = x - o, whose fp32 value d is rounded.  Rounding is monotonic, so
// d > border (rounded) says delta > border (exactly) and d < border the opposite; only where they are equal are the 64-bit numbers compared, and d is
// moved to its neighbour beyond the border where delta lies beyond.  Then fp32 comparisons are right, and nothing but d depends on that rare branch.
template <int V, bool MASKED>
__device__ __forceinline__ void policy_entries(const PolicyArgs& a, const float (&x)[V], const float (&o)[V], const float (&q)[V], const float (&adv)[V],
                                               const float (&w)[V], unsigned ok, bool has_ref, bool row_weight, PolicySums& sums, float (&g)[V]) {
  float d[V];
  bool close = false;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    d[k] = adv[k] == 0.0f ? 0.0f : x[k] - o[k];  // (no advantage: nothing, whatever the ratio; 0 is never beyond a border)
    close |= (d[k] == (adv[k] > 0.0f ? a.log_hi_f : a.log_lo_f)) | (d[k] == a.log_dual_f);
  }
  if (close) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double delta = (double)x[k] - (double)o[k];
      if (adv[k] > 0.0f && d[k] == a.log_hi_f && delta > a.log_hi) d[k] = nextafterf(d[k], HUGE_VALF);
      if (adv[k] < 0.0f && d[k] == a.log_lo_f && delta < a.log_lo) d[k] = nextafterf(d[k], -HUGE_VALF);
      if (adv[k] < 0.0f && d[k] == a.log_dual_f && delta > a.log_dual) d[k] = nextafterf(d[k], HUGE_VALF);
    }
  }
  float surrogate[V], slope[V], kl[V];
  unsigned clips = 0;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const bool up = adv[k] > 0.0f, over = !up & (d[k] > a.log_dual_f);
    const bool beyond = (up ? d[k] : -d[k]) > (up ? a.log_hi_f : -a.log_lo_f), clipped = beyond | over;
    const float bound = over ? a.dual : up ? a.hi : a.lo, r = fast_exp(d[k]);
    surrogate[k] = -adv[k] * (clipped ? bound : r);
    slope[k] = clipped ? 0.0f : surrogate[k];
    kl[k] = 0.0f;
    if (MASKED)
      clips |= clipped ? 1u << k : 0u;
    else
      sums.clipped += clipped;
  }
  if (has_ref) {
    float kl_slope[V];
    kl_terms<V>(a.p.kl, x, q, kl, kl_slope);
#pragma unroll
    for (int k = 0; k < V; ++k) slope[k] = fmaf(a.kl_coef, kl_slope[k], slope[k]);
  }
  if (row_weight) {  // (rounded once more each, 2^-24 of themselves: the common weight of SDEH_REDUCE_STEPS is applied to the 64-bit sum instead)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      surrogate[k] *= w[k];
      kl[k] *= w[k];
    }
  }
  // V entries are added in 32 bits, off by at most V 2^-24 of their absolute sum, all further sums in 64: each entry in 64 bits would be two conversions and
  // two 64-bit additions more of a pass that its instructions bound already
  float policy = 0.0f, kls = 0.0f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const bool in = !MASKED || (ok >> k & 1u) != 0u;
    policy += in ? surrogate[k] : 0.0f;
    kls += in ? kl[k] : 0.0f;
    g[k] = in ? slope[k] * w[k] : 0.0f;
  }
  if (MASKED) sums.clipped += __popc(clips & ok);
  sums.valid += MASKED ? __popc(ok) : V;
  sums.policy += (double)policy;
  sums.kl += (double)kls;
}

// bit k of the result: byte k of the word is not 0
__device__ __forceinline__ unsigned byte_bits(unsigned m) {
  const unsigned t = (((m & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | m) & 0x80808080u;
  return (t >> 7 & 1u) | (t >> 14 & 2u) | (t >> 21 & 4u) | (t >> 28 & 8u);
}

// the same of V bytes (4 or 8, aligned to as many)
template <int V>
__device__ __forceinline__ unsigned byte_mask(const uint8_t* m) {
  const Pack<unsigned, V / 4> k = *reinterpret_cast<const Pack<unsigned, V / 4>*>(m);
  unsigned ok = byte_bits(k.v[0]);
  if constexpr (V == 8) ok |= byte_bits(k.v[1]) << 4;
  return ok;
}

// what a pass needs throughout
struct PolicyView {
  bool has_ref, row_weight;
  float w_all, factor;
};

__device__ __forceinline__ PolicyView policy_view(const PolicyArgs& a, double w_common) {
  PolicyView v;
  v.has_ref = a.p.ref_log_prob.data != nullptr;
  v.row_weight = a.p.reduction == SDEH_REDUCE_ROWS;
  // a row's weight is taken from its count where there is a mask; without one all rows have as many entries
  v.w_all = (float)(v.row_weight && a.p.mask.data == nullptr ? w_common / (double)a.p.steps : w_common);
  v.factor = a.grad_factor * (a.grad_scale != nullptr ? *a.grad_scale : 1.0f);
  return v;
}

// one entry of planes with any strides
template <typename T>
__device__ __forceinline__ void policy_one(const PolicyArgs& a, const PolicyView& v, long long row, long long col, PolicySums& sums) {
  const SdehPolicyLoss& p = a.p;
  const auto at = [&](const SdehPlane& q) { return (float)static_cast<const T*>(q.data)[row * q.row_stride + col * q.step_stride]; };
  float g[1] = {0.0f};
  if (p.mask.data == nullptr || static_cast<const uint8_t*>(p.mask.data)[row * p.mask.row_stride + col * p.mask.step_stride] != 0) {
    const float x[1] = {at(p.log_prob)}, o[1] = {p.old_log_prob.data != nullptr ? at(p.old_log_prob) : 0.0f}, q[1] = {v.has_ref ? at(p.ref_log_prob) : 0.0f};
    const float adv[1] = {load_as(p.advantage.data, p.advantage_dtype, row * p.advantage.row_stride + col * p.advantage.step_stride)};
    const float w[1] = {v.row_weight && p.mask.data != nullptr ? v.w_all / (float)a.row_count[row] : v.w_all};
    policy_entries<1, false>(a, x, o, q, adv, w, 1u, v.has_ref, v.row_weight, sums, g);
  }
  if (a.grad != nullptr) static_cast<T*>(a.grad)[row * p.steps + col] = static_cast<T>(g[0] * v.factor);
}

// All entries.  V > 1: every plane is contiguous and aligned, V neighbours a thread; V = 1: any strides.  ROW: the entry's row matters (an advantage or a
// weight of its own); without it the entries are one stream.
//
// V = 1 reads an entry a lane, along the steps: on transposed planes ([steps, rows] in memory, as step_log_ratio leaves them) neighbouring lanes are a
// column apart.  2048 x 200 fp32, KL, value and gradient: 23 us transposed, 21 by rows (host); 65536 x 200: 201 and 42 us, with a mask 280 and 59.
//
// The grid goes over the entries in rounds, a tile of NT V neighbours a workgroup.  With rows that end early, a workgroup that met the same place of
// every row would have nothing but valid entries, another nothing but padding, wherever a round's length is near a multiple of `steps`: the workgroups
// change places from round to round.
template <typename T, int V, int NT, bool ROW>
__device__ __forceinline__ PolicySums policy_pass(const PolicyArgs& a) {
  PolicySums sums{0.0, 0.0, 0, 0};
  const SdehPolicyLoss& p = a.p;
  const long long me = (long long)blockIdx.x * NT + threadIdx.x, body = a.n / V * V;
  const unsigned shift = (unsigned)((unsigned long long)gridDim.x * 382u / 1000u) | 1u;
  const auto place = [&](long long round) {  // first entry of this workgroup's tile
    const unsigned at = (unsigned)((blockIdx.x + (unsigned long long)round * shift) % gridDim.x);
    return (round * gridDim.x + at) * ((long long)NT * V);
  };
  const long long rounds = (body + (long long)gridDim.x * NT * V - 1) / ((long long)gridDim.x * NT * V);
  if constexpr (V == 1) {
    const PolicyView v = policy_view(a, common_weight<NT>(a, a.n_count));
    for (long long round = 0; round < rounds; ++round) {
      const long long i = place(round) + threadIdx.x;
      if (i < body) {
        long long row, col;
        split_index(i, p.steps, row, col);
        policy_one<T>(a, v, row, col, sums);
      }
    }
  } else {
    const T* lp = static_cast<const T*>(p.log_prob.data);
    const T* old = static_cast<const T*>(p.old_log_prob.data);
    const T* ref = static_cast<const T*>(p.ref_log_prob.data);
    const uint8_t* mask = static_cast<const uint8_t*>(p.mask.data);
    T* grad = static_cast<T*>(a.grad);
    const bool row_adv = p.advantage.step_stride == 0;
    constexpr unsigned kAll = (1u << V) - 1u;
    // Two vectors ahead its mask, one vector ahead its values are on their way: what is loaded depends on the mask, and four or five waves of this many
    // registers do not cover both latencies by themselves.
    const auto load_mask = [&](long long at) {
      Pack<unsigned, V / 4> m{};
      if (mask != nullptr && at < body) m = *reinterpret_cast<const Pack<unsigned, V / 4>*>(mask + at);
      return m;
    };
    const auto valid = [&](const Pack<unsigned, V / 4>& m, long long at) {
      if (at >= body) return 0u;
      if (mask == nullptr) return kAll;
      unsigned ok = byte_bits(m.v[0]);
      if constexpr (V == 8) ok |= byte_bits(m.v[1]) << 4;
      return ok;
    };
    // (absent planes are read from log_prob's place, so that no load waits behind a branch, and count as 0)
    const T* old_at = old != nullptr ? old : lp;
    const T* ref_at = ref != nullptr ? ref : lp;
    Raw next_x{}, next_o{}, next_q{}, next_a[V / 4]{};
    const auto load_values = [&](long long at, unsigned ok) {
      if (ok != 0u) {  // (a stretch of padding is neither read nor computed)
        next_x = load_raw(lp + at);
        next_o = load_raw(old_at + at);
        next_q = load_raw(ref_at + at);
        if constexpr (!ROW) {  // (the advantage is fp32 and laid out like the rest)
#pragma unroll
          for (int k = 0; k < V / 4; ++k) next_a[k] = load_raw(static_cast<const float*>(p.advantage.data) + at + 4 * k);
        }
      }
    };
    const long long mine = (long long)threadIdx.x * V;
    long long start = place(0), start_next = rounds > 1 ? place(1) : body;
    unsigned ok_next = valid(load_mask(start + mine), start + mine);
    load_values(start + mine, ok_next);
    Pack<unsigned, V / 4> m = load_mask(start_next + mine);
    const PolicyView v = policy_view(a, common_weight<NT>(a, a.n_count));
    const bool count = v.row_weight && mask != nullptr;
    for (long long round = 0; round < rounds; ++round) {
      const long long i = start + mine;
      const unsigned ok = ok_next;
      float x[V], o[V], q[V], adv[V], w[V];
      unpack<T, V>(next_x, x);
      unpack<T, V>(next_o, o);
      unpack<T, V>(next_q, q);
      if constexpr (!ROW) {
#pragma unroll
        for (int k = 0; k < V; ++k) adv[k] = __uint_as_float(next_a[k / 4][k % 4]);
      }
      ok_next = valid(m, start_next + mine);
      load_values(start_next + mine, ok_next);
      long long row = 0, col = 0;
      if constexpr (ROW) {  // (the tile's place by 64-bit arithmetic of the whole wave, the thread's in it by 32-bit arithmetic)
        long long r0, c0;
        split_index(start, p.steps, r0, c0);
        const unsigned t = (unsigned)c0 + (unsigned)mine, r = t / (unsigned)p.steps;
        row = r0 + r;
        col = t - r * (unsigned)p.steps;
      }
      start = start_next;
      start_next = round + 2 < rounds ? place(round + 2) : body;
      m = load_mask(start_next + mine);
      float g[V];
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = 0.0f;
      if (ok != 0u) {
        if (old == nullptr) {
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] = 0.0f;
        }
        if constexpr (!ROW) {
#pragma unroll
          for (int k = 0; k < V; ++k) w[k] = v.w_all;
        } else if (row_adv && col + V <= p.steps) {  // (one row)
          const float A = load_as(p.advantage.data, p.advantage_dtype, row * p.advantage.row_stride);
          const float wr = count ? v.w_all / (float)a.row_count[row] : v.w_all;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            adv[k] = A;
            w[k] = wr;
          }
        } else {
          long long r = row, c = col;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            adv[k] = load_as(p.advantage.data, p.advantage_dtype, r * p.advantage.row_stride + c * p.advantage.step_stride);
            w[k] = count ? v.w_all / (float)a.row_count[r] : v.w_all;  // (a row without a valid entry: nothing of it is added)
            if (++c == p.steps) {
              c = 0;
              ++r;
            }
          }
        }
        if (ok == kAll)
          policy_entries<V, false>(a, x, o, q, adv, w, ok, v.has_ref, v.row_weight, sums, g);
        else
          policy_entries<V, true>(a, x, o, q, adv, w, ok, v.has_ref, v.row_weight, sums, g);
      }
      if (grad != nullptr) {
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] *= v.factor;
        if (i < body) store_pack<T, V>(grad + i, g);
      }
    }
    if (me < a.n - body) policy_one<T>(a, v, (body + me) / p.steps, (body + me) % p.steps, sums);  // (less than a vector is left)
  }
  return sums;
}

// out = loss, policy, kl, clipped share, valid entries; the sums of SDEH_REDUCE_STEPS still want their common weight
__device__ __forceinline__ void policy_result(const PolicyArgs& a, double policy, double kl, double clipped, double valid) {
  const double n = valid > 0.0 ? valid : 1.0;
  if (a.p.reduction == SDEH_REDUCE_STEPS) {
    policy /= n;
    kl /= n;
  }
  a.out[0] = (float)(policy + a.p.kl_coef * kl);
  a.out[1] = (float)policy;
  a.out[2] = (float)kl;
  a.out[3] = (float)(clipped / n);
  a.out[4] = (float)valid;
}

template <int NT>
__global__ __launch_bounds__(NT) void policy_count_kernel(PolicyArgs a) {
  count_pass<NT>(a);
}

template <typename T, int V, bool ROW>
__global__ __launch_bounds__(kThreads) void policy_kernel(PolicyArgs a) {
  const PolicySums s = policy_pass<T, V, kThreads, ROW>(a);
  if (a.out == nullptr) return;
  const double policy = block_sum<kThreads>(s.policy), kl = block_sum<kThreads>(s.kl);
  const long long clipped = block_sum<kThreads>((long long)s.clipped), valid = block_sum<kThreads>((long long)s.valid);
  if (threadIdx.x == 0) {
    double* o = a.part + 4 * blockIdx.x;
    o[0] = policy;
    o[1] = kl;
    o[2] = (double)clipped;
    o[3] = (double)valid;
  }
}

__global__ __launch_bounds__(kThreads) void policy_final_kernel(PolicyArgs a) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < a.n_part; i += kThreads)
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += a.part[4 * i + k];
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = block_sum<kThreads>(s[k]);
  if (threadIdx.x == 0) policy_result(a, s[0], s[1], s[2], s[3]);
}

// few entries: counting, the pass and the result by one workgroup in one launch
template <typename T, int V>
__global__ __launch_bounds__(kSmallThreads) void policy_small_kernel(PolicyArgs a) {
  if (needs_counts(a)) {
    count_pass<kSmallThreads>(a);
    __threadfence_block();
    __syncthreads();
  }
  const PolicySums s = policy_pass<T, V, kSmallThreads, true>(a);
  if (a.out == nullptr) return;
  const double policy = block_sum<kSmallThreads>(s.policy), kl = block_sum<kSmallThreads>(s.kl);
  const long long clipped = block_sum<kSmallThreads>((long long)s.clipped), valid = block_sum<kSmallThreads>((long long)s.valid);
  if (threadIdx.x == 0) policy_result(a, policy, kl, (double)clipped, (double)valid);
}

// Entries that one workgroup takes, in one launch.  Replayed from a graph, fp32 with a mask and row weights: 1024 entries 10.7 us, 4096 13.1, 8192 17.3;
// in three launches 12.0 us from 16384 on (without a mask 7.1, 7.9, 9.6; in two launches 7.6).  On the host each launch less saves 3 us.
constexpr long long kPolicySmall = 4096;

bool dense(const SdehPlane& q, long long steps, size_t bytes) {
  return q.data == nullptr || (q.step_stride == 1 && q.row_stride == steps && aligned_to(q.data, bytes));
}

template <typename T>
int launch_policy_t(PolicyArgs a, bool reuse_counts, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  const SdehPolicyLoss& p = a.p;
  const bool adv_ok = p.advantage.step_stride == 0 || p.advantage.step_stride == 1;
  const bool wide = dense(p.log_prob, p.steps, 16) && dense(p.old_log_prob, p.steps, 16) && dense(p.ref_log_prob, p.steps, 16) &&
                    dense(p.mask, p.steps, V) && adv_ok && aligned_to(a.grad, 16);
  const bool stream_only = wide && p.advantage_dtype == SDEH_F32 && dense(p.advantage, p.steps, 16) && (p.reduction != SDEH_REDUCE_ROWS || p.mask.data == nullptr);
  const int v = wide ? V : 1;
  const bool small = a.n <= kPolicySmall;
  const int nt = small ? kSmallThreads : kThreads;
  const long long tiles = (a.n + (long long)nt * v - 1) / ((long long)nt * v), most = wide && V == 8 ? kPolicyBlocks / 2 : kPolicyBlocks;
  const long long blocks = small || tiles == 0 ? 1 : tiles > most ? most : tiles;  // (as many as are resident at once)
  a.n_part = (int)blocks;
  if (small) {
    a.n_count = 1;
    if (wide)
      hipLaunchKernelGGL((policy_small_kernel<T, V>), dim3(1), dim3(kSmallThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((policy_small_kernel<T, 1>), dim3(1), dim3(kSmallThreads), 0, stream, a);
    return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
  }
  const bool span = p.reduction == SDEH_REDUCE_STEPS && p.mask.step_stride == 1 && p.mask.row_stride == p.steps, long_rows = p.steps > kLongRow;
  const long long count_blocks = span ? (a.n + 16 * kThreads - 1) / (16 * kThreads) : long_rows ? p.rows : (p.rows + kThreads / 64 - 1) / (kThreads / 64);
  a.n_count = (int)(count_blocks > kCountBlocks ? kCountBlocks : count_blocks);
  if (p.mask.data != nullptr && p.reduction != SDEH_REDUCE_SUM && !reuse_counts) {
    if (long_rows && !span)
      hipLaunchKernelGGL(policy_count_kernel<kSmallThreads>, dim3(a.n_count), dim3(kSmallThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(policy_count_kernel<kThreads>, dim3(a.n_count), dim3(kThreads), 0, stream, a);
  }
  if (stream_only)
    hipLaunchKernelGGL((policy_kernel<T, V, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
  else if (wide)
    hipLaunchKernelGGL((policy_kernel<T, V, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((policy_kernel<T, 1, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
  if (a.out != nullptr) hipLaunchKernelGGL(policy_final_kernel, dim3(1), dim3(kThreads), 0, stream, a);
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

}  // namespace

// scratch: partial sums, partial counts, row counts
long long policy_scratch_floats(long long rows, long long steps, bool masked) {
  if (!masked && rows * steps <= kPolicySmall) return 0;
  return kPolicyBlocks * 8ll + kCountBlocks * 2ll + (rows + 1) / 2 * 2;
}

int launch_policy_loss(const SdehPolicyLoss& p, float* scratch, int reuse_counts, const float* grad_scale, float grad_factor, float* out,
                       void* grad, hipStream_t stream) {
  PolicyArgs a{};
  a.p = p;
  a.n = p.rows * p.steps;
  a.log_hi = log1p(p.clip_high);
  a.log_lo = p.clip_low < 1.0 ? log1p(-p.clip_low) : -HUGE_VAL;
  a.log_dual = p.dual_clip > 0.0 ? log(p.dual_clip) : HUGE_VAL;
  a.log_hi_f = (float)a.log_hi;
  a.log_lo_f = (float)a.log_lo;
  a.log_dual_f = (float)a.log_dual;
  a.hi = (float)(1.0 + p.clip_high);
  a.lo = (float)(1.0 - p.clip_low);
  a.dual = (float)p.dual_clip;
  a.kl_coef = (float)p.kl_coef;
  a.grad_scale = grad_scale;
  a.grad_factor = grad_factor;
  a.grad = grad;
  a.out = out;
  a.part = reinterpret_cast<double*>(scratch);
  a.part_n = reinterpret_cast<long long*>(scratch + kPolicyBlocks * 8ll);
  a.row_count = reinterpret_cast<int*>(scratch + kPolicyBlocks * 8ll + kCountBlocks * 2ll);
  return p.dtype == SDEH_F32 ? launch_policy_t<float>(a, reuse_counts != 0, stream)
                             : p.dtype == SDEH_BF16 ? launch_policy_t<bf16_t>(a, reuse_counts != 0, stream)
                                                    : launch_policy_t<f16_t>(a, reuse_counts != 0, stream);
}

namespace {

// -------------------------------------------------------------------------------------------------------------------------------------------
// preference loss: sums of the rows (split over their length where rows are few and long), the pairs, the gradients
//
// A pair's slope is known only when both its rows are summed, so the gradient -- the slope again and again, 0 in the padding -- is a second
// pass; it reads nothing but the mask.  24 pairs of 2.6e5 and 2.0e5 fp16 entries: sums 15 us, pairs 5, gradients 9 (77 MB, 12 us at the rate of a large
// copy); up to 4096 entries everything in one launch, 6 to 9 us.
// -------------------------------------------------------------------------------------------------------------------------------------------
constexpr int kPairBlocks = 256;

struct PreferenceArgs {
  SdehPreferenceLoss p;
  int splits;               // parts of a row
  long long first;          // workgroups of the launches before (preference_sum_kernel)
  long long chunk;          // entries of a part
  double* sum;              // [2 pairs][splits]   scratch
  long long* count;         // [2 pairs][splits]
  double* part;             // [kPairBlocks][2]
  int n_pair_blocks;
  float* out;
  const float* slopes;      // [2][pairs]
  const float* grad_scale;
  float grad_factor;
  void* grad[2];
  long long d_row[2], d_col[2];
};

// Sum and number of the valid entries [lo, hi) of a row, this thread's share: `me` of `team` threads, U vectors at a time.
template <typename T, int V, int U>
__device__ __forceinline__ void row_share(const SdehPreferenceSide& s, long long row, long long lo, long long hi, int me, int team, double& sum,
                                          long long& count) {
  const T* x = static_cast<const T*>(s.log_prob.data) + row * s.log_prob.row_stride;
  const T* q = s.ref_log_prob.data == nullptr ? nullptr : static_cast<const T*>(s.ref_log_prob.data) + row * s.ref_log_prob.row_stride;
  const uint8_t* m = s.mask.data == nullptr ? nullptr : static_cast<const uint8_t*>(s.mask.data) + row * s.mask.row_stride;
  const auto one = [&](long long i) {
    if (m == nullptr || m[i * s.mask.step_stride] != 0) {
      const double a = (double)(float)x[i * s.log_prob.step_stride];
      sum += q == nullptr ? a : a - (double)(float)q[i * s.ref_log_prob.step_stride];
      ++count;
    }
  };
  if constexpr (V == 1) {
    for (long long i = lo + me; i < hi; i += team) one(i);
    return;
  } else {
    // contiguous planes with one row stride: entries up to the first 16-byte border (the same in every plane), vectors, the rest
    const long long flat = row * s.log_prob.row_stride;
    long long head = lo + (V - (flat + lo) % V) % V;
    if (head > hi) head = hi;
    const long long body = head + (hi - head) / V * V;
    for (long long i = lo + me; i < head; i += team) one(i);
    // the masks' loads, then the loads of those vectors that have a valid entry, then the sums
    const T* q_at = q != nullptr ? q : x;
    constexpr unsigned kAll = (1u << V) - 1u;
    const long long step = (long long)team * V;
    for (long long i = head + (long long)me * V; i < body; i += U * step) {
      unsigned ok[U];
      Raw a[U]{}, b[U]{};
#pragma unroll
      for (int t = 0; t < U; ++t) {
        ok[t] = i + t * step < body ? kAll : 0u;
        if (m != nullptr && ok[t] != 0u) ok[t] = byte_mask<V>(m + i + t * step);
      }
#pragma unroll
      for (int t = 0; t < U; ++t) {
        if (ok[t] != 0u) {
          a[t] = load_raw(x + i + t * step);
          b[t] = load_raw(q_at + i + t * step);
        }
      }
#pragma unroll
      for (int t = 0; t < U; ++t) {
        if (ok[t] != 0u) {
          float fa[V], fb[V];
          unpack<T, V>(a[t], fa);
          unpack<T, V>(b[t], fb);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float at = ok[t] >> j & 1u ? fa[j] : 0.0f, bt = q != nullptr && (ok[t] >> j & 1u) ? fb[j] : 0.0f;
            sum += (double)at - (double)bt;
          }
          count += __popc(ok[t]);
        }
      }
    }
    for (long long i = body + me; i < hi; i += team) one(i);
  }
}

// one workgroup a part of a row
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void preference_sum_kernel(PreferenceArgs a) {
  const long long part = a.first + blockIdx.x, line = part / a.splits;
  const int split = (int)(part - line * a.splits);
  const bool second = line >= a.p.pairs;
  const SdehPreferenceSide& s = second ? a.p.rejected : a.p.chosen;
  const long long lo = split * a.chunk, hi = lo + a.chunk < s.steps ? lo + a.chunk : s.steps;
  double sum = 0.0;
  long long count = 0;
  if (lo < hi) row_share<T, V, 4>(s, second ? line - a.p.pairs : line, lo, hi, threadIdx.x, kThreads, sum, count);
  sum = block_sum<kThreads>(sum);
  count = block_sum<kThreads>(count);
  if (threadIdx.x == 0) {
    a.sum[part] = sum;
    a.count[part] = count;
  }
}

// short rows: one wave a row
template <typename T, int V, int NT>
__device__ __forceinline__ void short_rows(const PreferenceArgs& a, long long first, long long step) {
  for (long long line = first; line < 2 * a.p.pairs; line += step) {
    const bool second = line >= a.p.pairs;
    const SdehPreferenceSide& s = second ? a.p.rejected : a.p.chosen;
    double sum = 0.0;
    long long count = 0;
    row_share<T, V, 1>(s, second ? line - a.p.pairs : line, 0, s.steps, threadIdx.x & 63, 64, sum, count);
    sum = wave_sum(sum);
    count = wave_sum(count);
    if ((threadIdx.x & 63) == 0) {
      a.sum[line] = sum;
      a.count[line] = count;
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void preference_short_kernel(PreferenceArgs a) {
  short_rows<T, V, kThreads>(a, (long long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), (long long)gridDim.x * (kThreads / 64));
}

// loss and slope of one pair from its rows' sums; adds to (loss, correct)
__device__ __forceinline__ void one_pair(const PreferenceArgs& a, long long i, double sc, long long nc, double sr, long long nr, double& loss,
                                         double& correct) {
  const long long P = a.p.pairs;
  double wc = 1.0, wr = 1.0;
  if (a.p.average) {
    wc = 1.0 / (double)(nc > 0 ? nc : 1);
    wr = 1.0 / (double)(nr > 0 ? nr : 1);
  }
  sc *= wc;
  sr *= wr;
  const double beta = a.p.beta, gap = sc - sr, h = beta * gap, eps = a.p.label_smoothing;
  double l, slope;
  if (a.p.kind == SDEH_PREF_LOGISTIC) {
    const double e = exp(-fabs(h)), tail = log1p(e);  // -log sigmoid(+-h) = log1p(e^-|h|) + max(-+h, 0)
    l = (1.0 - eps) * (tail + (h < 0.0 ? -h : 0.0)) + (eps > 0.0 ? eps * (tail + (h > 0.0 ? h : 0.0)) : 0.0);
    const double away = h >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);  // sigmoid(-h)
    slope = beta * (eps - away);
  } else if (a.p.kind == SDEH_PREF_HINGE) {
    l = h < 1.0 ? 1.0 - h : 0.0;
    slope = h < 1.0 ? -beta : 0.0;
    if (h != h) l = slope = h;
  } else {
    const double r = gap - 0.5 / beta;
    l = r * r;
    slope = 2.0 * r;
  }
  slope /= (double)P;
  float* o = a.out + 2;
  o[i] = (float)(beta * sc);
  o[P + i] = (float)(beta * sr);
  o[2 * P + i] = (float)(slope * wc);
  o[3 * P + i] = (float)(-slope * wr);
  loss += l;
  correct += h > 0.0 ? 1.0 : 0.0;
}

// splits == 1: a thread a pair, else a wave
template <int NT>
__device__ __forceinline__ void pairs_pass(const PreferenceArgs& a, double& loss, double& correct) {
  const long long P = a.p.pairs;
  const int S = a.splits;
  if (S == 1) {
    for (long long i = (long long)blockIdx.x * NT + threadIdx.x; i < P; i += (long long)gridDim.x * NT)
      one_pair(a, i, a.sum[i], a.count[i], a.sum[P + i], a.count[P + i], loss, correct);
    return;
  }
  const int lane = threadIdx.x & 63;
  for (long long i = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); i < P; i += (long long)gridDim.x * (NT / 64)) {
    double s[2] = {0.0, 0.0};
    long long n[2] = {0, 0};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      for (int k = lane; k < S; k += 64) {
        s[side] += a.sum[(side * P + i) * S + k];
        n[side] += a.count[(side * P + i) * S + k];
      }
      s[side] = wave_sum(s[side]);
      n[side] = wave_sum(n[side]);
    }
    if (lane == 0) one_pair(a, i, s[0], n[0], s[1], n[1], loss, correct);
  }
}

__global__ __launch_bounds__(kThreads) void preference_pair_kernel(PreferenceArgs a) {
  double loss = 0.0, correct = 0.0;
  pairs_pass<kThreads>(a, loss, correct);
  loss = block_sum<kThreads>(loss);
  correct = block_sum<kThreads>(correct);
  if (threadIdx.x == 0) {
    const double P = (double)a.p.pairs;
    if (gridDim.x == 1) {
      a.out[0] = (float)(loss / P);
      a.out[1] = (float)(correct / P);
    } else {
      a.part[2 * blockIdx.x] = loss;
      a.part[2 * blockIdx.x + 1] = correct;
    }
  }
}

// the means, from the workgroups' sums
__device__ __forceinline__ void preference_means(const PreferenceArgs& a) {
  double loss = 0.0, correct = 0.0;
  for (int i = threadIdx.x; i < a.n_pair_blocks; i += kThreads) {
    loss += a.part[2 * i];
    correct += a.part[2 * i + 1];
  }
  loss = block_sum<kThreads>(loss);
  correct = block_sum<kThreads>(correct);
  if (threadIdx.x == 0) {
    a.out[0] = (float)(loss / (double)a.p.pairs);
    a.out[1] = (float)(correct / (double)a.p.pairs);
  }
}

__global__ __launch_bounds__(kThreads) void preference_final_kernel(PreferenceArgs a) { preference_means(a); }

// gradients of one side: the pair's slope on valid entries
template <typename T, int V, int NT>
__device__ __forceinline__ void spread_pass(const PreferenceArgs& a, int side, const float* slopes) {
  const SdehPreferenceSide& s = side ? a.p.rejected : a.p.chosen;
  const uint8_t* m = static_cast<const uint8_t*>(s.mask.data);
  T* grad = static_cast<T*>(a.grad[side]);
  const float factor = a.grad_factor * (a.grad_scale != nullptr ? *a.grad_scale : 1.0f);
  const long long n = a.p.pairs * s.steps, stride = (long long)gridDim.x * NT * V;
  long long i = ((long long)blockIdx.x * NT + threadIdx.x) * V;
  if (i >= n) return;
  long long row, col;
  split_index(i, s.steps, row, col);
  for (; i < n; i += stride) {
    if (V > 1 && n - i >= V) {
      float g[V];
      if constexpr (V > 1) {
        const unsigned ok = m == nullptr ? (1u << V) - 1u : byte_mask<V>(m + i);
        const float slope = slopes[row] * factor;
        if (col + V <= s.steps) {  // (one row)
#pragma unroll
          for (int k = 0; k < V; ++k) g[k] = ok >> k & 1u ? slope : 0.0f;
        } else {
          long long r = row, c = col;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            g[k] = ok >> k & 1u ? slopes[r] * factor : 0.0f;
            if (++c == s.steps) {
              c = 0;
              r += k + 1 < V;
            }
          }
        }
      }
      store_pack<T, V>(grad + i, g);
    } else {
      long long r = row, c = col;
      for (long long k = i; k < n && k < i + V; ++k) {
        const bool ok = m == nullptr || m[V > 1 ? k : r * s.mask.row_stride + c * s.mask.step_stride] != 0;
        grad[k] = static_cast<T>(ok ? slopes[r] * factor : 0.0f);
        if (++c == s.steps) {
          c = 0;
          ++r;
        }
      }
    }
    row += a.d_row[side];
    col += a.d_col[side];
    if (col >= s.steps) {
      col -= s.steps;
      ++row;
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void preference_grad_kernel(PreferenceArgs a) {
  const int side = blockIdx.y;
  spread_pass<T, V, kThreads>(a, side, a.slopes + side * a.p.pairs);
  if (a.n_pair_blocks > 1 && blockIdx.x == 0 && side == 0) preference_means(a);  // (a launch less)
}

// few and short rows: everything by one workgroup
template <typename T, int V>
__global__ __launch_bounds__(kSmallThreads) void preference_small_kernel(PreferenceArgs a) {
  short_rows<T, V, kSmallThreads>(a, threadIdx.x >> 6, kSmallThreads / 64);
  __threadfence_block();
  __syncthreads();
  double loss = 0.0, correct = 0.0;
  pairs_pass<kSmallThreads>(a, loss, correct);
  __threadfence_block();
  loss = block_sum<kSmallThreads>(loss);
  correct = block_sum<kSmallThreads>(correct);
  if (threadIdx.x == 0) {
    a.out[0] = (float)(loss / (double)a.p.pairs);
    a.out[1] = (float)(correct / (double)a.p.pairs);
  }
  if (a.grad[0] != nullptr) {
    spread_pass<T, V, kSmallThreads>(a, 0, a.out + 2 + 2 * a.p.pairs);
    spread_pass<T, V, kSmallThreads>(a, 1, a.out + 2 + 3 * a.p.pairs);
  }
}

// Entries of both sides that one workgroup takes, in one launch: 1024 entries 6.4 us, 4096 8.5, 8192 11.6; in three launches 7.6 us from 16384 on.
constexpr long long kPreferenceSmall = 4096;
constexpr long long kShortRow = 1024;         // rows that a wave sums
constexpr int kMaxSplits = 64;

// parts of a row: a workgroup a part of 4096 entries or more, and 2048 workgroups where rows are few (those that get padding end at once).  24 pairs of 2.6
// million fp16 entries and their gradients: 132 us with 2048 or 4096 workgroups, 141 with 1024.  At most 64 parts, which a wave adds up in one go; only
// one or two pairs of many million entries would gain by more (a pair of 16 million: 66 us, in 256 parts 41).
int preference_splits(const SdehPreferenceLoss& p) {
  const long long longest = p.chosen.steps > p.rejected.steps ? p.chosen.steps : p.rejected.steps;
  if (longest <= kShortRow) return 1;
  long long s = (2048 + 2 * p.pairs - 1) / (2 * p.pairs), most = (longest + 4095) / 4096;
  s = s > most ? most : s;
  return (int)(s > kMaxSplits ? kMaxSplits : s < 1 ? 1 : s);
}

bool dense_side(const SdehPreferenceSide& s, int v) {
  return dense(s.log_prob, s.steps, 16) && dense(s.ref_log_prob, s.steps, 16) && dense(s.mask, s.steps, v);
}

void grad_strides(PreferenceArgs& a, long long blocks, int nt, int v) {
  const long long steps[2] = {a.p.chosen.steps, a.p.rejected.steps};
  for (int k = 0; k < 2; ++k) {
    a.d_row[k] = steps[k] > 0 ? blocks * nt * v / steps[k] : 0;
    a.d_col[k] = steps[k] > 0 ? blocks * nt * v % steps[k] : 0;
  }
}

template <typename T>
int launch_spread_t(PreferenceArgs a, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  const SdehPreferenceLoss& p = a.p;
  const bool wide = dense(p.chosen.mask, p.chosen.steps, V) && dense(p.rejected.mask, p.rejected.steps, V) && aligned_to(a.grad[0], 16) &&
                    aligned_to(a.grad[1], 16);
  const long long n = p.pairs * (p.chosen.steps > p.rejected.steps ? p.chosen.steps : p.rejected.steps);
  if (n == 0) return SDEH_OK;
  const int v = wide ? V : 1;
  long long blocks = (n + (long long)kThreads * v - 1) / ((long long)kThreads * v);
  if (blocks > 4096) blocks = 4096;
  grad_strides(a, blocks, kThreads, v);
  if (wide)
    hipLaunchKernelGGL((preference_grad_kernel<T, V>), dim3((unsigned)blocks, 2), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((preference_grad_kernel<T, 1>), dim3((unsigned)blocks, 2), dim3(kThreads), 0, stream, a);
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

template <typename T>
int launch_preference_t(PreferenceArgs a, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  const SdehPreferenceLoss& p = a.p;
  const long long longest = p.chosen.steps > p.rejected.steps ? p.chosen.steps : p.rejected.steps;
  const bool wide = dense_side(p.chosen, V) && dense_side(p.rejected, V);
  if (p.pairs * (p.chosen.steps + p.rejected.steps) <= kPreferenceSmall && longest <= kShortRow && p.pairs <= kSmallThreads) {
    const bool grad_wide = wide && aligned_to(a.grad[0], 16) && aligned_to(a.grad[1], 16);
    grad_strides(a, 1, kSmallThreads, grad_wide ? V : 1);
    if (grad_wide)
      hipLaunchKernelGGL((preference_small_kernel<T, V>), dim3(1), dim3(kSmallThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((preference_small_kernel<T, 1>), dim3(1), dim3(kSmallThreads), 0, stream, a);
    return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
  }
  a.chunk = (longest + a.splits - 1) / a.splits;
  a.chunk = (a.chunk + 15) / 16 * 16;
  if (longest <= kShortRow) {
    const long long blocks = (2 * p.pairs + kThreads / 64 - 1) / (kThreads / 64);
    const dim3 grid((unsigned)(blocks > 8192 ? 8192 : blocks));
    if (wide)
      hipLaunchKernelGGL((preference_short_kernel<T, V>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((preference_short_kernel<T, 1>), grid, dim3(kThreads), 0, stream, a);
  } else {
    launch_pieces(2 * p.pairs * a.splits, [&](long long first, dim3 grid) {
      a.first = first;
      if (wide)
        hipLaunchKernelGGL((preference_sum_kernel<T, V>), grid, dim3(kThreads), 0, stream, a);
      else
        hipLaunchKernelGGL((preference_sum_kernel<T, 1>), grid, dim3(kThreads), 0, stream, a);
    });
  }
  const long long per = a.splits == 1 ? kThreads : kThreads / 64;
  long long pair_blocks = (p.pairs + per - 1) / per;
  a.n_pair_blocks = (int)(pair_blocks > kPairBlocks ? kPairBlocks : pair_blocks);
  hipLaunchKernelGGL(preference_pair_kernel, dim3(a.n_pair_blocks), dim3(kThreads), 0, stream, a);
  if (a.n_pair_blocks > 1 && (a.grad[0] == nullptr || longest == 0)) hipLaunchKernelGGL(preference_final_kernel, dim3(1), dim3(kThreads), 0, stream, a);
  if (hipGetLastError() != hipSuccess) return SDEH_ERR_HIP;
  if (a.grad[0] == nullptr || longest == 0) return SDEH_OK;
  a.slopes = a.out + 2 + 2 * p.pairs;
  return launch_spread_t<T>(a, stream);
}

}  // namespace

// scratch: partial losses, sums, counts
long long preference_scratch_floats(const SdehPreferenceLoss& p) { return kPairBlocks * 4ll + 8ll * p.pairs * preference_splits(p); }

int launch_preference_loss(const SdehPreferenceLoss& p, float* scratch, float grad_factor, float* out, void* grad_c, void* grad_r,
                           hipStream_t stream) {
  PreferenceArgs a{};
  a.p = p;
  a.splits = preference_splits(p);
  a.part = reinterpret_cast<double*>(scratch);
  a.sum = a.part + 2 * kPairBlocks;
  a.count = reinterpret_cast<long long*>(a.sum + 2 * p.pairs * a.splits);
  a.out = out;
  a.grad_factor = grad_factor;
  a.grad[0] = grad_c;
  a.grad[1] = grad_r;
  return p.dtype == SDEH_F32 ? launch_preference_t<float>(a, stream)
                             : p.dtype == SDEH_BF16 ? launch_preference_t<bf16_t>(a, stream) : launch_preference_t<f16_t>(a, stream);
}

int launch_preference_grad(const SdehPreferenceLoss& p, const float* out, const float* grad_scale, float grad_factor, void* grad_c, void* grad_r,
                           hipStream_t stream) {
  PreferenceArgs a{};
  a.p = p;
  a.slopes = out + 2 + 2 * p.pairs;
  a.grad_scale = grad_scale;
  a.grad_factor = grad_factor;
  a.grad[0] = grad_c;
  a.grad[1] = grad_r;
  return p.dtype == SDEH_F32 ? launch_spread_t<float>(a, stream)
                             : p.dtype == SDEH_BF16 ? launch_spread_t<bf16_t>(a, stream) : launch_spread_t<f16_t>(a, stream);
}

}  // namespace sdeh
