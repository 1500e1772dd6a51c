// One AdamW step over many tensors, moments in 32 or in 8 bits, gradients clipped by their global norm (include/sdeh.h, ABI v8).
//
// With 32-bit moments bounded by memory: fp32 reads and writes 28 bytes an entry (and the gradient's 4 once more for the norm); 150 M entries take
// 0.78 ms (5.4 TB/s; a large elementwise kernel reaches 6.2) after 0.12 ms for the norm.  With 8-bit moments it is 10 bytes of bf16 (and 2) but some 65
// vector instructions an entry -- codes, two hashed roundings, the update --: 100 M entries take 0.21 ms, of which the instructions alone 0.17, and the
// norm 0.04.  Small models are bounded by two launches, 9 us.
//
// Two launches for each 48 tensors: the first forms partial sums of the gradients' squares and the tensors' coefficients (step counters, bias
// corrections), the second adds the partial sums up again in every workgroup -- up to 2048 doubles from L2 -- and updates.  The tensors' pointers travel as
// kernel arguments: no table on the device, nothing to keep or to invalidate.
#include "sdeh_elem.hpp"

namespace sdeh {

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 48;       // of one launch: 48 x 72 bytes of arguments (4 KB are certain)
constexpr int kNormBlocks = 2048;  // partial sums of a step, over all its launches
constexpr int kBlock = SDEH_MOMENT_BLOCK;
constexpr long long kCacheBytes = 256ll << 20;
static_assert(kBlock == 256, "a wave holds a block of moments, four entries a lane");

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* m_top;
  uint8_t* v_top;
  float* step;
  long long n;
  unsigned first_block;
  unsigned chunk_end;  // units of work up to and including this tensor
};

struct Batch {
  Tensor t[kTensors];
  int n, first;     // tensors here; the first one's place among all
  unsigned chunks;  // units of work: `chunk` entries of one tensor, a multiple of four blocks of moments
  int chunk;
};

struct Coef {
  float step_size, inv_root, decay;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr weight_decay
  unsigned key;                      // of the rounding bits: seed and t
};

struct Hyper {
  double lr, beta1, beta2, weight_decay;
  const float* lr_dev;
  const uint8_t* ok;
  unsigned seed;
  Coef* coef;
};

struct Common {
  float beta1, beta2, rest1, rest2, eps;
  double max_norm;
  const uint8_t* ok;
  const double* part;
  int n_part;
  Coef* coef;
  float* norm;
};

__device__ __forceinline__ int find_tensor(const Batch& b, unsigned chunk) {
  int lo = 0, hi = b.n - 1;  // (uniform: scalar loads)
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (chunk < b.t[mid].chunk_end)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// step counters and what follows from them, one thread a tensor
__device__ __forceinline__ void begin_step(const Batch& b, const Hyper& h) {
  const int i = threadIdx.x;
  if (i >= b.n || (h.ok != nullptr && *h.ok == 0)) return;
  const float t = *b.t[i].step + 1.0f;
  *b.t[i].step = t;
  const double lr = h.lr_dev != nullptr ? (double)*h.lr_dev : h.lr;
  Coef c;
  c.step_size = (float)(lr / (1.0 - pow(h.beta1, (double)t)));
  c.inv_root = (float)(1.0 / sqrt(1.0 - pow(h.beta2, (double)t)));
  c.decay = (float)(1.0 - lr * h.weight_decay);
  c.key = h.seed * 0x3C6EF373u + (unsigned)t * 0xBB67AE85u;
  h.coef[b.first + i] = c;
}

__global__ __launch_bounds__(64) void adamw_begin_kernel(Batch b, Hyper h) { begin_step(b, h); }

// partial sums of the gradients' squares, by workgroups 1 ..; workgroup 0 begins the step
template <typename G>
__global__ __launch_bounds__(kThreads) void adamw_norm_kernel(Batch b, Hyper h, double* part) {
  if (blockIdx.x == 0) {
    begin_step(b, h);
    return;
  }
  constexpr int V = 16 / (int)sizeof(G);
  double s = 0.0;
  int k = blockIdx.x - 1 < b.chunks ? find_tensor(b, blockIdx.x - 1) : 0;
  for (unsigned chunk = blockIdx.x - 1; chunk < b.chunks; chunk += gridDim.x - 1) {
    while (chunk >= b.t[k].chunk_end) ++k;  // (from where the last unit was: a search would be six loads in a row)
    const unsigned first = k > 0 ? b.t[k - 1].chunk_end : 0u;
    const long long at = (long long)(chunk - first) * b.chunk;
    const int n = (int)(b.t[k].n - at < b.chunk ? b.t[k].n - at : b.chunk);
    const G* g = static_cast<const G*>(b.t[k].g) + at;
    if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
      const int body = n / V * V;
#pragma unroll 4
      for (int j = V * threadIdx.x; j < body; j += V * kThreads) {
        float x[V];
        unpack<G, V>(load_raw(g + j), x);
#pragma unroll
        for (int e = 0; e < V; ++e) s = fma((double)x[e], (double)x[e], s);
      }
      for (int j = body + threadIdx.x; j < n; j += kThreads) s = fma((double)(float)g[j], (double)(float)g[j], s);
    } else {
      for (int j = threadIdx.x; j < n; j += kThreads) s = fma((double)(float)g[j], (double)(float)g[j], s);
    }
  }
  s = block_sum<kThreads>(s);
  if (threadIdx.x == 0) part[blockIdx.x - 1] = s;
}

// 32 bits that are a function of key and place: an odd multiple of the place, mixed by two rounds of shift, xor and multiplication (constants: 2^32 over
// the golden ratio, and binary digits of the square roots of 2 and 3)
__device__ __forceinline__ unsigned rounding_bits(unsigned x) {  // x = place * 0x9E3779B1 + key
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

template <bool SIGNED>
__device__ __forceinline__ float from_code(unsigned c, int base) {  // base = 8 (top - depth)
  const unsigned mag = SIGNED ? c & 127u : c;
  const unsigned bits = mag == 0u ? 0u : (unsigned)(base + (int)mag) << 20;
  return __uint_as_float(SIGNED ? bits | (c & 128u) << 24 : bits);
}

// The moments' recursions round every product and sum by itself (no fused multiply-add, which the compiler forms unless told not to), so that a
// moment's bits -- and with them the code it is rounded to -- follow from the formula alone.
__device__ __forceinline__ float blend(float keep, float x, float rest, float y) {
#pragma clang fp contract(off)
  return x * keep + y * rest;
}
__device__ __forceinline__ float product(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}

// The hardware's square root and reciprocal (one unit in the last place each) are enough for an update that is lr times smaller than what it is added to.
// Its square root may take a subnormal number for 0, i.e. be off by 2^-63: beside an eps of kPlainRoots or more that is nothing; below, small numbers are
// scaled first.
constexpr float kPlainRoots = 1e-11f;
__device__ __forceinline__ void new_params(float (&p)[4], const float (&m)[4], const float (&v)[4], const Coef& c, float eps) {
  float root[4];
  if (eps >= kPlainRoots) {
#pragma unroll
    for (int e = 0; e < 4; ++e) root[e] = __builtin_amdgcn_sqrtf(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool low = v[e] < 0x1p-96f;
      root[e] = __builtin_amdgcn_sqrtf(low ? v[e] * 0x1p64f : v[e]) * (low ? 0x1p-32f : 1.0f);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) p[e] = fmaf(p[e], c.decay, -c.step_size * (m[e] * __builtin_amdgcn_rcpf(fmaf(root[e], c.inv_root, eps))));
}

// the largest value of a wave, in a scalar register (shifts within rows of 16 lanes, then rows to rows; 0 comes in from outside)
__device__ __forceinline__ unsigned wave_max(unsigned x) {
#define SDEH_MAX_STEP(ctrl)                                                                                   \
  {                                                                                                           \
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);                \
    x = y > x ? y : x;                                                                                        \
  }
  SDEH_MAX_STEP(0x111)  // row_shr:1
  SDEH_MAX_STEP(0x112)
  SDEH_MAX_STEP(0x114)
  SDEH_MAX_STEP(0x118)
  SDEH_MAX_STEP(0x142)  // row_bcast:15
  SDEH_MAX_STEP(0x143)  // row_bcast:31
#undef SDEH_MAX_STEP
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Codes of four moments from q = (bits + random) >> 20: eight bits of exponent, three of mantissa, rounded.
template <bool SIGNED>
__device__ __forceinline__ unsigned to_codes(const unsigned (&q)[4], const float (&x)[4], int top) {
  const int base = 8 * (top - (SIGNED ? 15 : 31));
  unsigned out = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned bits = __float_as_uint(x[e]);
    unsigned c;
    if (SIGNED)
      c = (unsigned)clamp_int((int)q[e] - base, 0, 127);  // (127 cuts a NaN whose payload is all ones)
    else
      c = (bits & 0x7FFFFFFFu) == 0u ? 0u : (unsigned)clamp_int((int)q[e] - base, 1, 255);  // (a second moment above 0 stays above 0: it divides)
    out |= c << (8 * e);
  }
  if (SIGNED) {  // the four top bytes side by side; of each its sign
    const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0C0C0703u);
    const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07030C0Cu);
    out |= (lo | hi) & 0x80808080u;
  }
  return out;
}

// Four neighbouring entries of a lane, a block of 256 of a wave.  STREAM: past the caches (sdeh_elem.hpp).
template <typename T, bool STREAM>
__device__ __forceinline__ void get(const T* __restrict__ p, float (&x)[4]) {
  if constexpr (STREAM)
    stream_in<T, 4>(p, x);
  else
    load_pack<T, 4>(p, x);
}
template <typename T, bool STREAM>
__device__ __forceinline__ void put(T* __restrict__ p, const float (&x)[4]) {
  if constexpr (STREAM)
    stream_out<T, 4>(p, x);
  else
    store_pack<T, 4>(p, x);
}
template <bool STREAM>
__device__ __forceinline__ unsigned get_codes(const uint8_t* p) {
  const unsigned* q = reinterpret_cast<const unsigned*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <bool STREAM>
__device__ __forceinline__ void put_codes(uint8_t* p, unsigned c) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(c, reinterpret_cast<unsigned*>(p));
  else
    *reinterpret_cast<unsigned*>(p) = c;
}

template <typename P, int BITS, bool STREAM>
struct Four {
  float p[4], g[4], m[4], v[4];
  unsigned cm, cv, tm, tv;

  // `live` of the four exist; FAST: all of them, and aligned
  template <bool FAST>
  __device__ __forceinline__ void load(const Tensor& t, long long i, int live) {
    const P* tp = static_cast<const P*>(t.p) + i;
    const P* tg = static_cast<const P*>(t.g) + i;
    if (FAST) {
      get<P, STREAM>(tp, p);
      get<P, STREAM>(tg, g);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = e < live ? (float)tp[e] : 0.0f;
        g[e] = e < live ? (float)tg[e] : 0.0f;
      }
    }
    if constexpr (BITS == 8) {
      const uint8_t* m8 = static_cast<const uint8_t*>(t.m) + i;
      const uint8_t* v8 = static_cast<const uint8_t*>(t.v) + i;
      if (FAST) {
        cm = get_codes<STREAM>(m8);
        cv = get_codes<STREAM>(v8);
      } else {
        cm = cv = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < live) {
            cm |= (unsigned)m8[e] << (8 * e);
            cv |= (unsigned)v8[e] << (8 * e);
          }
        }
      }
      tm = t.m_top[i >> 8];  // (i - 4 lane is a multiple of 256, and i >> 8 the block, in every lane)
      tv = t.v_top[i >> 8];
    } else {
      const float* fm = static_cast<const float*>(t.m) + i;
      const float* fv = static_cast<const float*>(t.v) + i;
      if (FAST) {
        get<float, STREAM>(fm, m);
        get<float, STREAM>(fv, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[e] = e < live ? fm[e] : 0.0f;
          v[e] = e < live ? fv[e] : 0.0f;
        }
      }
    }
  }

  template <bool FAST>
  __device__ __forceinline__ void update(const Tensor& t, const Common& a, const Coef& c, float scale, long long i, int live) {
    if constexpr (BITS == 8) {
      const int bm = 8 * ((int)tm - 15), bv = 8 * ((int)tv - 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = from_code<true>(cm >> (8 * e) & 255u, bm);
        v[e] = from_code<false>(cv >> (8 * e) & 255u, bv);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = product(g[e], scale);  // (scale is 1 without clipping: exact)
      m[e] = blend(a.beta1, m[e], a.rest1, y);
      v[e] = blend(a.beta2, v[e], a.rest2, product(y, y));
    }
    new_params(p, m, v, c, a.eps);
    P* tp = static_cast<P*>(t.p) + i;
    if (FAST) {
      put<P, STREAM>(tp, p);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < live) tp[e] = static_cast<P>(p[e]);
    }
    if constexpr (BITS == 8) {
      unsigned qm[4], qv[4], most_m = 0, most_v = 0;
      const unsigned x = ((t.first_block << 8) + (unsigned)i) * 0x9E3779B1u + c.key;  // (place modulo 2^32)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned r = rounding_bits(x + e * 0x9E3779B1u);
        qm[e] = ((__float_as_uint(m[e]) & 0x7FFFFFFFu) + ((r << 4 & 0xFFFF0u) | 8u)) >> 20;
        qv[e] = ((__float_as_uint(v[e]) & 0x7FFFFFFFu) + ((r >> 12 & 0xFFFF0u) | 8u)) >> 20;
        if (FAST || e < live) {
          most_m = qm[e] > most_m ? qm[e] : most_m;
          most_v = qv[e] > most_v ? qv[e] : most_v;
        }
      }
      const int top_m = clamp_int((int)(wave_max(most_m) >> 3), 16, 255), top_v = clamp_int((int)(wave_max(most_v) >> 3), 32, 255);
      cm = to_codes<true>(qm, m, top_m);
      cv = to_codes<false>(qv, v, top_v);
      uint8_t* m8 = static_cast<uint8_t*>(t.m) + i;
      uint8_t* v8 = static_cast<uint8_t*>(t.v) + i;
      if (FAST) {
        put_codes<STREAM>(m8, cm);
        put_codes<STREAM>(v8, cv);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < live) {
            m8[e] = (uint8_t)(cm >> (8 * e));
            v8[e] = (uint8_t)(cv >> (8 * e));
          }
        }
      }
      if ((threadIdx.x & 63) == 0) {
        t.m_top[i >> 8] = (uint8_t)top_m;
        t.v_top[i >> 8] = (uint8_t)top_v;
      }
    } else {
      float* fm = static_cast<float*>(t.m) + i;
      float* fv = static_cast<float*>(t.v) + i;
      if (FAST) {
        put<float, STREAM>(fm, m);
        put<float, STREAM>(fv, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < live) {
            fm[e] = m[e];
            fv[e] = v[e];
          }
        }
      }
    }
  }
};

template <typename P, int BITS, bool STREAM>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Batch b, Common a) {
  if (a.ok != nullptr && *a.ok == 0) return;
  float scale = 1.0f;
  if (a.max_norm > 0.0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < a.n_part; i += kThreads) s += a.part[i];
    const double norm = sqrt(block_sum<kThreads>(s));
    const double c = a.max_norm / (norm + 1e-6);
    scale = c < 1.0 || c != c ? (float)c : 1.0f;
    if (a.norm != nullptr && b.first == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // (from the last entries to the first: the gradients that the norm read last may still be in the cache)
  int k = blockIdx.x < b.chunks ? find_tensor(b, b.chunks - 1 - blockIdx.x) : 0;
  for (unsigned turn = blockIdx.x; turn < b.chunks; turn += gridDim.x) {
    const unsigned chunk = b.chunks - 1 - turn;
    while (k > 0 && chunk < b.t[k - 1].chunk_end) --k;
    const Tensor& t = b.t[k];
    const unsigned first = k > 0 ? b.t[k - 1].chunk_end : 0u;
    const Coef coef = a.coef[b.first + k];
    const long long at = (long long)(chunk - first) * b.chunk;
    const long long end = t.n - at < b.chunk ? t.n : at + b.chunk;
    const bool wide = (reinterpret_cast<uintptr_t>(t.p) & (4 * sizeof(P) - 1)) == 0 && (reinterpret_cast<uintptr_t>(t.g) & (4 * sizeof(P) - 1)) == 0 &&
                      ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & (BITS == 8 ? 3 : 15)) == 0;
    long long j = at + kBlock * wave;
    if (wide) {
      // four blocks at a time: all their loads are on their way before the first is computed (two at a time: 0.80 ms instead of 0.78 for 150 M fp32 entries
      // with 32-bit moments, 0.23 instead of 0.21 for 100 M of bf16 with 8-bit ones)
      constexpr int U = 4, kStep = kThreads * 4;
      for (; j + (U - 1) * kStep + kBlock <= end; j += U * kStep) {
        Four<P, BITS, STREAM> x[U];
        const long long i = j + 4 * lane;
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].template load<true>(t, i + u * kStep, 4);
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].template update<true>(t, a, coef, scale, i + u * kStep, 4);
      }
    }
    for (; j < end; j += kThreads * 4) {
      Four<P, BITS, STREAM> x;
      const long long i = j + 4 * lane;
      if (wide && j + kBlock <= end) {
        x.template load<true>(t, i, 4);
        x.template update<true>(t, a, coef, scale, i, 4);
      } else {
        const int live = end - i < 0 ? 0 : end - i < 4 ? (int)(end - i) : 4;
        x.template load<false>(t, i, live);
        x.template update<false>(t, a, coef, scale, i, live);
      }
    }
  }
}

// 10 bytes an entry, 8 of them written: 100 M entries in 0.2 ms, 5 TB/s
template <bool STREAM>
__global__ __launch_bounds__(kThreads) void adamw_moments_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ m_top,
                                                                 const uint8_t* __restrict__ v, const uint8_t* __restrict__ v_top, long long n,
                                                                 float* __restrict__ om, float* __restrict__ ov) {
  const long long stride = (long long)gridDim.x * kThreads * 4;
  for (long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += stride) {
    const unsigned km = *reinterpret_cast<const unsigned*>(m + i), kv = *reinterpret_cast<const unsigned*>(v + i);
    const int bm = 8 * ((int)m_top[i / kBlock] - 15), bv = 8 * ((int)v_top[i / kBlock] - 31);
    float xm[4], xv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      xm[e] = from_code<true>(km >> (8 * e) & 255u, bm);
      xv[e] = from_code<false>(kv >> (8 * e) & 255u, bv);
    }
    put<float, STREAM>(om + i, xm);
    put<float, STREAM>(ov + i, xv);
  }
}

template <typename P, int BITS>
void launch_update_b(const Batch& b, const Common& c, bool past_caches, unsigned grid, hipStream_t stream) {
  if (past_caches)
    hipLaunchKernelGGL((adamw_kernel<P, BITS, true>), dim3(grid), dim3(kThreads), 0, stream, b, c);
  else
    hipLaunchKernelGGL((adamw_kernel<P, BITS, false>), dim3(grid), dim3(kThreads), 0, stream, b, c);
}

template <typename P>
void launch_update(const Batch& b, const Common& c, int bits, bool past_caches, unsigned grid, hipStream_t stream) {
  if (bits == 8)
    launch_update_b<P, 8>(b, c, past_caches, grid, stream);
  else
    launch_update_b<P, 32>(b, c, past_caches, grid, stream);
}

}  // namespace

// scratch: partial sums, coefficients
long long adamw_scratch_floats(int n_tensors) { return kNormBlocks * 2ll + 4ll * n_tensors; }

int launch_adamw_step(const SdehAdamw& p, const SdehAdamwGroup* groups, const SdehAdamwTensor* tensors, float* scratch, hipStream_t stream) {
  double* part = reinterpret_cast<double*>(scratch);
  Coef* coef = reinterpret_cast<Coef*>(scratch + kNormBlocks * 2ll);
  int batches = 0, n_part = 0;
  long long entries = 0, bytes = 0;
  for (int k = 0, at = 0; k < p.n_groups; ++k) {
    batches += (groups[k].n_tensors + kTensors - 1) / kTensors;
    const int each = (groups[k].dtype == SDEH_F32 ? 8 : 4) + groups[k].state_bits / 4;
    for (const int end = at + groups[k].n_tensors; at < end; ++at) {
      entries += tensors[at].numel;
      bytes += tensors[at].numel * each;
    }
  }
  if (batches > kNormBlocks) return SDEH_ERR_UNSUPPORTED;
  // small units while there are not enough of them to go round (13 tensors of a 64-channel network: 5.3 us in units of 1024, 7.4 in units of 4096;
  // above 2 M entries a unit's start costs more than the balance gives)
  const int chunk = entries <= 2048ll * 1024 ? 1024 : 8192;
  // what does not fit the 256 MB cache anyway goes past it and leaves it to the gradients, which are read twice (150 M fp32 entries: update 826 -> 790 us,
  // norm 158 -> 118); smaller states stay in it from step to step
  const bool past_caches = bytes > kCacheBytes;
  // pass 0: refuse what does not fit, before anything runs; pass 1: coefficients and norm; pass 2: update
  for (int pass = 0; pass < 3; ++pass) {
    int first = 0, left = batches;
    for (int k = 0; k < p.n_groups; ++k) {
      const SdehAdamwGroup& g = groups[k];
      for (int from = 0; from < g.n_tensors; from += kTensors, --left) {
        Batch b;
        b.first = first + from;
        b.n = g.n_tensors - from < kTensors ? g.n_tensors - from : kTensors;
        long long chunks = 0;
        for (int i = 0; i < b.n; ++i) {
          const SdehAdamwTensor& t = tensors[b.first + i];
          chunks += (t.numel + chunk - 1) / chunk;
          if (chunks > 0x7FFFFFFFll || t.first_block + (t.numel + kBlock - 1) / kBlock > 0xFFFFFFFFll) return SDEH_ERR_UNSUPPORTED;
          b.t[i] = Tensor{t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_top, t.exp_avg_sq_top, t.step, t.numel,
                          (unsigned)t.first_block, (unsigned)chunks};
        }
        b.chunks = (unsigned)chunks;
        b.chunk = chunk;
        if (pass == 1) {
          const Hyper h{g.lr, g.beta1, g.beta2, g.weight_decay, g.lr_dev, p.ok, p.seed, coef};
          if (p.max_norm > 0.0 && chunks > 0) {
            const long long room = (kNormBlocks - n_part) / left;  // (each batch its share of the partial sums)
            const unsigned grid = (unsigned)(chunks < room ? chunks : room);
            if (g.dtype == SDEH_F32)
              hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(grid + 1), dim3(kThreads), 0, stream, b, h, part + n_part);
            else if (g.dtype == SDEH_BF16)
              hipLaunchKernelGGL(adamw_norm_kernel<bf16_t>, dim3(grid + 1), dim3(kThreads), 0, stream, b, h, part + n_part);
            else
              hipLaunchKernelGGL(adamw_norm_kernel<f16_t>, dim3(grid + 1), dim3(kThreads), 0, stream, b, h, part + n_part);
            n_part += (int)grid;
          } else {
            hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(64), 0, stream, b, h);
          }
        } else if (pass == 2) {
          Common c{};
          c.beta1 = (float)g.beta1;
          c.beta2 = (float)g.beta2;
          c.rest1 = (float)(1.0 - g.beta1);
          c.rest2 = (float)(1.0 - g.beta2);
          c.eps = (float)g.eps;
          c.max_norm = p.max_norm;
          c.ok = p.ok;
          c.part = part;
          c.n_part = n_part;
          c.coef = coef;
          c.norm = p.norm;
          const unsigned grid = (unsigned)(chunks < 2048 ? (chunks > 0 ? chunks : 1) : 2048);
          if (g.dtype == SDEH_F32)
            launch_update<float>(b, c, g.state_bits, past_caches, grid, stream);
          else if (g.dtype == SDEH_BF16)
            launch_update<bf16_t>(b, c, g.state_bits, past_caches, grid, stream);
          else
            launch_update<f16_t>(b, c, g.state_bits, past_caches, grid, stream);
        }
      }
      first += g.n_tensors;
    }
  }
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

int launch_adamw_moments(const uint8_t* m, const uint8_t* m_top, const uint8_t* v, const uint8_t* v_top, long long blocks, float* om, float* ov,
                         hipStream_t stream) {
  const long long n = blocks * kBlock, wanted = (n / 4 + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(wanted < 4096 ? wanted : 4096));
  if (n * 8 > kCacheBytes)  // (100 M entries, step and values together: 460 us through the caches, 439 past them)
    hipLaunchKernelGGL(adamw_moments_kernel<true>, grid, dim3(kThreads), 0, stream, m, m_top, v, v_top, n, om, ov);
  else
    hipLaunchKernelGGL(adamw_moments_kernel<false>, grid, dim3(kThreads), 0, stream, m, m_top, v, v_top, n, om, ov);
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

}  // namespace sdeh
