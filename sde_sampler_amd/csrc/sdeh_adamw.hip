// One AdamW step over many tensors, moments in 32 or in 8 bits, gradients clipped by their global norm (include/sdeh.h, ABI v8).
//
// Bounded by memory: fp32 with 32-bit moments reads and writes 28 bytes an entry (and the gradient's 4 once more for the norm), bf16 with 8-bit
// moments 10 (and 2).  Two launches, however many tensors: the first forms partial sums of the gradients' squares and the tensors' coefficients
// (step counters, bias corrections), the second adds the partial sums up again in every workgroup -- 512 doubles from L2 -- and updates.  The
// tensors' pointers travel as kernel arguments, 48 tensors a launch: no table on the device, nothing to keep or to invalidate.
#include "sdeh_elem.hpp"

namespace sdeh {

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 48;       // of one launch: 48 x 64 bytes of arguments (4 KB are certain)
constexpr int kNormBlocks = 512;   // partial sums of a step, over all its launches
constexpr int kBlock = SDEH_MOMENT_BLOCK;
constexpr int kChunk = 4096;       // entries of a unit of work: 16 blocks of 8-bit moments
static_assert(kChunk % kBlock == 0 && kBlock == 256, "a wave holds a block of moments, four entries a lane");

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* m_top;
  uint8_t* v_top;
  long long n;
  unsigned first_block;
  unsigned chunk_end;  // units of work up to and including this tensor
};

struct Batch {
  Tensor t[kTensors];
  int n, first;       // tensors here; the first one's place among all
  unsigned chunks;
};

struct Coef {
  float step_size, inv_root, decay;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr weight_decay
  unsigned key;                      // of the rounding bits: seed and t
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

struct BeginArgs {
  float* step[kTensors];
  int n, first;
  double lr, beta1, beta2, weight_decay;
  const float* lr_dev;
  const uint8_t* ok;
  unsigned seed;
  Coef* coef;
};

// step counters and what follows from them, one thread a tensor
__global__ __launch_bounds__(64) void adamw_begin_kernel(BeginArgs a) {
  const int i = threadIdx.x;
  if (i >= a.n || (a.ok != nullptr && *a.ok == 0)) return;
  const float t = *a.step[i] + 1.0f;
  *a.step[i] = t;
  const double lr = a.lr_dev != nullptr ? (double)*a.lr_dev : a.lr;
  Coef c;
  c.step_size = (float)(lr / (1.0 - pow(a.beta1, (double)t)));
  c.inv_root = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
  c.decay = (float)(1.0 - lr * a.weight_decay);
  c.key = a.seed * 0x3C6EF373u + (unsigned)t * 0xBB67AE85u;
  a.coef[a.first + i] = c;
}

template <typename G>
__global__ __launch_bounds__(kThreads) void adamw_norm_kernel(Batch b, double* part) {
  double s = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < b.chunks; chunk += gridDim.x) {
    const int k = find_tensor(b, chunk);
    const unsigned first = k > 0 ? b.t[k - 1].chunk_end : 0u;
    const long long at = (long long)(chunk - first) * kChunk;
    const int n = (int)(b.t[k].n - at < kChunk ? b.t[k].n - at : kChunk);
    const G* g = static_cast<const G*>(b.t[k].g) + at;
    if (n == kChunk && (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(G) - 1)) == 0) {
#pragma unroll
      for (int j = 0; j < kChunk; j += 4 * kThreads) {
        float x[4];
        load_pack<G, 4>(g + j + 4 * threadIdx.x, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma((double)x[e], (double)x[e], s);
      }
    } else {
      for (int j = threadIdx.x; j < n; j += kThreads) s = fma((double)(float)g[j], (double)(float)g[j], s);
    }
  }
  s = block_sum<kThreads>(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// 32 bits that are a function of key and place: an odd multiple of the place, mixed by two rounds of shift, xor and multiplication (constants: 2^32 over
// the golden ratio, and binary digits of the square roots of 2 and 3)
__device__ __forceinline__ unsigned rounding_bits(unsigned key, unsigned place) {
  unsigned x = place * 0x9E3779B1u + key;
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

__device__ __forceinline__ float new_param(float p, float m, float v, const Coef& c, float eps) {
  const float denom = fmaf(sqrtf(v), c.inv_root, eps);
  return fmaf(p, c.decay, -c.step_size * (m / denom));
}

// One entry block of 8-bit moments per wave: lane l holds entries 4 l .. 4 l + 3 (x, n_live of them).  Returns the four codes and the block's top.
template <bool SIGNED>
__device__ __forceinline__ unsigned to_codes(const unsigned (&q)[4], const float (&x)[4], int top) {
  const int depth = SIGNED ? 15 : 31, base = 8 * (top - depth);
  unsigned out = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    int c = (int)q[e] - base;
    const unsigned bits = __float_as_uint(x[e]);
    if (SIGNED) {
      c = c < 1 ? 0 : c > 127 ? 127 : c;  // (above: a NaN whose payload is all ones)
      c |= (bits >> 24) & 128u;
    } else {
      c = (bits & 0x7FFFFFFFu) == 0u ? 0 : c < 1 ? 1 : c > 255 ? 255 : c;  // (a second moment above 0 stays above 0: it divides)
    }
    out |= (unsigned)c << (8 * e);
  }
  return out;
}

template <typename P, typename G, int BITS>
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
  for (unsigned chunk = blockIdx.x; chunk < b.chunks; chunk += gridDim.x) {
    const int k = find_tensor(b, chunk);
    const Tensor& t = b.t[k];
    const unsigned first = k > 0 ? b.t[k - 1].chunk_end : 0u;
    const Coef coef = a.coef[b.first + k];
    const long long at = (long long)(chunk - first) * kChunk;
    P* p = static_cast<P*>(t.p) + at;
    const G* g = static_cast<const G*>(t.g) + at;
    const int n = (int)(t.n - at < kChunk ? t.n - at : kChunk);
    const bool wide = (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(P) - 1)) == 0 && (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(G) - 1)) == 0 &&
                      (reinterpret_cast<uintptr_t>(t.m) & 15) == 0 && (reinterpret_cast<uintptr_t>(t.v) & 15) == 0;
    for (int j = kBlock * wave; j < n; j += kBlock * (kThreads / 64)) {
      const int i = j + 4 * lane, live = n - i < 0 ? 0 : n - i < 4 ? n - i : 4;
      const bool fast = wide && live == 4;
      float xp[4] = {0.f, 0.f, 0.f, 0.f}, xg[4] = {0.f, 0.f, 0.f, 0.f}, xm[4] = {0.f, 0.f, 0.f, 0.f}, xv[4] = {0.f, 0.f, 0.f, 0.f};
      if (fast) {
        load_pack<P, 4>(p + i, xp);
        load_pack<G, 4>(g + i, xg);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < live) {
            xp[e] = (float)p[i + e];
            xg[e] = (float)g[i + e];
          }
      }
      const long long block = (at + j) / kBlock;
      if constexpr (BITS == 8) {
        const uint8_t* cm = static_cast<const uint8_t*>(t.m) + at + i;
        const uint8_t* cv = static_cast<const uint8_t*>(t.v) + at + i;
        unsigned km = 0, kv = 0;
        if (fast) {
          km = *reinterpret_cast<const unsigned*>(cm);
          kv = *reinterpret_cast<const unsigned*>(cv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < live) {
              km |= (unsigned)cm[e] << (8 * e);
              kv |= (unsigned)cv[e] << (8 * e);
            }
        }
        const int bm = 8 * ((int)t.m_top[block] - 15), bv = 8 * ((int)t.v_top[block] - 31);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          xm[e] = from_code<true>(km >> (8 * e) & 255u, bm);
          xv[e] = from_code<false>(kv >> (8 * e) & 255u, bv);
        }
      } else {
        const float* fm = static_cast<const float*>(t.m) + at + i;
        const float* fv = static_cast<const float*>(t.v) + at + i;
        if (fast) {
          load_pack<float, 4>(fm, xm);
          load_pack<float, 4>(fv, xv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < live) {
              xm[e] = fm[e];
              xv[e] = fv[e];
            }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = a.max_norm > 0.0 ? product(xg[e], scale) : xg[e];
        xm[e] = blend(a.beta1, xm[e], a.rest1, y);
        xv[e] = blend(a.beta2, xv[e], a.rest2, product(y, y));
        xp[e] = new_param(xp[e], xm[e], xv[e], coef, a.eps);
      }
      if (fast) {
        store_pack<P, 4>(p + i, xp);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < live) p[i + e] = static_cast<P>(xp[e]);
      }
      if constexpr (BITS == 8) {
        unsigned qm[4], qv[4], most_m = 0, most_v = 0;
        const unsigned place = (t.first_block + (unsigned)block) * (unsigned)kBlock + 4u * lane;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned r = rounding_bits(coef.key, place + e);
          qm[e] = ((__float_as_uint(xm[e]) & 0x7FFFFFFFu) + ((r & 0xFFFFu) << 4) + 8u) >> 20;
          qv[e] = ((__float_as_uint(xv[e]) & 0x7FFFFFFFu) + ((r >> 16) << 4) + 8u) >> 20;
          if (e < live) {
            most_m = qm[e] > most_m ? qm[e] : most_m;
            most_v = qv[e] > most_v ? qv[e] : most_v;
          }
        }
        // (both maxima in one word: 16 bits hold eight bits of exponent)
        unsigned most = (most_m >> 3) << 16 | (most_v >> 3);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const unsigned other = __shfl_xor(most, o, 64);
          const unsigned h = other >> 16 > most >> 16 ? other & 0xFFFF0000u : most & 0xFFFF0000u;
          const unsigned l = (other & 0xFFFFu) > (most & 0xFFFFu) ? other & 0xFFFFu : most & 0xFFFFu;
          most = h | l;
        }
        int top_m = (int)(most >> 16), top_v = (int)(most & 0xFFFFu);
        top_m = top_m < 16 ? 16 : top_m > 255 ? 255 : top_m;
        top_v = top_v < 32 ? 32 : top_v > 255 ? 255 : top_v;
        const unsigned km = to_codes<true>(qm, xm, top_m), kv = to_codes<false>(qv, xv, top_v);
        uint8_t* cm = static_cast<uint8_t*>(t.m) + at + i;
        uint8_t* cv = static_cast<uint8_t*>(t.v) + at + i;
        if (fast) {
          *reinterpret_cast<unsigned*>(cm) = km;
          *reinterpret_cast<unsigned*>(cv) = kv;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < live) {
              cm[e] = (uint8_t)(km >> (8 * e));
              cv[e] = (uint8_t)(kv >> (8 * e));
            }
        }
        if (lane == 0) {
          t.m_top[block] = (uint8_t)top_m;
          t.v_top[block] = (uint8_t)top_v;
        }
      } else {
        float* fm = static_cast<float*>(t.m) + at + i;
        float* fv = static_cast<float*>(t.v) + at + i;
        if (fast) {
          store_pack<float, 4>(fm, xm);
          store_pack<float, 4>(fv, xv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < live) {
              fm[e] = xm[e];
              fv[e] = xv[e];
            }
        }
      }
    }
  }
}

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
    store_pack<float, 4>(om + i, xm);
    store_pack<float, 4>(ov + i, xv);
  }
}

template <typename P, typename G>
void launch_update(const Batch& b, const Common& c, int bits, unsigned grid, hipStream_t stream) {
  if (bits == 8)
    hipLaunchKernelGGL((adamw_kernel<P, G, 8>), dim3(grid), dim3(kThreads), 0, stream, b, c);
  else
    hipLaunchKernelGGL((adamw_kernel<P, G, 32>), dim3(grid), dim3(kThreads), 0, stream, b, c);
}

template <typename P>
void launch_update_g(const Batch& b, const Common& c, int grad_dtype, int bits, unsigned grid, hipStream_t stream) {
  if (grad_dtype == SDEH_F32)
    launch_update<P, float>(b, c, bits, grid, stream);
  else if (grad_dtype == SDEH_BF16)
    launch_update<P, bf16_t>(b, c, bits, grid, stream);
  else
    launch_update<P, f16_t>(b, c, bits, grid, stream);
}

}  // namespace

// scratch: partial sums, coefficients
long long adamw_scratch_floats(int n_tensors) { return kNormBlocks * 2ll + 4ll * n_tensors; }

int launch_adamw_step(const SdehAdamw& p, const SdehAdamwGroup* groups, const SdehAdamwTensor* tensors, float* scratch, hipStream_t stream) {
  double* part = reinterpret_cast<double*>(scratch);
  Coef* coef = reinterpret_cast<Coef*>(scratch + kNormBlocks * 2ll);
  int batches = 0, n_part = 0;
  for (int k = 0; k < p.n_groups; ++k) batches += (groups[k].n_tensors + kTensors - 1) / kTensors;
  if (batches > kNormBlocks) return SDEH_ERR_UNSUPPORTED;
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
          chunks += (t.numel + kChunk - 1) / kChunk;
          if (chunks > 0x7FFFFFFFll || t.first_block + (t.numel + kBlock - 1) / kBlock > 0xFFFFFFFFll) return SDEH_ERR_UNSUPPORTED;
          b.t[i] = Tensor{t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_top, t.exp_avg_sq_top, t.numel, (unsigned)t.first_block, (unsigned)chunks};
        }
        b.chunks = (unsigned)chunks;
        if (pass == 1) {
          BeginArgs begin{};
          for (int i = 0; i < b.n; ++i) begin.step[i] = tensors[b.first + i].step;
          begin.n = b.n;
          begin.first = b.first;
          begin.lr = g.lr;
          begin.beta1 = g.beta1;
          begin.beta2 = g.beta2;
          begin.weight_decay = g.weight_decay;
          begin.lr_dev = g.lr_dev;
          begin.ok = p.ok;
          begin.seed = p.seed;
          begin.coef = coef;
          hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(64), 0, stream, begin);
          if (p.max_norm > 0.0 && chunks > 0) {
            const long long room = (kNormBlocks - n_part) / left;  // (each batch its share of the partial sums)
            const unsigned grid = (unsigned)(chunks < room ? chunks : room);
            if (g.grad_dtype == SDEH_F32)
              hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(grid), dim3(kThreads), 0, stream, b, part + n_part);
            else if (g.grad_dtype == SDEH_BF16)
              hipLaunchKernelGGL(adamw_norm_kernel<bf16_t>, dim3(grid), dim3(kThreads), 0, stream, b, part + n_part);
            else
              hipLaunchKernelGGL(adamw_norm_kernel<f16_t>, dim3(grid), dim3(kThreads), 0, stream, b, part + n_part);
            n_part += (int)grid;
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
            launch_update_g<float>(b, c, g.grad_dtype, g.state_bits, grid, stream);
          else if (g.dtype == SDEH_BF16)
            launch_update_g<bf16_t>(b, c, g.grad_dtype, g.state_bits, grid, stream);
          else
            launch_update_g<f16_t>(b, c, g.grad_dtype, g.state_bits, grid, stream);
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
  hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)(wanted < 4096 ? wanted : 4096)), dim3(kThreads), 0, stream, m, m_top, v, v_top, n, om, ov);
  return hipGetLastError() == hipSuccess ? SDEH_OK : SDEH_ERR_HIP;
}

}  // namespace sdeh
