// Distillation from a teacher's top logits: the loss and its gradient with respect to the student's logits.
//
// Per row, with student logits z [V], teacher entries (t_j, v_j), j < K, J = {v_j}, temperature tau, and the teacher's
// remaining mass given as rest = log sum_{v not in J} exp(teacher_v / tau):
//   L = log(sum_j exp(t_j / tau) + exp(rest)),   p_j = exp(t_j / tau - L),   r = exp(rest - L)
//   q = softmax(z / tau),                        Q = sum_{v not in J} q_v
//   loss = sum_j p_j (log p_j - log q_{v_j}) + r (log r - log Q)
//   d loss / d z_v = (1 / tau) * { q_v - sum_{j: v_j = v} p_j   for v in J
//                                { q_v - r q_v / Q              otherwise
// i.e. the KL divergence between two distributions over K + 1 outcomes, the last one being "any other class".
//
// Numerics: everything fp32; the row is held in its own type and each gradient is rounded to that type once.  The listed
// classes are masked out of the row before anything is summed, so Q is a sum of positive terms relative to the largest of
// ITS terms (no 1 - sum cancellation, no underflow when the student puts nearly everything on the list).
#include "token_common.hpp"

namespace bde {

struct DistillArgs {
  const void* z;
  int64_t ldz;
  const void* values;
  int values_dtype;
  const void* indices;
  int indices64;
  const float* rest;         // [N] or NULL: r = 0
  const float* weight;       // [N] or NULL: 1
  const float* inv_weight;   // one float on the device (1 / sum of the weights) or NULL: 1
  const float* upstream;     // GRAD: d objective / d loss_i, or NULL: 1
  int64_t upstream_stride;   // 0: one value for all rows
  int skip_if_one;           // GRAD: rows whose upstream value is exactly 1 are left as they are
  float* loss;               // [N] or NULL
  void* grad;                // [N, ldg]
  int64_t ldg;
  int N, V, K;
  float coef;                // factor of every row's loss
  float inv_tau;
};

constexpr int kDistillMaxK = 1024;
constexpr int kDistillMaxV = 262144;

// One workgroup of NT threads per row, the row in registers (NV granules of 16 bytes per thread; NV = 0: rows that do not
// fit, read again from the caches by each phase).
template <typename T, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT) void distill_topk_kernel(DistillArgs a) {
  constexpr int GN = Granule<T>::N, W = NT / 64;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float w = a.weight ? a.weight[row] : 1.0f;
  float up = 1.0f;
  if (GRAD && a.upstream) {
    up = a.upstream[row * a.upstream_stride];
    if (a.skip_if_one && up == 1.0f) return;
  }
  const RowView<T> z(static_cast<const T*>(a.z) + row * a.ldz, a.V);
  T* const g_row = GRAD ? static_cast<T*>(a.grad) + row * a.ldg : nullptr;
  const bool same_shift = GRAD && RowView<T>(g_row, a.V).shift == z.shift;
  // one granule of the gradient row; element by element at the ends, and everywhere when the two rows start at different
  // places of their 16 bytes
  auto store = [&](int g, const float* f) {
    if (g >= z.granules) return;
    const int e0 = z.first(g);
    if (same_shift && z.whole(g)) {
      *reinterpret_cast<u32x4*>(g_row + e0) = granule_pack<T>(f);
    } else {
#pragma unroll
      for (int i = 0; i < GN; ++i)
        if (e0 + i >= 0 && e0 + i < a.V) g_row[e0 + i] = static_cast<T>(f[i]);
    }
  };
  auto store_zeros = [&]() {
    float f[GN];
#pragma unroll
    for (int i = 0; i < GN; ++i) f[i] = 0.0f;
    for (int g = tid; g < z.granules; g += NT) store(g, f);
  };
  // a row that nobody asks for (weight or upstream value 0): loss 0 and gradient 0 whatever its logits hold, nothing read
  if (w == 0.0f || up == 0.0f) {
    if (a.loss && tid == 0) a.loss[row] = 0.0f;
    if constexpr (GRAD) store_zeros();
    return;
  }

  extern __shared__ uint32_t lds[];
  const int words = (a.V + GN + 31) / 32 + 1;
  uint32_t* const bits = lds;                                   // bit shift + v: class v is listed
  float* const t_l = reinterpret_cast<float*>(lds + words);     // [K] the teacher's logit (-inf: entry not used)
  float* const z_l = t_l + a.K;                                 // [K] the student's logit of that class
  int* const v_l = reinterpret_cast<int*>(z_l + a.K);           // [K] the class (-1: entry not used)
  __shared__ float slots[2 * W];
  __shared__ float teacher[3], listed[2];
  __shared__ int dup;

  u32x4 reg[NV > 0 ? NV : 1];
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) reg[j] = z.load(tid + j * NT);
  }
  for (int i = tid; i < words; i += NT) bits[i] = 0u;
  if (tid == 0) dup = 0;
  __syncthreads();
  for (int j = tid; j < a.K; j += NT) {
    const int v = load_index(a.indices, a.indices64, row * a.K + j, a.V);
    v_l[j] = v;
    t_l[j] = v < 0 ? neg_inf() : load_as_float(a.values, a.values_dtype, row * a.K + j);
    z_l[j] = v < 0 ? neg_inf() : static_cast<float>(z.p[v]);
    if (v >= 0) {
      const uint32_t bit = 1u << ((v + z.shift) & 31);
      if (atomicOr(&bits[(v + z.shift) >> 5], bit) & bit) dup = 1;
    }
  }
  __syncthreads();

  // mask the listed classes out of the row; the largest of the others
  auto mask = [&](u32x4& x, int g) {
    const int b = g * GN;
    const uint32_t m = (bits[b >> 5] >> (b & 31)) & ((1u << GN) - 1u);
    if (m) {
#pragma unroll
      for (int i = 0; i < GN; ++i)
        if ((m >> i) & 1u) granule_set<T>(x, i, static_cast<T>(neg_inf()));
    }
  };
  float other = neg_inf();
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (tid + j * NT < z.granules) mask(reg[j], tid + j * NT);
#pragma unroll
      for (int i = 0; i < GN; ++i) other = fmaxf(other, granule_get<T>(reg[j], i));
    }
  } else {
    for (int g = tid; g < z.granules; g += NT) {
      u32x4 x = z.load(g);
      mask(x, g);
#pragma unroll
      for (int i = 0; i < GN; ++i) other = fmaxf(other, granule_get<T>(x, i));
    }
  }
  // exponentials: e^(x / tau) relative to e^(ref / tau) is 2^((x - ref) c); the difference first, so that a reference as large as
  // the type's lowest value (a mask) leaves no residue
  const float c = a.inv_tau * kLog2e;
  const float rest = a.rest ? a.rest[row] : neg_inf();
  if (wave == 0) {               // the teacher's largest exponent (natural units) and its sum relative to it
    float t_top = neg_inf(), bad = rest == neg_inf() ? 0.0f : rest - rest;    // NaN: a NaN or +inf among the teacher's numbers
    for (int j = lane; j < a.K; j += 64) {
      const float t = t_l[j];
      t_top = fmaxf(t_top, t);
      if (t != neg_inf()) bad += t - t;
    }
    t_top = wave_all_max(t_top);
    bad = wave_all_sum(bad);
    const float ref = t_top > neg_inf() ? t_top : 0.0f;
    float sum = 0.0f;
    for (int j = lane; j < a.K; j += 64) sum += exp2_hw((t_l[j] - ref) * c);
    sum = wave_all_sum(sum);
    if (lane == 0) {
      // log of the whole, relative to ref: log(sum + e^(rest - ref / tau)), from the larger of the two
      const float gap = rest - ref * a.inv_tau;
      const float own = t_top > neg_inf() ? kLn2 * __builtin_amdgcn_logf(sum) : neg_inf(), hi = fmaxf(own, gap);
      teacher[0] = ref;
      teacher[1] = bad != 0.0f ? __builtin_nanf("")
                   : hi == neg_inf() ? hi        // the teacher says nothing about this row
                                     : hi + kLn2 * __builtin_amdgcn_logf(exp2_hw((own - hi) * kLog2e) + exp2_hw((gap - hi) * kLog2e));
      teacher[2] = gap;
    }
  }
  if (wave == 1 % W) {           // the student's listed classes, each counted once
    float l_top = neg_inf();
    for (int j = lane; j < a.K; j += 64) l_top = fmaxf(l_top, z_l[j]);
    l_top = wave_all_max(l_top);
    const float ref = l_top > neg_inf() ? l_top : 0.0f;
    float sum = 0.0f;
    for (int j = lane; j < a.K; j += 64) {
      bool first = v_l[j] >= 0;
      if (dup)
        for (int i = 0; i < j; ++i) first = first && v_l[i] != v_l[j];
      if (first) sum += exp2_hw((z_l[j] - ref) * c);
    }
    sum = wave_all_sum(sum);
    if (lane == 0) {
      listed[0] = l_top;
      listed[1] = sum;
    }
  }
  other = block_all_max<NT>(other, slots);
  const float ref = other > neg_inf() ? other : 0.0f;
  float tail = 0.0f;             // sum over the classes not listed, relative to the largest of them
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float part = 0.0f;
      stay_packed(reg[j]);
#pragma unroll
      for (int i = 0; i < GN; ++i) part += exp2_hw((granule_get<T>(reg[j], i) - ref) * c);
      tail += part;
    }
  } else {
    for (int g = tid; g < z.granules; g += NT) {
      u32x4 x = z.load(g);
      mask(x, g);
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < GN; ++i) part += exp2_hw((granule_get<T>(x, i) - ref) * c);
      tail += part;
    }
  }
  tail = block_all_sum<NT>(tail, slots + W);

  // every thread: the row's normalisers
  const float t_ref = teacher[0], t_log = teacher[1], r_log = teacher[2] - t_log, r = rest > neg_inf() ? exp2_hw(r_log * kLog2e) : 0.0f;
  const bool silent = t_log == neg_inf();
  const float l_top = listed[0], top = fmaxf(other, l_top);
  const float o_scale = exp2_hw((other - top) * c), l_scale = l_top > neg_inf() ? exp2_hw((l_top - top) * c) : 0.0f;
  const float sum = tail * o_scale + listed[1] * l_scale;
  const float s_log = kLn2 * __builtin_amdgcn_logf(sum);
  const float factor = a.coef * w * (a.inv_weight ? *a.inv_weight : 1.0f);
  auto log_p = [&](int j) { return (t_l[j] - t_ref) * a.inv_tau - t_log; };

  if (a.loss && wave == 2 % W) {
    float acc = 0.0f;
    for (int j = lane; j < a.K; j += 64) {
      const float lp = log_p(j), p = exp2_hw(lp * kLog2e);
      if (p != 0.0f) acc += p * (lp - ((z_l[j] - top) * a.inv_tau - s_log));
    }
    acc = wave_all_sum(acc);
    if (r != 0.0f) acc += r * (r_log - ((other - top) * a.inv_tau + kLn2 * __builtin_amdgcn_logf(tail) - s_log));
    if (lane == 0) a.loss[row] = silent ? 0.0f : factor * acc;
  }
  if constexpr (GRAD) {
    if (silent) {
      store_zeros();
      return;
    }
    const float k = factor * up * a.inv_tau, inv = 1.0f / sum;
    // (no class but the listed ones has any weight: they get 0)
    const float f0 = k * (o_scale * inv - (r != 0.0f && tail != 0.0f ? r / tail : 0.0f));
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[GN];
        stay_packed(reg[j]);
#pragma unroll
        for (int i = 0; i < GN; ++i) f[i] = f0 * exp2_hw((granule_get<T>(reg[j], i) - ref) * c);
        store(tid + j * NT, f);
      }
    } else {
      for (int g = tid; g < z.granules; g += NT) {
        const u32x4 x = z.load(g);
        float f[GN];
#pragma unroll
        for (int i = 0; i < GN; ++i) f[i] = f0 * exp2_hw((granule_get<T>(x, i) - ref) * c);
        store(g, f);
      }
    }
    // the listed classes, over what was just stored for them (entries of one class all write the same value)
    __syncthreads();
    for (int j = tid; j < a.K; j += NT) {
      const int v = v_l[j];
      if (v < 0) continue;
      float p = exp2_hw(log_p(j) * kLog2e);
      if (dup) {
        p = 0.0f;
        for (int i = 0; i < a.K; ++i)
          if (v_l[i] == v) p += exp2_hw(log_p(i) * kLog2e);
      }
      g_row[v] = static_cast<T>(k * (exp2_hw((z_l[j] - top) * c) * inv - p));
    }
  }
}

// 1 / sum of the rows' weights (0 when the sum is 0), in a fixed order
__global__ __launch_bounds__(1024) void distill_inv_weight_kernel(const float* weight, int n, float* inv) {
  __shared__ double smem[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += weight[i];
  s = block_sum(s, smem);
  if (threadIdx.x == 0) *inv = s != 0.0 ? static_cast<float>(1.0 / s) : 0.0f;
}
// the rows' losses -> one number, in a fixed order
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* loss, int n, float* out) {
  __shared__ double smem[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += loss[i];
  s = block_sum(s, smem);
  if (threadIdx.x == 0) *out = static_cast<float>(s);
}

template <typename T, int NT, int NV, bool GRAD>
static int distill_launch(const DistillArgs& a, hipStream_t s) {
  const size_t lds = 4 * (static_cast<size_t>((a.V + Granule<T>::N + 31) / 32 + 1) + 3 * static_cast<size_t>(a.K));
  hipLaunchKernelGGL((distill_topk_kernel<T, NT, NV, GRAD>), dim3(a.N), dim3(NT), lds, s, a);
  return to_err(hipGetLastError());
}
// Workgroup and registers by the granules of a row: the smallest workgroup that holds it (fewer barriers between waves),
// four granules a thread before more waves than 16.
template <typename T, bool GRAD>
static int distill_pick(const DistillArgs& a, hipStream_t s) {
  constexpr int GN = Granule<T>::N;
  const bool aligned = aligned16(a.z) && (a.ldz % GN == 0 || a.N == 1);
  const int granules = (a.V + (aligned ? 0 : GN - 1) + GN - 1) / GN;
  if (granules <= 64) return distill_launch<T, 64, 1, GRAD>(a, s);
  if (granules <= 256) return distill_launch<T, 256, 1, GRAD>(a, s);
  if (granules <= 1024) return distill_launch<T, 256, 4, GRAD>(a, s);
  if (granules <= 4096) return distill_launch<T, 1024, 4, GRAD>(a, s);
  if (granules <= 8192) return distill_launch<T, 1024, 8, GRAD>(a, s);
  if (granules <= 16384) return distill_launch<T, 1024, 16, GRAD>(a, s);
  return distill_launch<T, 1024, 0, GRAD>(a, s);
}
template <bool GRAD>
static int distill_dispatch(const DistillArgs& a, int dtype, hipStream_t s) {
  if (dtype == BDE_F32) return distill_pick<float, GRAD>(a, s);
  if (dtype == BDE_BF16) return distill_pick<bf16_t, GRAD>(a, s);
  return distill_pick<f16_t, GRAD>(a, s);
}

static bool distill_args_ok(const DistillArgs& a, int dtype) {
  if (!dtype_ok(dtype) || !dtype_ok(a.values_dtype) || a.N < 0 || a.V < 1 || a.V > kDistillMaxV || a.K < 1 || a.K > kDistillMaxK)
    return false;
  if (!(a.inv_tau > 0.0f) || !(a.inv_tau < __builtin_inff()) || a.ldz < a.V) return false;
  if (a.N > 0 && (!a.z || !a.values || !a.indices)) return false;
  return reinterpret_cast<uintptr_t>(a.z) % dtype_bytes(dtype) == 0;
}

}  // namespace bde

using namespace bde;

extern "C" int bde_distill_limits(int* max_classes, int* max_entries) {
  if (max_classes) *max_classes = kDistillMaxV;
  if (max_entries) *max_entries = kDistillMaxK;
  return 0;
}

extern "C" int bde_distill_fwd(const void* logits, int dtype, int64_t ldz, const void* values, int values_dtype,
                               const void* indices, int indices64, const float* rest, const float* weight, int reduction,
                               float scale, float temperature, int N, int V, int K, float* loss_rows, float* loss, void* grad,
                               float* inv_weight, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  DistillArgs a{};
  a.z = logits; a.ldz = ldz; a.values = values; a.values_dtype = values_dtype; a.indices = indices; a.indices64 = indices64;
  a.rest = rest; a.weight = weight; a.loss = loss_rows; a.grad = grad; a.ldg = V; a.N = N; a.V = V; a.K = K;
  a.coef = scale; a.inv_tau = 1.0f / temperature;
  if (!(temperature > 0.0f) || !distill_args_ok(a, dtype) || reduction < 0 || reduction > 2) return BDE_ERR_INVALID;
  if ((N > 0 && !loss_rows) || (reduction != 0 && !loss) || (reduction == 2 && weight && !inv_weight)) return BDE_ERR_INVALID;
  if (reduction == 2) {
    if (weight) {
      a.inv_weight = inv_weight;
      hipLaunchKernelGGL(distill_inv_weight_kernel, dim3(1), dim3(1024), 0, s, weight, N, inv_weight);
      if (const int rc = to_err(hipGetLastError())) return rc;
    } else if (N > 0) {
      a.coef = static_cast<float>(static_cast<double>(scale) / N);
    }
  }
  if (N > 0) {
    const int rc = grad ? distill_dispatch<true>(a, dtype, s) : distill_dispatch<false>(a, dtype, s);
    if (rc) return rc;
  }
  if (reduction != 0) {
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, s, static_cast<const float*>(loss_rows), N, loss);
    return to_err(hipGetLastError());
  }
  return 0;
}

extern "C" int bde_distill_bwd(const void* logits, int dtype, int64_t ldz, const void* values, int values_dtype,
                               const void* indices, int indices64, const float* rest, const float* weight,
                               const float* inv_weight, int mean, float scale, float temperature, const float* upstream,
                               int64_t upstream_stride, int skip_if_one, int N, int V, int K, void* grad, void* stream) {
  DistillArgs a{};
  a.z = logits; a.ldz = ldz; a.values = values; a.values_dtype = values_dtype; a.indices = indices; a.indices64 = indices64;
  a.rest = rest; a.weight = weight; a.upstream = upstream; a.upstream_stride = upstream_stride; a.skip_if_one = skip_if_one;
  a.grad = grad; a.ldg = V; a.N = N; a.V = V; a.K = K; a.coef = scale; a.inv_tau = 1.0f / temperature;
  if (!(temperature > 0.0f) || !distill_args_ok(a, dtype) || (N > 0 && (!grad || !upstream)) || (upstream_stride != 0 && upstream_stride != 1) ||
      (mean && weight && !inv_weight))
    return BDE_ERR_INVALID;
  if (N == 0) return 0;
  if (mean) {
    if (weight) a.inv_weight = inv_weight;
    else a.coef = static_cast<float>(static_cast<double>(scale) / N);
  }
  return distill_dispatch<true>(a, dtype, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("hidden"))) int bde_internal_load_distill(void) {
  hipFuncAttributes attr;
  return to_err(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&distill_sum_kernel)));
}
