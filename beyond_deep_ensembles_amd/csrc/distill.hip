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
// classes are masked out of the row before anything is summed, so Q is a sum of positive terms (no 1 - sum cancellation).  Each
// wave sums its part relative to a number near that part's largest element -- of its first granules, or, where the part rises far
// above those, of all --, so nothing underflows when the student puts nearly everything on the list.
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
  int64_t row0;              // first row of this launch
  int stream_out;            // the gradient is too large to stay in the caches until it is read
  float coef;                // factor of every row's loss
  float inv_tau;
};

constexpr int kDistillMaxK = 1024;
constexpr int kDistillMaxV = 262144;

// NT threads per row: its first NT * NV granules of 16 bytes are kept in registers, what a longer row has
// beyond them is read again (from the caches) for the gradient.
template <typename T, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT * kRowsPerGroup<NT>) void distill_topk_kernel(DistillArgs a) {
  constexpr int GN = Granule<T>::N, W = NT / 64, ROWS = kRowsPerGroup<NT>;
  const int mine = ROWS > 1 ? __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / NT) : 0;
  const int64_t row = a.row0 + static_cast<int64_t>(blockIdx.x) * ROWS + mine;
  if (ROWS > 1 && row >= a.N) return;          // (waves that share a workgroup share nothing else)
  const int tid = static_cast<int>(threadIdx.x) % NT, lane = tid & 63, wave = tid >> 6;
  const int wave_first = __builtin_amdgcn_readfirstlane(tid);       // a wave whose granules all lie behind the row skips them
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
      if (a.stream_out) __builtin_nontemporal_store(granule_pack<T>(f), reinterpret_cast<u32x4*>(g_row + e0));
      else *reinterpret_cast<u32x4*>(g_row + e0) = granule_pack<T>(f);
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
  uint32_t* const bits = lds + mine * (words + 3 * a.K);        // bit shift + v: class v is listed
  float* const t_l = reinterpret_cast<float*>(bits + words);    // [K] the teacher's logit (-inf: entry not used)
  float* const z_l = t_l + a.K;                                 // [K] the student's logit of that class
  int* const v_l = reinterpret_cast<int*>(z_l + a.K);           // [K] the class (-1: entry not used)
  __shared__ float teacher_[ROWS][3], listed_[ROWS][2 * W], others_[ROWS][2 * W];
  __shared__ int dup_[ROWS];
  float *const teacher = teacher_[mine], *const listed = listed_[mine], *const others = others_[mine];
  int& dup = dup_[mine];

  // Loads return in the order they were issued: a thread's own entry of the list goes first and stays raw until the row's loads
  // are out; the student's logit of that class comes last and is not looked at before the row has been summed.
  int64_t raw_v = -1;
  uint32_t raw_t = 0;
  if (tid < a.K) {
    raw_v = a.indices64 ? static_cast<const int64_t*>(a.indices)[row * a.K + tid] : static_cast<const int*>(a.indices)[row * a.K + tid];
    raw_t = a.values_dtype == BDE_F32 ? static_cast<const uint32_t*>(a.values)[row * a.K + tid]
                                      : static_cast<const uint16_t*>(a.values)[row * a.K + tid];
  }
  u32x4 reg[NV];
  if (wave_first < z.granules) reg[0] = z.load(tid);
  for (int i = tid; i < words; i += NT) bits[i] = 0u;
  if (tid == 0) dup = 0;
  row_sync<NT>();                // (also: every wave's first granule is asked for before any wave's second)
#pragma unroll
  for (int j = 1; j < NV; ++j)
    if (wave_first + j * NT < z.granules) reg[j] = z.load(tid + j * NT);
  auto list = [&](int j, int v, float t) {
    v_l[j] = v;
    t_l[j] = v < 0 ? neg_inf() : t;
    if (v >= 0) {
      const uint32_t bit = 1u << ((v + z.shift) & 31);
      if (atomicOr(&bits[(v + z.shift) >> 5], bit) & bit) dup = 1;
    }
  };
  int own_v = -1;
  if (tid < a.K) {
    own_v = raw_v >= 0 && raw_v < a.V ? static_cast<int>(raw_v) : -1;
    list(tid, own_v, a.values_dtype == BDE_F32    ? __uint_as_float(raw_t)
                     : a.values_dtype == BDE_BF16 ? __uint_as_float(raw_t << 16)
                                                  : static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(raw_t))));
  }
  for (int j = tid + NT; j < a.K; j += NT) {
    const int v = load_index(a.indices, a.indices64, row * a.K + j, a.V);
    list(j, v, load_as_float(a.values, a.values_dtype, row * a.K + j));
    z_l[j] = v < 0 ? neg_inf() : static_cast<float>(z.p[v]);
  }
  T own_z = static_cast<T>(neg_inf());
  if (own_v >= 0) own_z = z.p[own_v];
  row_sync<NT>();

  // the listed classes are masked out of the row before it is summed
  auto mask = [&](u32x4& x, int g) {
    const int b = g * GN;
    const uint32_t m = (bits[b >> 5] >> (b & 31)) & ((1u << GN) - 1u);
    if (m) {
#pragma unroll
      for (int i = 0; i < GN; ++i)
        if ((m >> i) & 1u) granule_set<T>(x, i, static_cast<T>(neg_inf()));
    }
  };
  auto largest = [&](const u32x4& x, float m) {
#pragma unroll
    for (int i = 0; i < GN; ++i) m = fmaxf(m, granule_get<T>(x, i));
    return m;
  };
  // exponentials: e^(x / tau) relative to e^(ref / tau) is 2^((x - ref) c); the difference first, so that a reference as large as
  // the type's lowest value (a mask) leaves no residue
  const float c = a.inv_tau * kLog2e;
  const float rest = a.rest ? a.rest[row] : neg_inf();
  if (wave == 0) {               // the teacher's largest exponent (natural units) and its sum relative to it
    float t_top = neg_inf();
    bool bad = rest - rest != 0.0f && rest != neg_inf();          // a NaN or +inf among the teacher's numbers
    for (int j = lane; j < a.K; j += 64) {
      const float t = t_l[j];
      t_top = fmaxf(t_top, t);
      bad = bad || (t - t != 0.0f && t != neg_inf());
    }
    t_top = wave_all_max(t_top);
    bad = __ballot(bad) != 0;
    const float ref = t_top > neg_inf() ? t_top : 0.0f;
    float sum = 0.0f;
    for (int j = lane; j < a.K; j += 64) sum += exp2_hw((t_l[j] - ref) * c);
    sum = wave_all_sum(sum);
    if (lane == 0) {
      // log of the whole, relative to ref: log(sum + e^(rest - ref / tau)), from the larger of the two
      // (a list of the type's lowest value, a mask, may leave the range at a temperature below 1)
      const float gap = rest > neg_inf() ? fminf(rest - ref * a.inv_tau, 3.0e38f) : neg_inf();
      const float own = t_top > neg_inf() ? kLn2 * __builtin_amdgcn_logf(sum) : neg_inf(), hi = fmaxf(own, gap);
      teacher[0] = ref;
      teacher[1] = bad                ? __builtin_nanf("")
                   : hi == neg_inf() ? hi        // the teacher says nothing about this row
                                     : hi + kLn2 * __builtin_amdgcn_logf(exp2_hw((own - hi) * kLog2e) + exp2_hw((gap - hi) * kLog2e));
      teacher[2] = gap;
    }
  }
  // Each wave sums its part of the classes not listed, as the loads arrive, relative to a reference of its own: the largest of
  // its first granules.  Any number near its maximum will do -- unless its part rises far above that, or was masked there: then
  // the maximum itself.
  float ref = neg_inf(), tail = 0.0f;
  auto sum_up = [&](bool masked) {
    const float from = ref > neg_inf() ? ref : 0.0f;
    tail = 0.0f;
    auto add = [&](const u32x4& x) {
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < GN; ++i) part += exp2_hw((granule_get<T>(x, i) - from) * c);
      tail += part;
      settle(tail);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (wave_first + j * NT >= z.granules) continue;
      if (!masked && j > 0 && tid + j * NT < z.granules) mask(reg[j], tid + j * NT);
      stay_packed(reg[j]);
      add(reg[j]);
    }
    for (int g = tid + NV * NT; g < z.granules; g += NT) {
      u32x4 x = z.load(g);
      mask(x, g);
      add(x);
    }
    tail = wave_all_sum(tail);
  };
  if (wave_first < z.granules) {
    if (tid < z.granules) mask(reg[0], tid);
    ref = wave_all_max(largest(reg[0], neg_inf()));
    sum_up(false);
    if (!(tail < 1.0e12f) || ref == neg_inf()) {
      ref = neg_inf();
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (wave_first + j * NT < z.granules) {
          stay_packed(reg[j]);
          ref = largest(reg[j], ref);
        }
      for (int g = tid + NV * NT; g < z.granules; g += NT) {
        u32x4 x = z.load(g);
        mask(x, g);
        ref = largest(x, ref);
      }
      ref = wave_all_max(ref);
      sum_up(true);
    }
  }
  // the student's listed classes, each counted once: a part per wave that has entries
  float l_top = neg_inf(), l_sum = 0.0f;
  if (wave * 64 < a.K) {
    if (tid < a.K) z_l[tid] = static_cast<float>(own_z);
    for (int j = tid; j < a.K; j += NT) l_top = fmaxf(l_top, z_l[j]);
    l_top = wave_all_max(l_top);
    const float l_ref = l_top > neg_inf() ? l_top : 0.0f;
    for (int j = tid; j < a.K; j += NT) {
      bool first = v_l[j] >= 0;
      if (dup)
        for (int i = 0; i < j; ++i) first = first && v_l[i] != v_l[j];
      if (first) l_sum += exp2_hw((z_l[j] - l_ref) * c);
    }
    l_sum = wave_all_sum(l_sum);
    if (W > 1 && lane == 0) {
      listed[2 * wave] = l_top;
      listed[2 * wave + 1] = l_sum;
    }
  }
  if (W > 1 && lane == 0) {
    others[2 * wave] = ref;
    others[2 * wave + 1] = tail;
  }
  row_sync<NT>();

  // every thread: the row's normalisers, from the waves' parts
  auto join = [&](const float* parts, int n, float& top, float& sum) {
    const float m = lane < n ? parts[2 * lane] : neg_inf();
    top = wave_all_max(m);
    sum = wave_all_sum(lane < n && parts[2 * lane + 1] != 0.0f ? parts[2 * lane + 1] * exp2_hw((m - (top > neg_inf() ? top : 0.0f)) * c) : 0.0f);
  };
  const float t_ref = teacher[0], t_log = teacher[1], r_log = teacher[2] - t_log, r = rest > neg_inf() ? exp2_hw(r_log * kLog2e) : 0.0f;
  const bool silent = t_log == neg_inf();
  float other = ref;
  if constexpr (W > 1) {
    join(others, W, other, tail);
    join(listed, min(W, (a.K + 63) >> 6), l_top, l_sum);
  }
  const float top = fmaxf(other, l_top);
  const float o_scale = exp2_hw((other - top) * c);
  const float sum = tail * o_scale + (l_top > neg_inf() ? l_sum * exp2_hw((l_top - top) * c) : 0.0f);
  const float s_log = kLn2 * __builtin_amdgcn_logf(sum);
  const float factor = a.coef * w * (a.inv_weight ? *a.inv_weight : 1.0f);
  auto log_p = [&](int j) { return (t_l[j] - t_ref) * a.inv_tau - t_log; };

  if (a.loss && wave == 2 % W) {
    // p (log p - log q), log q = gap / tau + inner - s_log.  A finite gap of 1e38 (a masked class) over a temperature below 1 may leave the range where
    // the term does not: then p goes in first, and nothing else of the term counts beside it
    auto term = [&](float p, float lp, float gap, float inner) {
      const float x = gap * a.inv_tau;
      return x == neg_inf() && gap > neg_inf() ? -(p * gap) * a.inv_tau : p * (lp - (x + inner - s_log));
    };
    float acc = 0.0f;
    for (int j = lane; j < a.K; j += 64) {
      const float lp = log_p(j), p = exp2_hw(lp * kLog2e);
      if (p != 0.0f) acc += term(p, lp, z_l[j] - top, 0.0f);
    }
    acc = wave_all_sum(acc);
    if (r != 0.0f) acc += term(r, r_log, other - top, kLn2 * __builtin_amdgcn_logf(tail));
    if (lane == 0) a.loss[row] = silent ? 0.0f : factor * acc;
  }
  if constexpr (GRAD) {
    if (silent) {
      store_zeros();
      return;
    }
    const float k = factor * up * a.inv_tau, inv = 1.0f / sum;
    // (no class but the listed ones has any weight: they get 0)
    const float from = ref > neg_inf() ? ref : 0.0f;
    const float f0 = k * (ref > neg_inf() ? exp2_hw((ref - other) * c) : 0.0f) * (o_scale * inv - (r != 0.0f && tail != 0.0f ? r / tail : 0.0f));
    auto put = [&](const u32x4& x, int g) {
      float f[GN];
#pragma unroll
      for (int i = 0; i < GN; ++i) f[i] = f0 * exp2_hw((granule_get<T>(x, i) - from) * c);
      store(g, f);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (wave_first + j * NT >= z.granules) continue;
      stay_packed(reg[j]);
      put(reg[j], tid + j * NT);
    }
    for (int g = tid + NV * NT; g < z.granules; g += NT) put(z.load(g), g);
    // the listed classes, over what was just stored for them (entries of one class all write the same value)
    row_sync<NT>();
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
  for (int64_t i = threadIdx.x; i < n; i += 4096) {       // four loads in flight
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i + 1024 * u < n ? weight[i + 1024 * u] : 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) s += x[u];
  }
  s = block_sum(s, smem);
  if (threadIdx.x == 0) *inv = s != 0.0 ? static_cast<float>(1.0 / s) : 0.0f;
}
// the rows' losses -> one number, in a fixed order
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* loss, int n, float* out) {
  __shared__ double smem[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 4096) {       // four loads in flight
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i + 1024 * u < n ? loss[i + 1024 * u] : 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) s += x[u];
  }
  s = block_sum(s, smem);
  if (threadIdx.x == 0) *out = static_cast<float>(s);
}

// Above this many bytes the gradient is stored past the caches: 2,048 rows of 32,000 / 50,021 / 64,000 bf16 classes 51 / 88 / 104
// us against 57 / 106 / 116 with plain stores; 8,192 x 8,000 the same either way.
constexpr int64_t kStreamBytes = 64 << 20;

template <typename T, int NT, int NV, bool GRAD>
static int distill_launch(DistillArgs a, hipStream_t s) {
  constexpr int ROWS = kRowsPerGroup<NT>;
  const size_t lds = 4 * ROWS * (static_cast<size_t>((a.V + Granule<T>::N + 31) / 32 + 1) + 3 * static_cast<size_t>(a.K));
  for (a.row0 = 0; a.row0 < a.N; a.row0 += kRowsPerLaunch) {
    const int rows = static_cast<int>(std::min<int64_t>(kRowsPerLaunch, a.N - a.row0));
    hipLaunchKernelGGL((distill_topk_kernel<T, NT, NV, GRAD>), dim3((rows + ROWS - 1) / ROWS), dim3(NT * ROWS), lds, s, a);
    if (const int rc = to_err(hipGetLastError())) return rc;
  }
  return 0;
}
// Threads and registers by the granules of a row: four to eight granules a thread (enough loads in flight, several rows per CU
// whose phases overlap) and as few waves as hold the row -- a barrier costs per wave.  bf16, forward with gradient: 32,000 classes
// 53 us with 512 x 8 (76 with 1024 x 4) for 2,048 rows; 64,000 classes 118 us with 512 x 16 (151 with 1024 x 8); 8,000 classes 56 us
// with 256 x 4 (68 with 512 x 2) for 8,192 rows; 131,072 classes 504 us with 1024 x 16, 531 with 512 x 16 and half a row read again.
template <typename T, bool GRAD>
static int distill_pick(DistillArgs a, hipStream_t s) {
  constexpr int GN = Granule<T>::N;
  a.stream_out = static_cast<int64_t>(a.N) * a.V * static_cast<int64_t>(sizeof(T)) > kStreamBytes;
  const bool aligned = aligned16(a.z) && (a.ldz % GN == 0 || a.N == 1);
  const int granules = (a.V + (aligned ? 0 : GN - 1) + GN - 1) / GN;
  if (granules <= 64) return distill_launch<T, 64, 1, GRAD>(a, s);
  if (granules <= 128) return distill_launch<T, 64, 2, GRAD>(a, s);
  if (granules <= 256) return distill_launch<T, 64, 4, GRAD>(a, s);
  if (granules <= 512) return distill_launch<T, 128, 4, GRAD>(a, s);
  if (granules <= 1024) return distill_launch<T, 256, 4, GRAD>(a, s);
  if (granules <= 2048) return distill_launch<T, 512, 4, GRAD>(a, s);
  if (granules <= 4096) return distill_launch<T, 512, 8, GRAD>(a, s);
  if (granules <= 8192) return distill_launch<T, 512, 16, GRAD>(a, s);
  return distill_launch<T, 1024, 16, GRAD>(a, s);
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
