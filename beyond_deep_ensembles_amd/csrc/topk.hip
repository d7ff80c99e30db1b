// A teacher's top logits: per row of logits z [V] the k largest values in falling order with their classes, and what the
// other classes weigh together,
//   rest = log sum_{v not selected} exp(z_v / tau),
// which is all a distillation loss needs of the row (distill.hip).
//
// Selection is exact: elements are ordered by (value, lower class first), -0 equals +0, a NaN is larger than every number.
// One pass over the row in registers finds each thread's largest element; the k-th largest of those is a lower bound of the
// row's k-th largest element, so the elements not below it are candidates -- about k of them in a row without structure.
// They are compacted into LDS and ranked by counting (pairs of a 64-bit key, all different).  Rows that leave more candidates
// than the LDS list holds (long runs of equal values) refine the bound by bisection, first over the value, then over the class,
// until exactly k are left.  Nothing depends on the order in which candidates arrive in the list.
#include "token_common.hpp"

namespace bde {

struct TopkArgs {
  const void* z;
  int64_t ldz;
  void* values;       // [N, K], the logits' type
  int64_t* indices;   // [N, K]
  float* rest;        // [N] or NULL
  int N, V, K;
  float inv_tau;
  int64_t row0;       // first row of this launch
};

constexpr int kTopkMaxK = 256;
constexpr int kTopkMaxV = 262144;

// whole numbers in the order of the floats: -0 as +0, every NaN above +inf
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if (x != x) return 0xFFFFFFFFu;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

constexpr uint32_t kKeyNegInf = 0x007FFFFFu;      // order_key(-inf): the smallest
// an entry of the candidate list: larger first, the lower class ahead among equals; no two are the same
__device__ __forceinline__ uint64_t candidate(uint32_t key, int v) {
  return (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(~v);
}

template <int NT>
__device__ __forceinline__ int row_count(int n, int* slots) {
  constexpr int W = NT / 64;
  n = static_cast<int>(wave_all_sum(static_cast<float>(n)));      // <= 2^24: exact
  row_sync<NT>();                                                 // the slots' last readers are done
  if constexpr (W == 1) return n;
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = n;
  row_sync<NT>();
  int r = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) r += slots[i];
  return r;
}

// One wave: a key that at least k of the 64 * M keys reach (k <= 64 * M) and, unless they are equal, not many more -- bisection over
// the keys, counts by ballot.
template <int M>
__device__ __forceinline__ uint32_t reach_of(const uint32_t* keys, int k) {
  uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    low = min(low, keys[i]);
    high = max(high, keys[i]);
  }
  // ends of the range over the wave: the upper 16 bits are exact as floats
  uint32_t lo = static_cast<uint32_t>(-wave_all_max(-static_cast<float>(low >> 16))) << 16;
  uint32_t hi = (static_cast<uint32_t>(wave_all_max(static_cast<float>(high >> 16))) << 16) | 0xFFFFu;
  while (lo < hi) {            // invariant: count(>= lo) >= k, count(> hi) < k
    const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
    int n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) n += __popcll(__ballot(keys[i] >= mid));
    if (n >= k) {
      lo = mid;
      if (n <= k + (k >> 2) + 4) break;
    } else {
      hi = mid - 1u;
    }
  }
  return lo;
}

// NT threads per row: its first NT * NV granules of 16 bytes are kept in registers, what a longer row has
// beyond them is read again (from the caches) by the second pass.
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT * kRowsPerGroup<NT>) void topk_logits_kernel(TopkArgs a) {
  constexpr int GN = Granule<T>::N, W = NT / 64, ROWS = kRowsPerGroup<NT>;
  constexpr int kCap = NT == 64 ? 64 + 64 * NV : 1024;      // entries of the candidate list
  const int row_of_group = ROWS > 1 ? __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / NT) : 0;
  const int64_t row = a.row0 + static_cast<int64_t>(blockIdx.x) * ROWS + row_of_group;
  if (ROWS > 1 && row >= a.N) return;                // (waves that share a workgroup share nothing else)
  const int tid = static_cast<int>(threadIdx.x) % NT, lane = tid & 63;
  const int wave_first = __builtin_amdgcn_readfirstlane(tid);       // a wave whose granules all lie behind the row skips them
  const RowView<T> z(static_cast<const T*>(a.z) + row * a.ldz, a.V);
  __shared__ uint64_t cand_[ROWS][kCap];
  __shared__ int hits_[ROWS][kCap];
  __shared__ uint32_t maxima_[ROWS][W > 1 ? NT : 1];
  __shared__ float slots_[ROWS][2 * W];
  __shared__ int counts_[ROWS][W];
  __shared__ uint32_t bound_[ROWS];
  __shared__ int n_hit_[ROWS], n_cand_[ROWS];
  uint64_t* const cand = cand_[row_of_group];
  int *const hits = hits_[row_of_group], *const counts = counts_[row_of_group];
  uint32_t* const maxima = maxima_[row_of_group];
  float* const slots = slots_[row_of_group];
  uint32_t& bound = bound_[row_of_group];
  int &n_hit = n_hit_[row_of_group], &n_cand = n_cand_[row_of_group];

  u32x4 reg[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (wave_first + j * NT < z.granules) reg[j] = z.load(tid + j * NT);
  // f(granule, its number) for this thread's granules
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (wave_first + j * NT >= z.granules) continue;
      stay_packed(reg[j]);
      f(reg[j], tid + j * NT);
    }
    for (int g = tid + NV * NT; g < z.granules; g += NT) f(z.load(g), g);
  };
  // the maxima the bound comes from: each thread's, or -- a row of one wave, when k comes near its 64 lanes -- each granule's
  float best = neg_inf();
  uint32_t own[NV];
  const bool by_granule = W == 1 && a.K > 24;
  if (by_granule) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float g = neg_inf();
      if (j * NT < z.granules) {
#pragma unroll
        for (int i = 0; i < GN; ++i) g = fmaxf(g, granule_get<T>(reg[j], i));
      }
      own[j] = order_key(g);
    }
  } else {
    each([&](const u32x4& x, int) {
#pragma unroll
      for (int i = 0; i < GN; ++i) best = fmaxf(best, granule_get<T>(x, i));
    });
  }
  if constexpr (W > 1) maxima[tid] = order_key(best);
  if (tid == 0) n_hit = n_cand = 0;
  row_sync<NT>();
  if (tid < 64) {
    uint32_t lo = 0;
    if constexpr (W > 1) {
      uint32_t top[W];
#pragma unroll
      for (int i = 0; i < W; ++i) top[i] = maxima[lane + 64 * i];
      if (a.K < NT) lo = reach_of<W>(top, a.K);
    } else if (by_granule) {
      if (a.K < NT * NV) lo = reach_of<NV>(own, a.K);
    } else {
      const uint32_t top = order_key(best);
      lo = reach_of<1>(&top, a.K);
    }
    if (lane == 0) bound = max(lo, kKeyNegInf);
  }
  row_sync<NT>();
  const float c = a.inv_tau * kLog2e;
  float least = order_value(bound);                     // (keys between two floats' keys do not exist)
  float ref = least - least == 0.0f ? least : 0.0f;
  // the elements below the bound are summed relative to it; granules that hold others are listed, then looked through
  float others = 0.0f;
  each([&](const u32x4& x, int g) {
    float part = 0.0f;
    bool hit = false;
#pragma unroll
    for (int i = 0; i < GN; ++i) {
      const float e = granule_get<T>(x, i), p = exp2_hw((e - ref) * c);
      const bool below = e < least;
      part += below ? p : 0.0f;
      hit = hit || !below;
    }
    others += part;
    settle(others);
    if (hit && g < z.granules) {
      const int at = atomicAdd(&n_hit, 1);
      if (at < kCap) hits[at] = g;
    }
  });
  row_sync<NT>();
  if (n_hit <= kCap) {
    for (int q = tid; q < n_hit; q += NT) {
      const int e0 = z.first(hits[q]);
      for (int i = 0; i < GN; ++i) {
        const int v = e0 + i;
        if (v < 0 || v >= a.V) continue;
        const float e = static_cast<float>(z.p[v]);
        if (e < least) continue;
        const int at = atomicAdd(&n_cand, 1);
        if (at < kCap) cand[at] = candidate(order_key(e), v);
      }
    }
  }
  row_sync<NT>();
  int n = n_hit <= kCap ? n_cand : kCap + 1;
  uint32_t key = bound;                                 // when exactly k are listed: they lie above it, or on it up to class v_hi
  int v_hi = a.V - 1;
  if (n > kCap) {
    // Too many elements reach the bound (they are equal, or nearly all of the row is): the k-th largest key itself, then the
    // class up to which the elements equal to it belong.  Counts over the row, read again.
    auto count = [&](uint32_t key, int v_last) {        // elements above `key`, or equal to it up to class v_last
      int m = 0;
      for (int g = tid; g < z.granules; g += NT) {
        const u32x4 x = z.load(g);
        const int e0 = z.first(g);
#pragma unroll
        for (int i = 0; i < GN; ++i) {
          const int v = e0 + i;
          const uint32_t k = order_key(granule_get<T>(x, i));
          m += (v >= 0 && v < a.V && (k > key || (k == key && v <= v_last))) ? 1 : 0;
        }
      }
      return row_count<NT>(m, counts);
    };
    if (count(key, -1) >= a.K) {
      uint32_t lo = key + 1u, hi = 0xFFFFFFFFu;         // invariant: count(>= lo) >= k, count(> hi) < k
      while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (count(mid, -1) >= a.K) lo = mid + 1u;       // elements above mid
        else hi = mid;
      }
      key = lo;
    }
    int v_lo = -1;                                      // invariant: too few with v <= v_lo, enough with v <= v_hi
    while (v_hi - v_lo > 1) {
      const int mid = v_lo + ((v_hi - v_lo) >> 1);
      if (count(key, mid) >= a.K) v_hi = mid;
      else v_lo = mid;
    }
    row_sync<NT>();
    if (tid == 0) n_cand = 0;
    row_sync<NT>();
    least = key == 0xFFFFFFFFu ? __builtin_nanf("") : order_value(key);
    ref = least - least == 0.0f ? least : 0.0f;
    others = 0.0f;
    for (int g = tid; g < z.granules; g += NT) {
      const u32x4 x = z.load(g);
      const int e0 = z.first(g);
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        const int v = e0 + i;
        const float e = granule_get<T>(x, i);
        const uint32_t k = order_key(e);
        if (v < 0 || v >= a.V) continue;
        if (k > key || (k == key && v <= v_hi)) cand[atomicAdd(&n_cand, 1)] = candidate(k, v);      // exactly K of them
        else part += exp2_hw((e - ref) * c);
      }
      others += part;
    }
    row_sync<NT>();
    n = a.K;
  }
  // rank by counting; what is not selected goes back to the list's front in the order of its rank
  constexpr int kMine = (kCap + NT - 1) / NT;
  uint64_t mine[kMine];
  int rank[kMine];
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    const int i = tid + q * NT;
    mine[q] = i < n ? cand[i] : 0;
    rank[q] = 0;
    if (i < n)
      for (int j = 0; j < n; ++j) rank[q] += cand[j] > mine[q] ? 1 : 0;
  }
  others = row_all_sum<NT>(others, slots);   // (its barrier: the list has been read)
  if (a.rest && n == a.K && n < a.V && !(others >= 1.0e-20f && others < __builtin_inff())) {
    // The selected elements are infinite, or so far above the others that those vanish beside them: the others' sum relative to
    // the largest of them, over the row read again.
    auto over_others = [&](auto f) {
      for (int g = tid; g < z.granules; g += NT) {
        const u32x4 x = z.load(g);
        const int e0 = z.first(g);
        for (int i = 0; i < GN; ++i) {
          const int v = e0 + i;
          const float e = granule_get<T>(x, i);
          const uint32_t k = order_key(e);
          if (v >= 0 && v < a.V && (k < key || (k == key && v > v_hi))) f(e);
        }
      }
    };
    float m = neg_inf(), sum = 0.0f;
    over_others([&](float e) { m = fmaxf(m, e); });
    m = row_all_max<NT>(m, slots + W);
    ref = m - m == 0.0f ? m : 0.0f;
    over_others([&](float e) { sum += exp2_hw((e - ref) * c); });
    others = row_all_sum<NT>(sum, slots);
  }
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    if (tid + q * NT >= n) continue;
    const int v = static_cast<int>(~static_cast<uint32_t>(mine[q]));
    if (rank[q] < a.K) {
      static_cast<T*>(a.values)[row * a.K + rank[q]] = z.p[v];
      a.indices[row * a.K + rank[q]] = v;
    } else {
      cand[rank[q] - a.K] = mine[q];
    }
  }
  if (!a.rest) return;
  row_sync<NT>();
  // the candidates left over, relative to the largest of them
  const int left = n - a.K;
  float more = 0.0f, from = 0.0f;
  if (left > 0) {                              // (only without the bisection: then a.K + left candidates were listed)
    const float first = order_value(static_cast<uint32_t>(cand[0] >> 32));
    from = first - first == 0.0f ? first : 0.0f;
    for (int i = tid; i < left; i += NT) {
      const uint32_t key = static_cast<uint32_t>(cand[i] >> 32);
      more += exp2_hw(((key == 0xFFFFFFFFu ? __builtin_nanf("") : order_value(key)) - from) * c);
    }
  }
  more = row_all_sum<NT>(more, slots + W);
  if (tid == 0) {
    float r = neg_inf();
    if (left > 0 && more != 0.0f)              // ref <= from where anything lies below the bound: the others' sum relative to it
      r = from * a.inv_tau + kLn2 * __builtin_amdgcn_logf(more + (others != 0.0f ? others * exp2_hw((ref - from) * c) : 0.0f));
    else if (others != 0.0f)
      r = ref * a.inv_tau + kLn2 * __builtin_amdgcn_logf(others);
    a.rest[row] = r;
  }
}

template <typename T, int NT, int NV>
static int topk_launch(TopkArgs a, hipStream_t s) {
  constexpr int ROWS = kRowsPerGroup<NT>;
  for (a.row0 = 0; a.row0 < a.N; a.row0 += kRowsPerLaunch) {
    const int rows = static_cast<int>(std::min<int64_t>(kRowsPerLaunch, a.N - a.row0));
    hipLaunchKernelGGL((topk_logits_kernel<T, NT, NV>), dim3((rows + ROWS - 1) / ROWS), dim3(NT * ROWS), 0, s, a);
    if (const int rc = to_err(hipGetLastError())) return rc;
  }
  return 0;
}
// Threads and registers by the granules of a row, as distill.hip: as few waves as hold the row, four to eight granules a thread.
// The bound comes from the threads' (one wave: the granules') maxima: about twice k of them or more up to k = 128.  With fewer the
// bound falls, and with k of them or fewer there is none: the list overflows and the row is bisected.  2,048 rows of 16,000 bf16
// classes 36 us at k = 128, 57 at 160, 122 at 192, 655 at 256; of 8,000 fp32 classes 32, 46, 106 and 427; of 50,257 fp32 classes (1,024
// threads) 103, 107, 111 and 122.
// bf16, k = 64: 32,000 classes 36 us with 512 x 8 for 2,048 rows (47 with 1024 x 4); 131,072 classes 280 us with 1024 x 8 and the
// row's other half read again, 330 us with 1024 x 16 (one workgroup per CU, whose phases then overlap with no other's); one row
// of them 16 us with 1024 x 16, 19 with 1024 x 8.
template <typename T>
static int topk_pick(const TopkArgs& a, hipStream_t s) {
  constexpr int GN = Granule<T>::N;
  const bool aligned = aligned16(a.z) && (a.ldz % GN == 0 || a.N == 1);
  const int granules = (a.V + (aligned ? 0 : GN - 1) + GN - 1) / GN;
  if (granules <= 64 && 2 * a.K <= granules + 16) return topk_launch<T, 64, 1>(a, s);
  if (granules <= 256 && 2 * a.K <= granules + 16) return topk_launch<T, 64, 4>(a, s);
  if (granules <= 1024) return topk_launch<T, 256, 4>(a, s);
  if (granules <= 2048) return topk_launch<T, 256, 8>(a, s);
  if (granules <= 4096) return topk_launch<T, 512, 8>(a, s);
  if (granules <= 6144) return topk_launch<T, 512, 12>(a, s);
  if (a.N <= kCUs && granules <= 16384) return topk_launch<T, 1024, 16>(a, s);
  return topk_launch<T, 1024, 8>(a, s);
}

}  // namespace bde

using namespace bde;

extern "C" int bde_topk_limits(int* max_classes, int* max_k) {
  if (max_classes) *max_classes = kTopkMaxV;
  if (max_k) *max_k = kTopkMaxK;
  return 0;
}

extern "C" int bde_topk_logits(const void* logits, int dtype, int64_t ldz, float temperature, int N, int V, int K, void* values,
                               int64_t* indices, float* rest, void* stream) {
  if (!dtype_ok(dtype) || N < 0 || V < 1 || V > kTopkMaxV || K < 1 || K > kTopkMaxK || K > V || ldz < V || !(temperature > 0.0f) ||
      !(1.0f / temperature > 0.0f) || !(1.0f / temperature < __builtin_inff()))
    return BDE_ERR_INVALID;
  if (N == 0) return 0;
  if (!logits || !values || !indices || reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype) != 0) return BDE_ERR_INVALID;
  const TopkArgs a{logits, ldz, values, indices, rest, N, V, K, 1.0f / temperature, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == BDE_F32) return topk_pick<float>(a, s);
  if (dtype == BDE_BF16) return topk_pick<bf16_t>(a, s);
  return topk_pick<f16_t>(a, s);
}

extern "C" __attribute__((visibility("hidden"))) int bde_internal_load_topk(void) {
  hipFuncAttributes attr;
  return to_err(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&topk_logits_kernel<float, 64, 1>)));
}
