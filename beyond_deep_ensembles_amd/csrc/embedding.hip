// Scaled embedding lookup, plain and mean-field Gaussian, and its gradient by sorted tokens.
//
//   plain:     out_i = s W[t_i]                              dW[v]   = s sum_{i: t_i = v} g_i
//   Gaussian:  out_i = s (mu[t_i] + softplus(rho[t_i]) e)    dmu[v]  = s sum g_i,  drho[v] = s sigmoid(rho[v]) sum g_i e
// with e = eps[i] (noise by position: the local reparameterisation of a linear layer with a one-hot input, whose output
// variance is sigma[t]^2 itself) or e = eps[t_i] (noise by token: ONE draw of the table, of which only the touched rows are
// evaluated).  Without a noise tensor the kernels generate it (Philox, element i * D + d or t * D + d of the stream).
// The padding token has no noise and no gradient.  A token outside [0, V) gives a row of NaN and no gradient.
//
// The gradient is bit-reproducible: a stable counting sort of the positions by token, then every token's rows are added in the
// order of their positions, in fixed pieces of the sorted list (fp32), pieces in order.  No float atomics.
#include "token_common.hpp"

namespace bde {

constexpr int kNoiseNone = 0, kNoisePosition = 1, kNoiseToken = 2;

struct EmbedArgs {
  const void* weight;      // [V, ldw]  (mean of the Gaussian)
  int64_t ldw;
  const float* rho;        // [V, ldrho]
  int64_t ldrho;
  const void* tokens;
  int tokens64;
  const float* eps;        // [N or V, ldeps] or NULL: Philox
  int64_t ldeps;
  uint64_t seed, stream_id;
  float scale;
  int64_t padding;         // token without noise and gradient, -1: none
  void* out;               // [N, D]
  const void* g;           // [N, ldg]
  int64_t ldg;
  void* gw;                // [V, D]
  float* grho;             // [V, D]
  int64_t N;
  int V, D;
  // the gradient's workspace
  int* header;             // [0]: positions in the sorted list
  int* order;              // [N] positions, by token, then by position
  int* key;                // [N] their tokens
  float* part;             // [pieces][2][accumulators][D] sums of the runs that cross a piece's borders
  int piece;
  int bucket;              // tokens per workgroup of the sort
};

// VEC consecutive elements as fp32
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (VEC == 1) {
    f[0] = static_cast<float>(p[0]);
  } else if constexpr (sizeof(T) * VEC == 32) {
    const f32x4 a = ld4(reinterpret_cast<const float*>(p)), b = ld4(reinterpret_cast<const float*>(p) + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = a[i];
      f[4 + i] = b[i];
    }
  } else {
    struct alignas(sizeof(T) * VEC) Pack {
      T v[VEC];
    };
    const Pack b = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = static_cast<float>(b.v[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
    T v[VEC];
  };
  Pack b;
#pragma unroll
  for (int i = 0; i < VEC; ++i) b.v[i] = static_cast<T>(f[i]);
  *reinterpret_cast<Pack*>(p) = b;
}
// noise of VEC elements from `element` on (VEC = 4: `element` is a multiple of 4, one Philox group)
template <int VEC>
__device__ __forceinline__ void noise_vec(uint64_t seed, uint64_t stream_id, int64_t element, float* f) {
  const f32x4 z = philox_normal4(seed, stream_id, static_cast<uint64_t>(element) >> 2, kDomainDiag);
  if constexpr (VEC == 1) {
    const int k = static_cast<int>(element & 3);
    f[0] = k == 0 ? z.x : k == 1 ? z.y : k == 2 ? z.z : z.w;
  } else {
    static_assert(VEC == 4, "one Philox group");
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = z[i];
  }
}

// 2^log_lanes lanes per row
template <typename TW, typename TO, int NOISE, int VEC>
__global__ __launch_bounds__(kBlock) void embedding_fwd_kernel(EmbedArgs a, int log_lanes) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) >> log_lanes;
  if (row >= a.N) return;
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  const int t = load_index(a.tokens, a.tokens64, row, a.V);
  TO* const out = static_cast<TO*>(a.out) + row * a.D;
  const float scale = t >= 0 ? a.scale : __builtin_nanf("");
  const int64_t tr = t >= 0 ? t : 0;
  const TW* const w = static_cast<const TW*>(a.weight) + tr * a.ldw;
  const bool noisy = NOISE != kNoiseNone && t != a.padding;
  const int64_t noise_row = NOISE == kNoisePosition ? row : tr;
#pragma unroll 4
  for (int d = lane * VEC; d < a.D; d += lanes * VEC) {
    float f[VEC];
    load_vec<TW, VEC>(w + d, f);
    if constexpr (NOISE != kNoiseNone) {
      if (noisy) {
        float r[VEC], e[VEC];
        load_vec<float, VEC>(a.rho + tr * a.ldrho + d, r);
        if (a.eps) load_vec<float, VEC>(a.eps + noise_row * a.ldeps + d, e);
        else noise_vec<VEC>(a.seed, a.stream_id, noise_row * a.D + d, e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] += softplus(r[i]) * e[i];
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] *= scale;
    store_vec<TO, VEC>(out + d, f);
  }
}

// ---------------------------------------------------------------- gradient --
// Stable counting sort in ONE launch.  A workgroup owns the tokens [lo, lo + bucket): it reads ALL tokens, counts those of its
// own range (per wave and token) and those below its range -- the latter is where its part of the sorted list begins, so no
// scan between workgroups is needed -- and writes its positions in order.  The 16 waves take 16 consecutive parts of the list;
// a wave keeps the matches of its part in LDS and reads its part again only when they do not fit.  Rows of tokens that do not
// occur are zero-filled here.
// Work: (tokens / 64) wave-steps per workgroup, the list comes from L2 after the first reader.
constexpr int kSortThreads = 1024, kSortWaves = 16, kSortList = 256, kMaxBucket = 512;

template <typename TW>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(EmbedArgs a) {
  extern __shared__ int hist[];                     // [16][bucket] counts, then where the next one goes
  __shared__ int list_p[kSortWaves][kSortList];
  __shared__ uint16_t list_r[kSortWaves][kSortList];
  __shared__ int sums[kSortWaves], below[kSortWaves], totals[kMaxBucket];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = static_cast<int>(blockIdx.x) * a.bucket, hi = min(a.V, lo + a.bucket), own = hi - lo;
  for (int i = tid; i < kSortWaves * a.bucket; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  int* const mine = hist + wave * a.bucket;
  const int n = static_cast<int>(a.N), pad = static_cast<int>(a.padding);
  const int chunk = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int begin = min(n, wave * chunk), end = min(n, begin + chunk);
  const unsigned long long before = (1ull << lane) - 1ull;
  int listed = 0, less = 0;
  bool fits = true;
  for (int base = begin; base < end; base += 256) {
    int t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int p = base + 64 * u + lane;
      t[u] = p < end ? load_index(a.tokens, a.tokens64, p, a.V) : -1;
      if (t[u] == pad) t[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = t[u] >= lo && t[u] < hi;
      less += (t[u] >= 0 && t[u] < lo) ? 1 : 0;
      const unsigned long long m = __ballot(in);
      if (m == 0) continue;
      const int k = __popcll(m);
      fits = fits && listed + k <= kSortList;
      if (in) {
        atomicAdd(&mine[t[u] - lo], 1);
        if (fits) {
          const int at = listed + __popcll(m & before);
          list_p[wave][at] = base + 64 * u + lane;
          list_r[wave][at] = static_cast<uint16_t>(t[u] - lo);
        }
      }
      listed += k;
    }
  }
  less = static_cast<int>(wave_all_sum(static_cast<float>(less)));     // <= 2^24 per wave: exact
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // per token: its total, the exclusive sum over the tokens of the bucket, then each wave's share behind the ones before it
  int total = 0;
  if (tid < own)
    for (int w = 0; w < kSortWaves; ++w) total += hist[w * a.bucket + tid];
  int run = total;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int got = __shfl(run, (lane - off) & 63, 64);
    if (lane >= off) run += got;
  }
  if (lane == 63) sums[wave] = run;
  if (tid < own) totals[tid] = total;
  __syncthreads();
  int start = run - total, all = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    start += below[w] + (w < wave ? sums[w] : 0);
    all += below[w] + sums[w];
  }
  if (tid < own) {
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = hist[w * a.bucket + tid];
      hist[w * a.bucket + tid] = start;
      start += c;
    }
  }
  if (tid == 0 && hi == a.V) a.header[0] = all;
  __syncthreads();
  // positions in order: lanes of one token take consecutive places (the lanes that agree with this one on every bit of the
  // token's number in the bucket: a ballot per bit, whatever the tokens are)
  const int bits = 32 - __builtin_clz(a.bucket | 1);
  auto place = [&](bool in, int r, int p) {
    unsigned long long same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const bool set = (r >> b) & 1;
      const unsigned long long m = __ballot(set);
      same &= set ? m : ~m;
    }
    const int at = in ? mine[r] : 0, rank = __popcll(same & before);
    if (in) {
      a.order[at + rank] = p;
      a.key[at + rank] = lo + r;
      if (rank == 0) mine[r] = at + __popcll(same);
    }
  };
  if (fits) {
    for (int base = 0; base < listed; base += 64) {
      const bool in = base + lane < listed;
      place(in, in ? list_r[wave][base + lane] : 0, in ? list_p[wave][base + lane] : 0);
    }
  } else {
    for (int base = begin; base < end; base += 64) {
      const int p = base + lane;
      int t = p < end ? load_index(a.tokens, a.tokens64, p, a.V) : -1;
      if (t == pad) t = -1;
      const bool in = t >= lo && t < hi;
      place(in, in ? t - lo : 0, p);
    }
  }
  // rows of tokens that do not occur: zero
  const int64_t row_bytes = static_cast<int64_t>(a.D) * sizeof(TW);
  auto zero_row = [&](char* p, int64_t bytes) {
    if (bytes % 16 == 0) {
      const u32x4 z = {0u, 0u, 0u, 0u};
      for (int64_t b = lane * 16; b < bytes; b += 1024) *reinterpret_cast<u32x4*>(p + b) = z;
    } else if (bytes % 4 == 0) {
      for (int64_t b = lane * 4; b < bytes; b += 256) *reinterpret_cast<uint32_t*>(p + b) = 0u;
    } else {
      for (int64_t b = lane * 2; b < bytes; b += 128) *reinterpret_cast<uint16_t*>(p + b) = 0;
    }
  };
  for (int r = wave; r < own; r += kSortWaves) {
    if (totals[r]) continue;
    zero_row(static_cast<char*>(a.gw) + (lo + r) * row_bytes, row_bytes);
    if (a.grho) zero_row(reinterpret_cast<char*>(a.grho) + (lo + r) * static_cast<int64_t>(a.D) * 4, static_cast<int64_t>(a.D) * 4);
  }
}

// the sums of one token's run -> its gradient rows
template <typename TW, int NOISE, int VEC>
__device__ __forceinline__ void embedding_finish(const EmbedArgs& a, int t, int d, const float* acc, const float* acc2) {
  float f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = a.scale * acc[i];
  store_vec<TW, VEC>(static_cast<TW*>(a.gw) + static_cast<int64_t>(t) * a.D + d, f);
  if constexpr (NOISE != kNoiseNone) {
    float r[VEC], e[VEC];
    load_vec<float, VEC>(a.rho + t * a.ldrho + d, r);
    if constexpr (NOISE == kNoiseToken) {
      if (a.eps) load_vec<float, VEC>(a.eps + t * a.ldeps + d, e);
      else noise_vec<VEC>(a.seed, a.stream_id, static_cast<int64_t>(t) * a.D + d, e);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = a.scale * sigmoidf(r[i]) * (NOISE == kNoiseToken ? e[i] * acc[i] : acc2[i]);
    store_vec<float, VEC>(a.grho + static_cast<int64_t>(t) * a.D + d, f);
  }
}

// One wave per (piece of the sorted list, 64 * VEC columns): it adds the rows of g in order and writes the token's gradient
// where a run ends.  A run that began in an earlier piece leaves its sum in part[piece][0], one that begins here and goes on
// in part[piece][1].
template <typename TW, typename TG, int NOISE, int VEC>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(EmbedArgs a, int column_tiles) {
  constexpr int NACC = NOISE == kNoisePosition ? 2 : 1, kAhead = 8;
  const int lane = threadIdx.x & 63;
  const int id = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * (kBlock / 64) + static_cast<int>(threadIdx.x >> 6));
  const int piece = id / column_tiles, d = (id % column_tiles) * 64 * VEC + lane * VEC;
  const int n = a.header[0], s0 = piece * a.piece;
  if (s0 >= n) return;
  const int count = min(a.piece, n - s0);
  const bool active = d < a.D;
  const int my_pos = lane < count ? a.order[s0 + lane] : 0, my_key = lane < count ? a.key[s0 + lane] : -1;
  const int key_before = s0 > 0 ? a.key[s0 - 1] : -1, key_after = s0 + count < n ? a.key[s0 + count] : -1;
  float acc[VEC], acc2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = acc2[i] = 0.0f;
  int run_begin = 0;
  for (int s = 0; s < count; s += kAhead) {
    float g[kAhead][VEC], e[NACC == 2 ? kAhead : 1][VEC];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s + u < count) {
        const int64_t pos = __builtin_amdgcn_readlane(my_pos, s + u);
        if (active) {
          load_vec<TG, VEC>(static_cast<const TG*>(a.g) + pos * a.ldg + d, g[u]);
          if constexpr (NACC == 2) {
            if (a.eps) load_vec<float, VEC>(a.eps + pos * a.ldeps + d, e[u]);
            else noise_vec<VEC>(a.seed, a.stream_id, pos * a.D + d, e[u]);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s + u < count) {
        const int key = __builtin_amdgcn_readlane(my_key, s + u);
        const bool last = s + u + 1 == count;
        const int next = last ? key_after : __builtin_amdgcn_readlane(my_key, (s + u + 1) & 63);
        if (active) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            acc[i] += g[u][i];
            if constexpr (NACC == 2) acc2[i] = __builtin_fmaf(g[u][i], e[u][i], acc2[i]);
          }
        }
        if (next != key || last) {
          const bool begun_before = run_begin == 0 && key_before == key, goes_on = next == key;
          if (active) {
            if (begun_before || goes_on) {
              float* const p = a.part + ((static_cast<int64_t>(piece) * 2 + (begun_before ? 0 : 1)) * NACC) * a.D + d;
              store_vec<float, VEC>(p, acc);
              if constexpr (NACC == 2) store_vec<float, VEC>(p + a.D, acc2);
            } else {
              embedding_finish<TW, NOISE, VEC>(a, key, d, acc, acc2);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = acc2[i] = 0.0f;
          }
          run_begin = s + u + 1;
        }
      }
    }
  }
}

// One workgroup per (piece, 64 * VEC columns): if a run begins in this piece and goes on behind it, add its parts.  The four
// waves take every fourth part; their sums are added in order.
template <typename TW, int NOISE, int VEC>
__global__ __launch_bounds__(kBlock) void embedding_join_kernel(EmbedArgs a, int column_tiles) {
  constexpr int NACC = NOISE == kNoisePosition ? 2 : 1, kWaves = kBlock / 64;
  __shared__ float sums[kWaves - 1][NACC][64 * VEC];
  const int piece = static_cast<int>(blockIdx.x) / column_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = (static_cast<int>(blockIdx.x) % column_tiles) * 64 * VEC + lane * VEC;
  const int n = a.header[0], s0 = piece * a.piece, s1 = s0 + a.piece;
  if (s1 >= n) return;
  const int key = a.key[s1 - 1];
  if (a.key[s1] != key || (s0 > 0 && a.key[s0 - 1] == key)) return;     // (keys are sorted: equal ends mean equal in between)
  // parts of the pieces behind: those whose first key is this one
  int behind = 0;
  for (;;) {
    const int64_t s = (static_cast<int64_t>(piece) + 1 + behind + lane) * a.piece;
    const unsigned long long m = __ballot(s < n && a.key[s < n ? s : 0] == key);
    const int k = m == ~0ull ? 64 : __builtin_ctzll(~m);
    behind += k;
    if (k < 64) break;
  }
  float acc[VEC], acc2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = acc2[i] = 0.0f;
  if (d < a.D) {
#pragma unroll 8
    for (int q = wave; q <= behind; q += kWaves) {
      const float* const p = a.part + ((static_cast<int64_t>(piece + q) * 2 + (q == 0 ? 1 : 0)) * NACC) * a.D + d;
      float f[VEC];
      load_vec<float, VEC>(p, f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += f[i];
      if constexpr (NACC == 2) {
        load_vec<float, VEC>(p + a.D, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc2[i] += f[i];
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sums[wave - 1][0][i * 64 + lane] = acc[i];
      if constexpr (NACC == 2) sums[wave - 1][NACC - 1][i * 64 + lane] = acc2[i];
    }
  }
  __syncthreads();
  if (wave > 0 || d >= a.D) return;
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      acc[i] += sums[w][0][i * 64 + lane];
      if constexpr (NACC == 2) acc2[i] += sums[w][NACC - 1][i * 64 + lane];
    }
  embedding_finish<TW, NOISE, VEC>(a, key, d, acc, acc2);
}

// positions per piece: short pieces keep enough waves in flight when there are few tokens, long ones write fewer parts
static int embedding_piece(int64_t n) { return n <= 8192 ? 16 : n <= 65536 ? 32 : 64; }

template <typename TW, typename TO, int NOISE, int VEC>
static int embedding_fwd_launch(const EmbedArgs& a, hipStream_t s) {
  const int vecs = (a.D + VEC - 1) / VEC;
  int log_lanes = 3;
  while (log_lanes < 6 && (1 << log_lanes) < vecs) ++log_lanes;
  const int64_t blocks = ((a.N << log_lanes) + kBlock - 1) / kBlock;
  hipLaunchKernelGGL((embedding_fwd_kernel<TW, TO, NOISE, VEC>), dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, a, log_lanes);
  return to_err(hipGetLastError());
}
template <typename TW, typename TG, int NOISE, int VEC>
static int embedding_bwd_launch(const EmbedArgs& a, hipStream_t s) {
  const int buckets = (a.V + a.bucket - 1) / a.bucket;
  hipLaunchKernelGGL((embedding_sort_kernel<TW>), dim3(buckets), dim3(kSortThreads), sizeof(int) * kSortWaves * a.bucket, s, a);
  if (const int rc = to_err(hipGetLastError())) return rc;
  if (a.N == 0) return 0;
  const int tiles = (a.D + 64 * VEC - 1) / (64 * VEC), pieces = static_cast<int>((a.N + a.piece - 1) / a.piece);
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(pieces) * tiles + kBlock / 64 - 1) / (kBlock / 64));
  hipLaunchKernelGGL((embedding_sum_kernel<TW, TG, NOISE, VEC>), dim3(blocks), dim3(kBlock), 0, s, a, tiles);
  if (const int rc = to_err(hipGetLastError())) return rc;
  if (pieces > 1) hipLaunchKernelGGL((embedding_join_kernel<TW, NOISE, VEC>), dim3(pieces * tiles), dim3(kBlock), 0, s, a, tiles);
  return to_err(hipGetLastError());
}

static bool on_border(const void* p, int64_t ld, size_t element, int vec) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (element * vec > 16 ? 16 : element * vec) == 0 && ld % vec == 0);
}
template <typename TW, typename T2, int NOISE, bool BWD>
static int embedding_pick(const EmbedArgs& a, hipStream_t s) {
  constexpr int VEC = sizeof(TW) == 2 && sizeof(T2) == 2 && NOISE == kNoiseNone ? 8 : 4;
  const bool wide = a.D % VEC == 0 && on_border(a.weight, a.ldw, sizeof(TW), VEC) && on_border(a.rho, a.ldrho, 4, VEC) &&
                    on_border(a.eps, a.ldeps, 4, VEC) && on_border(a.out, a.D, sizeof(T2), VEC) && on_border(a.g, a.ldg, sizeof(T2), VEC) &&
                    on_border(a.gw, a.D, sizeof(TW), VEC) && on_border(a.grho, a.D, 4, VEC);
  if constexpr (BWD) return wide ? embedding_bwd_launch<TW, T2, NOISE, VEC>(a, s) : embedding_bwd_launch<TW, T2, NOISE, 1>(a, s);
  else return wide ? embedding_fwd_launch<TW, T2, NOISE, VEC>(a, s) : embedding_fwd_launch<TW, T2, NOISE, 1>(a, s);
}
// table type x activation type: equal, or an fp32 table with activations of any type; the Gaussian's tables are fp32
template <bool BWD>
static int embedding_dispatch(const EmbedArgs& a, int wdtype, int dtype, int noise, hipStream_t s) {
  if (noise == kNoiseNone) {
    if (wdtype == BDE_BF16) return embedding_pick<bf16_t, bf16_t, kNoiseNone, BWD>(a, s);
    if (wdtype == BDE_F16) return embedding_pick<f16_t, f16_t, kNoiseNone, BWD>(a, s);
    if (dtype == BDE_F32) return embedding_pick<float, float, kNoiseNone, BWD>(a, s);
    if (dtype == BDE_BF16) return embedding_pick<float, bf16_t, kNoiseNone, BWD>(a, s);
    return embedding_pick<float, f16_t, kNoiseNone, BWD>(a, s);
  }
  if (noise == kNoisePosition) {
    if (dtype == BDE_F32) return embedding_pick<float, float, kNoisePosition, BWD>(a, s);
    if (dtype == BDE_BF16) return embedding_pick<float, bf16_t, kNoisePosition, BWD>(a, s);
    return embedding_pick<float, f16_t, kNoisePosition, BWD>(a, s);
  }
  if (dtype == BDE_F32) return embedding_pick<float, float, kNoiseToken, BWD>(a, s);
  if (dtype == BDE_BF16) return embedding_pick<float, bf16_t, kNoiseToken, BWD>(a, s);
  return embedding_pick<float, f16_t, kNoiseToken, BWD>(a, s);
}
static bool embedding_args_ok(int wdtype, int dtype, int noise, int64_t N, int64_t V, int64_t D) {
  if (!dtype_ok(wdtype) || !dtype_ok(dtype) || (wdtype != BDE_F32 && wdtype != dtype)) return false;
  if (noise < kNoiseNone || noise > kNoiseToken || (noise != kNoiseNone && wdtype != BDE_F32)) return false;
  return N >= 0 && N <= BDE_EMBEDDING_MAX_TOKENS && V >= 1 && V <= BDE_EMBEDDING_MAX_ROWS && D >= 1 && D <= BDE_EMBEDDING_MAX_DIM;
}

}  // namespace bde

using namespace bde;

extern "C" int bde_embedding_fwd(const void* weight, int weight_dtype, int64_t ldw, const float* rho, int64_t ldrho,
                                 const void* tokens, int tokens64, const float* eps, int64_t ldeps, int noise, uint64_t seed,
                                 uint64_t stream_id, float scale, int64_t padding, void* out, int out_dtype, int64_t N, int64_t V,
                                 int64_t D, void* stream) {
  if (!embedding_args_ok(weight_dtype, out_dtype, noise, N, V, D) || ldw < D || (noise != kNoiseNone) != (rho != nullptr) ||
      (rho && ldrho < D) || (eps && (noise == kNoiseNone || ldeps < D)) || padding < -1 || padding >= V)
    return BDE_ERR_INVALID;
  if (N == 0) return 0;
  if (!weight || !tokens || !out) return BDE_ERR_INVALID;
  EmbedArgs a{};
  a.weight = weight; a.ldw = ldw; a.rho = rho; a.ldrho = ldrho; a.tokens = tokens; a.tokens64 = tokens64; a.eps = eps; a.ldeps = ldeps;
  a.seed = seed; a.stream_id = stream_id; a.scale = scale; a.padding = padding; a.out = out;
  a.N = N; a.V = static_cast<int>(V); a.D = static_cast<int>(D);
  return embedding_dispatch<false>(a, weight_dtype, out_dtype, noise, static_cast<hipStream_t>(stream));
}

extern "C" size_t bde_embedding_bwd_ws_bytes(int64_t N, int64_t D, int noise) {
  if (N < 0 || N > BDE_EMBEDDING_MAX_TOKENS || D < 1 || D > BDE_EMBEDDING_MAX_DIM) return 0;
  const int64_t lists = 256 + 2 * ((4 * N + 255) / 256 * 256);
  const int64_t pieces = (N + embedding_piece(N) - 1) / embedding_piece(N);
  return static_cast<size_t>(lists + pieces * 2 * (noise == kNoisePosition ? 2 : 1) * D * 4 + 16);
}

extern "C" int bde_embedding_bwd(const void* g, int g_dtype, int64_t ldg, const void* tokens, int tokens64, const float* rho,
                                 int64_t ldrho, const float* eps, int64_t ldeps, int noise, uint64_t seed, uint64_t stream_id,
                                 float scale, int64_t padding, void* g_weight, int weight_dtype, float* g_rho, int64_t N, int64_t V,
                                 int64_t D, void* ws, size_t ws_bytes, void* stream) {
  if (!embedding_args_ok(weight_dtype, g_dtype, noise, N, V, D) || (noise != kNoiseNone) != (rho != nullptr) ||
      (rho != nullptr) != (g_rho != nullptr) || (rho && ldrho < D) || (eps && (noise == kNoiseNone || ldeps < D)) || padding < -1 ||
      padding >= V || !g_weight || !aligned16(g_weight) || !aligned16(g_rho) || !ws || !aligned16(ws) || ws_bytes < bde_embedding_bwd_ws_bytes(N, D, noise))
    return BDE_ERR_INVALID;
  if (N > 0 && (!g || !tokens || ldg < 0)) return BDE_ERR_INVALID;
  EmbedArgs a{};
  a.rho = rho; a.ldrho = ldrho; a.tokens = tokens; a.tokens64 = tokens64; a.eps = eps; a.ldeps = ldeps; a.seed = seed;
  a.stream_id = stream_id; a.scale = scale; a.padding = padding; a.g = g; a.ldg = ldg; a.gw = g_weight; a.grho = g_rho;
  a.N = N; a.V = static_cast<int>(V); a.D = static_cast<int>(D);
  const int64_t list = (4 * N + 255) / 256 * 256;
  char* const base = static_cast<char*>(ws);
  a.header = reinterpret_cast<int*>(base);
  a.order = reinterpret_cast<int*>(base + 256);
  a.key = reinterpret_cast<int*>(base + 256 + list);
  a.part = reinterpret_cast<float*>(base + 256 + 2 * list);
  a.piece = embedding_piece(N);
  // 256 workgroups (one per CU), or as many as keep a bucket's counts in LDS
  const int64_t want = std::max<int64_t>(kCUs, (V + kMaxBucket - 1) / kMaxBucket);
  a.bucket = static_cast<int>((V + want - 1) / want);
  return embedding_dispatch<true>(a, weight_dtype, g_dtype, noise, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("hidden"))) int bde_internal_load_embedding(void) {
  hipFuncAttributes attr;
  return to_err(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&embedding_sort_kernel<float>)));
}
