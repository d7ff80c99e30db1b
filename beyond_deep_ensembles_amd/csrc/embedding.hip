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
  int log_groups, bucket;  // workgroups of the sort (a power of two) and the most tokens one of them owns
  int chunk;               // > 0: the tokens are dealt out to the sort's workgroups first, this many per workgroup of that
  int log_deal;            // into a power of two of groups, each for one workgroup of the sort or for several
  int* counts;             // [chunks][dealt groups]
  int* group_start;        // [dealt groups + 1]
  int* dealt_p;            // [N] positions by dealt group, in order
  int* dealt_t;            // [N] their tokens
  int stream_zeros;        // zero rows are stored past the caches
  int join0;               // first workgroup of this launch of the join
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

// 2^log_lanes lanes per row, ROWS rows per group of lanes (their loads in flight together)
template <typename TW, typename TO, int NOISE, int VEC, int ROWS>
__global__ __launch_bounds__(kBlock) void embedding_fwd_kernel(EmbedArgs a, int log_lanes) {
  const int64_t first = ((static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) >> log_lanes) * ROWS;
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  int t[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) t[u] = first + u < a.N ? load_index(a.tokens, a.tokens64, first + u, a.V) : -1;
  for (int d = lane * VEC; d < a.D; d += lanes * VEC) {
    float f[ROWS][VEC], r[NOISE != kNoiseNone ? ROWS : 1][VEC], e[NOISE != kNoiseNone ? ROWS : 1][VEC];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int64_t row = first + u, tr = t[u] >= 0 ? t[u] : 0;
      load_vec<TW, VEC>(static_cast<const TW*>(a.weight) + tr * a.ldw + d, f[u]);
      if constexpr (NOISE != kNoiseNone) {
        const int64_t noise_row = NOISE == kNoiseToken ? tr : row < a.N ? row : 0;
        load_vec<float, VEC>(a.rho + tr * a.ldrho + d, r[u]);
        if (a.eps) load_vec<float, VEC>(a.eps + noise_row * a.ldeps + d, e[u]);
        else noise_vec<VEC>(a.seed, a.stream_id, noise_row * a.D + d, e[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if constexpr (NOISE != kNoiseNone) {
        if (t[u] != a.padding) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) f[u][i] += softplus(r[u][i]) * e[u][i];
        }
      }
      const float scale = t[u] >= 0 ? a.scale : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[u][i] *= scale;
      if (first + u < a.N) store_vec<TO, VEC>(static_cast<TO*>(a.out) + (first + u) * a.D + d, f[u]);
    }
  }
}

// ---------------------------------------------------------------- gradient --
// Stable counting sort in ONE launch.  Workgroup b of a power of two owns the tokens t = b, b + count, b + 2 count, ... (strided,
// because frequent tokens lie side by side in a vocabulary): it reads ALL tokens, counts its own (per wave and token) and those
// of the workgroups before it -- which is where its part of the sorted list begins, so no scan between workgroups is needed --
// and writes its positions, one token after the other, each token's in order.  The 16 waves take 16 consecutive parts of the
// list; a wave keeps the matches of its part in LDS and reads its part again only when they do not fit.  Rows of tokens that do
// not occur are zero-filled here.
// Work: (tokens / 64) wave-steps per workgroup, the list comes from L2 after the first reader; with a large table the zero rows
// bound the kernel (a stream of stores).
constexpr int kSortThreads = 1024, kSortWaves = 16, kSortList = 256, kMaxBucket = 512, kMaxDealGroups = 512;

// a token as it lies in memory: looked at when it is used, not when it is loaded
__device__ __forceinline__ int64_t raw_token(const EmbedArgs& a, int64_t i) {
  return a.tokens64 ? static_cast<const int64_t*>(a.tokens)[i] : static_cast<const int*>(a.tokens)[i];
}
__device__ __forceinline__ bool live_token(const EmbedArgs& a, int64_t raw) {    // false: no gradient
  const uint32_t lo = static_cast<uint32_t>(raw), hi = static_cast<uint32_t>(static_cast<uint64_t>(raw) >> 32);
  return hi == 0 && lo < static_cast<uint32_t>(a.V) && lo != static_cast<uint32_t>(a.padding);
}

// With many tokens the workgroups do not read all of them: two short kernels deal the positions out first (count per chunk and
// group; then each chunk writes its positions behind those of the chunks before it).  Gradient of a 30,011 x 256
// fp32 table: 32,768 tokens 35 us without, 39 with; 65,536 tokens 65 and 49; 262,144 tokens 202 and 118.  A large table takes more
// workgroups in the sort than are dealt to (kMaxDealGroups): token t goes to group t mod that number, and the workgroups b, b +
// that number, ... of the sort read the group's share and find their own in it (when all of them read all tokens: 262,208 x 64, 65,536
// tokens 85 us against 64; 1,048,576 x 64, 262,144 tokens 386 against 147).
__global__ __launch_bounds__(kSortThreads) void embedding_count_kernel(EmbedArgs a, int log_groups) {
  __shared__ int count[kMaxDealGroups];
  const int groups = 1 << log_groups, n = static_cast<int>(a.N);
  for (int g = threadIdx.x; g < groups; g += kSortThreads) count[g] = 0;
  __syncthreads();
  const int begin = static_cast<int>(blockIdx.x) * a.chunk, end = min(n, begin + a.chunk);
#pragma unroll 4
  for (int p = begin + static_cast<int>(threadIdx.x); p < end; p += kSortThreads) {
    const int64_t t = raw_token(a, p);
    if (live_token(a, t)) atomicAdd(&count[static_cast<int>(t) & (groups - 1)], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kSortThreads) a.counts[static_cast<int64_t>(blockIdx.x) * groups + g] = count[g];
}

// the lanes that agree with this one in the low `bits` bits of r, of those that are `in`: a ballot per bit, whatever r is
__device__ __forceinline__ unsigned long long lanes_like(bool in, int r, int bits) {
  unsigned long long same = __ballot(in);
  for (int b = 0; b < bits; ++b) {
    const bool set = (r >> b) & 1;
    const unsigned long long m = __ballot(set);
    same &= set ? m : ~m;
  }
  return same;
}
// Exclusive sum over the threads of a workgroup of kSortThreads (`sums`: one per wave); *all: the whole.
__device__ __forceinline__ int scan_threads(int x, int* sums, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int run = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int got = __shfl(run, (lane - off) & 63, 64);
    if (lane >= off) run += got;
  }
  if (lane == 63) sums[wave] = run;
  __syncthreads();
  int start = run - x, total = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    start += w < wave ? sums[w] : 0;
    total += sums[w];
  }
  *all = total;
  return start;
}

__global__ __launch_bounds__(kSortThreads) void embedding_deal_kernel(EmbedArgs a, int log_groups, int chunks) {
  __shared__ int place[kSortWaves][kMaxDealGroups];
  __shared__ int sums[kSortWaves];
  const int groups = 1 << log_groups, n = static_cast<int>(a.N), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kSortWaves * kMaxDealGroups; i += kSortThreads) place[0][i] = 0;
  // where this chunk's share of each group begins (a thread per group: groups <= threads)
  int before_me = 0, in_group = 0;
  if (tid < groups) {
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
      const int k = a.counts[static_cast<int64_t>(c) * groups + tid];
      in_group += k;
      before_me += c < static_cast<int>(blockIdx.x) ? k : 0;
    }
  }
  int all;
  const int start = scan_threads(in_group, sums, &all);
  if (blockIdx.x == 0) {
    if (tid < groups) a.group_start[tid] = start;
    if (tid == 0) a.group_start[groups] = all;
  }
  const int begin = static_cast<int>(blockIdx.x) * a.chunk + wave * (a.chunk / kSortWaves), end = min(n, begin + a.chunk / kSortWaves);
  int* const mine = place[wave];
  for (int p = begin + lane; p < end; p += 64) {
    const int64_t t = raw_token(a, p);
    if (live_token(a, t)) atomicAdd(&mine[static_cast<int>(t) & (groups - 1)], 1);
  }
  __syncthreads();
  if (tid < groups) {
    int at = start + before_me;
    for (int w = 0; w < kSortWaves; ++w) {
      const int k = place[w][tid];
      place[w][tid] = at;
      at += k;
    }
  }
  __syncthreads();
  const unsigned long long before = (1ull << lane) - 1ull;
  for (int base = begin; base < end; base += 64) {
    const int64_t t = base + lane < end ? raw_token(a, base + lane) : -1;
    const bool in = live_token(a, t);
    const int g = in ? static_cast<int>(t) & (groups - 1) : 0;
    const unsigned long long same = lanes_like(in, g, log_groups);
    const int at = in ? mine[g] : 0, rank = __popcll(same & before);
    if (in) {
      a.dealt_p[at + rank] = base + lane;
      a.dealt_t[at + rank] = static_cast<int>(t);
      if (rank == 0) mine[g] = at + __popcll(same);
    }
  }
}

// the gradient rows of a token that does not occur, by one wave
__device__ __forceinline__ void zero_row(const EmbedArgs& a, char* p, int64_t bytes, int lane) {
  if (bytes % 16 == 0) {
    const u32x4 z = {0u, 0u, 0u, 0u};
    if (a.stream_zeros)
      for (int64_t b = lane * 16; b < bytes; b += 1024) __builtin_nontemporal_store(z, reinterpret_cast<u32x4*>(p + b));
    else
      for (int64_t b = lane * 16; b < bytes; b += 1024) *reinterpret_cast<u32x4*>(p + b) = z;
  } else if (bytes % 4 == 0) {
    for (int64_t b = lane * 4; b < bytes; b += 256) *reinterpret_cast<uint32_t*>(p + b) = 0u;
  } else {
    for (int64_t b = lane * 2; b < bytes; b += 128) *reinterpret_cast<uint16_t*>(p + b) = 0;
  }
}
template <typename TW>
__device__ __forceinline__ void zero_token(const EmbedArgs& a, int64_t t, int lane) {
  const int64_t row_bytes = static_cast<int64_t>(a.D) * sizeof(TW);
  zero_row(a, static_cast<char*>(a.gw) + t * row_bytes, row_bytes, lane);
  if (a.grho) zero_row(a, reinterpret_cast<char*>(a.grho) + t * a.D * 4, static_cast<int64_t>(a.D) * 4, lane);
}

template <typename TW, bool DEALT>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(EmbedArgs a, int log_groups) {
  extern __shared__ int hist[];                     // [16][bucket] counts, then where the next one goes
  __shared__ int list_p[kSortWaves][kSortList];
  __shared__ uint16_t list_r[kSortWaves][kSortList];
  __shared__ int sums[kSortWaves], below[kSortWaves], totals[kMaxBucket];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int group = static_cast<int>(blockIdx.x), groups = 1 << log_groups;
  const int own = group < a.V ? (a.V - group + groups - 1) >> log_groups : 0;      // tokens of this workgroup
  for (int i = tid; i < kSortWaves * a.bucket; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  int* const mine = hist + wave * a.bucket;
  const int deal = DEALT ? group & ((1 << a.log_deal) - 1) : 0;
  const int first = DEALT ? a.group_start[deal] : 0, n = DEALT ? a.group_start[deal + 1] : static_cast<int>(a.N);
  const int chunk = ((n - first + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int begin = min(n, first + wave * chunk), end = min(n, begin + chunk);
  const unsigned long long before = (1ull << lane) - 1ull;
  constexpr int kAhead = 8;
  int64_t next[kAhead];
  int next_p[DEALT ? kAhead : 1];
  // f(which lanes hold a token of this workgroup, which one before it, the token's number here, the position), 64 positions at a time
  auto scan = [&](auto f) {
    auto fetch = [&](int base) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int p = base + 64 * u + lane;
        if constexpr (DEALT) {
          next[u] = p < end ? a.dealt_t[p] : -1;
          next_p[u] = p < end ? a.dealt_p[p] : 0;
        } else {
          next[u] = p < end ? raw_token(a, p) : -1;
        }
      }
    };
    fetch(begin);
    for (int base = begin; base < end; base += 64 * kAhead) {
      int64_t now[kAhead];
      int now_p[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        now[u] = next[u];
        now_p[u] = DEALT ? next_p[DEALT ? u : 0] : base + 64 * u + lane;
      }
      if (base + 64 * kAhead < end) fetch(base + 64 * kAhead);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const bool live = DEALT ? now[u] >= 0 : live_token(a, now[u]);
        const int t = static_cast<int>(now[u]), theirs = t & (groups - 1);
        f(live && theirs == group, live && theirs < group, t >> log_groups, now_p[u]);
      }
    }
  };
  int listed = 0, less = 0;
  bool fits = true;
  scan([&](bool in, bool ahead, int r, int p) {
    less += __popcll(__ballot(ahead));
    const unsigned long long m = __ballot(in);
    if (m == 0) return;
    const int k = __popcll(m);
    fits = fits && listed + k <= kSortList;
    if (in) {
      atomicAdd(&mine[r], 1);
      if (fits) {
        const int at = listed + __popcll(m & before);
        list_p[wave][at] = p;
        list_r[wave][at] = static_cast<uint16_t>(r);
      }
    }
    listed += k;
  });
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // per token: its total, the exclusive sum over the tokens of the workgroup, then each wave's share behind the ones before it
  int total = 0;
  if (tid < own)
    for (int w = 0; w < kSortWaves; ++w) total += hist[w * a.bucket + tid];
  if (tid < own) totals[tid] = total;
  int all;
  int start = first + scan_threads(total, sums, &all);
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    start += below[w];
    all += below[w];
  }
  if (tid < own) {
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = hist[w * a.bucket + tid];
      hist[w * a.bucket + tid] = start;
      start += c;
    }
  }
  if (tid == 0 && group == groups - 1) a.header[0] = DEALT ? a.group_start[1 << a.log_deal] : all;
  __syncthreads();
  // positions in order: lanes of one token take consecutive places
  const int bits = 32 - __builtin_clz(a.bucket | 1);
  auto place = [&](bool in, int r, int p) {
    const unsigned long long same = lanes_like(in, r, bits);
    const int at = in ? mine[r] : 0, rank = __popcll(same & before);
    if (in) {
      a.order[at + rank] = p;
      a.key[at + rank] = (r << log_groups) + group;
      if (rank == 0) mine[r] = at + __popcll(same);
    }
  };
  auto place_list = [&](int n_listed) {
    for (int base = 0; base < n_listed; base += 64) {
      const bool in = base + lane < n_listed;
      place(in, in ? list_r[wave][base + lane] : 0, in ? list_p[wave][base + lane] : 0);
    }
  };
  if (!fits) {                    // the matches again, a list at a time
    listed = 0;
    scan([&](bool in, bool, int r, int p) {
      const unsigned long long m = __ballot(in);
      if (m == 0) return;
      const int k = __popcll(m);
      if (listed + k > kSortList) {
        place_list(listed);
        listed = 0;
      }
      if (in) {
        const int at = listed + __popcll(m & before);
        list_p[wave][at] = p;
        list_r[wave][at] = static_cast<uint16_t>(r);
      }
      listed += k;
    });
  }
  place_list(listed);
  for (int r = wave; r < own; r += kSortWaves)
    if (!totals[r]) zero_token<TW>(a, (static_cast<int64_t>(r) << log_groups) + group, lane);
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

constexpr int kJoinBlock = 512;
// One workgroup per (piece, 64 * VEC columns): if a run begins in this piece and goes on behind it, add its parts.  The
// eight waves take every eighth part; their sums are added in order.
template <typename TW, int NOISE, int VEC>
__global__ __launch_bounds__(kJoinBlock) void embedding_join_kernel(EmbedArgs a, int column_tiles) {
  constexpr int NACC = NOISE == kNoisePosition ? 2 : 1, kWaves = kJoinBlock / 64;
  __shared__ float sums[kWaves - 1][NACC][64 * VEC];
  const int id = a.join0 + static_cast<int>(blockIdx.x), piece = id / column_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = (id % column_tiles) * 64 * VEC + lane * VEC;
  const int n = a.header[0], s0 = piece * a.piece, s1 = s0 + a.piece;
  if (s1 >= n) return;
  const int key = a.key[s1 - 1];
  if (a.key[s1] != key || (s0 > 0 && a.key[s0 - 1] == key)) return;     // (a token's positions are side by side: equal ends mean equal in between)
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

// ---- few positions: the whole gradient in ONE launch
// Workgroup b owns the tokens it owns in the sort; it collects its positions in LDS as (token, position), ranks them by counting
// and adds the rows in that order: eight waves take consecutive pieces of the list, the parts of runs that cross pieces are
// added in order.  Nothing passes through memory, and the host, which bounds calls this small, launches once.
// What bounds the kernel are its zero rows, or one workgroup that owns most positions and reads most of g alone -- hence the
// limits.  Positions by word frequency / half of them one token / all of them, against the several launches: 64 x 256 bf16,
// 1,000 tokens 3.8 / 5.7 / 6.6 us against 11.9 / 11.9 / 11.1; 512 x 256 6.3 / 13.9 / 25.3 against 13.1 / 13.8 / 12.8; 512 x 256
// fp32, 30,011 tokens 9.5 / 19.8 / 31.7 against 16.2 / 17.2 / 15.5; beyond: 512 x 1,024 27 / 66 / 105 against 28 / 28 / 27.
constexpr int kSmallTokens = 512, kSmallThreads = 512, kSmallWaves = kSmallThreads / 64;
constexpr int64_t kSmallElements = 128 << 10;
static bool embedding_small(int64_t n, int64_t d) { return n <= kSmallTokens && n * d <= kSmallElements; }

template <typename TW, typename TG, int NOISE, int VEC>
__global__ __launch_bounds__(kSmallThreads) void embedding_small_kernel(EmbedArgs a, int log_groups) {
  constexpr int NACC = NOISE == kNoisePosition ? 2 : 1, kAhead = 8;
  static_assert(kSmallTokens <= kSmallThreads && kSmallTokens <= 1 << 10 && kSmallTokens % 16 == 0, "a thread per position; ten bits of an entry");
  __shared__ __attribute__((aligned(16))) uint32_t found[kSmallTokens], list[kSmallTokens];
  __shared__ uint32_t seen[kMaxBucket / 32];
  __shared__ float part[kSmallWaves][2][NACC][64 * VEC];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = static_cast<int>(blockIdx.x), groups = 1 << log_groups, n = static_cast<int>(a.N);
  const int own = group < a.V ? (a.V - group + groups - 1) >> log_groups : 0;
  const int64_t raw = tid < n ? raw_token(a, tid) : -1;
  if (tid < kMaxBucket / 32) seen[tid] = 0u;
  if (tid < kSmallTokens) found[tid] = ~0u;
  if (tid == 0) count = 0;
  __syncthreads();
  const int t = static_cast<int>(raw);
  if (live_token(a, raw) && (t & (groups - 1)) == group) {
    const int r = t >> log_groups;
    found[atomicAdd(&count, 1)] = static_cast<uint32_t>(r) << 10 | static_cast<uint32_t>(tid);
    atomicOr(&seen[r >> 5], 1u << (r & 31));
  }
  __syncthreads();
  const int m = __builtin_amdgcn_readfirstlane(count);
  if (tid < m) {
    const uint32_t mine = found[tid];                   // (the entries are all different, what is behind them is larger)
    int rank = 0;
    for (int j = 0; j < m; j += 16) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(found + j + 4 * q);
#pragma unroll
        for (int k = 0; k < 4; ++k) rank += x[k] < mine ? 1 : 0;
      }
    }
    list[rank] = mine;
  }
  __syncthreads();
  auto entry_token = [](int entry) { return static_cast<int>(static_cast<uint32_t>(entry) >> 10); };
  auto token = [&](int i) { return __builtin_amdgcn_readfirstlane(i >= 0 && i < m ? entry_token(static_cast<int>(list[i])) : -1); };
  float acc[VEC], acc2[VEC];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = acc2[i] = 0.0f;
  };
  const int tiles = (a.D + 64 * VEC - 1) / (64 * VEC);
  const bool alone = m <= kAhead;                        // one piece: the waves take the columns
  const int piece = max(kAhead, (m + kSmallWaves - 1) / kSmallWaves);
  const int begin = alone ? 0 : min(m, wave * piece), end = min(m, begin + piece);
  for (int c = alone ? wave : 0; c < tiles; c += alone ? kSmallWaves : 1) {
    const int d = c * 64 * VEC + lane * VEC;
    const bool active = d < a.D;
    // entries [begin, end) of the list: finished runs are stored, the parts of others kept
    clear();
    int run_begin = begin;
    const int before = token(begin - 1);
    for (int s = begin; s < end; s += kAhead) {
      const uint32_t mine = lane <= kAhead && s + lane < m ? list[s + lane] : ~0u;      // (one more: the entry behind)
      float g[kAhead][VEC], e[NACC == 2 ? kAhead : 1][VEC];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u < end) {
          const int64_t pos = __builtin_amdgcn_readlane(static_cast<int>(mine), u) & 1023;
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
        if (s + u < end) {
          const int r = entry_token(__builtin_amdgcn_readlane(static_cast<int>(mine), u));
          const int next = entry_token(__builtin_amdgcn_readlane(static_cast<int>(mine), u + 1));
          if (active) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              acc[i] += g[u][i];
              if constexpr (NACC == 2) acc2[i] = __builtin_fmaf(g[u][i], e[u][i], acc2[i]);
            }
          }
          if (next != r || s + u + 1 == end) {
            const bool begun_before = run_begin == begin && before == r;
            if (begun_before || next == r) {
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                part[wave][begun_before ? 0 : 1][0][i * 64 + lane] = acc[i];
                if constexpr (NACC == 2) part[wave][begun_before ? 0 : 1][NACC - 1][i * 64 + lane] = acc2[i];
              }
            } else if (active) {
              embedding_finish<TW, NOISE, VEC>(a, (r << log_groups) + group, d, acc, acc2);
            }
            clear();
            run_begin = s + u + 1;
          }
        }
      }
    }
    if (alone) continue;
    __syncthreads();
    // the wave in whose piece a run begins that goes on behind it
    const int r = token(end - 1);
    if (begin < end && end < m && token(end) == r && (begin == 0 || token(begin - 1) != r || token(begin) != r)) {
      clear();
      for (int w = wave; w < kSmallWaves && w * piece < m && (w == wave || token(w * piece) == r); ++w)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          acc[i] += part[w][w == wave ? 1 : 0][0][i * 64 + lane];
          if constexpr (NACC == 2) acc2[i] += part[w][w == wave ? 1 : 0][NACC - 1][i * 64 + lane];
        }
      if (active) embedding_finish<TW, NOISE, VEC>(a, (r << log_groups) + group, d, acc, acc2);
    }
    __syncthreads();
  }
  for (int r = wave; r < own; r += kSmallWaves)
    if (!((seen[r >> 5] >> (r & 31)) & 1u)) zero_token<TW>(a, (static_cast<int64_t>(r) << log_groups) + group, lane);
}

constexpr int64_t kDealTokens = 49152;
// positions per workgroup of the dealing kernels (0: no dealing): at most 256 chunks, whole waves of 64 positions
static int embedding_chunk(int64_t n) {
  if (n < kDealTokens) return 0;
  const int64_t chunk = std::max<int64_t>(4096, (n + 255) / 256);
  return static_cast<int>((chunk + 1023) / 1024 * 1024);
}
// When the table's gradient and what is read beside it are well beyond the 256 MB memory-side cache, zero rows that stay in it are
// pushed out again by the rows that the sums read: 65,536 tokens, 131,072 x 1,024 bf16, 131 us against 105 us past the caches (512
// tokens: 54 against 62; 92 MB of zero rows: 28 against 30).
constexpr int64_t kStreamZeros = 320 << 20;

// positions per piece: short pieces keep enough waves in flight when there are few tokens (4,800 x 768 Gaussian: sums 13.9 us with
// 8, 17.7 with 16, 51 with 64), long ones leave fewer parts to join (1,048,576 tokens: 41 us with 64, 138 with 16)
static int embedding_piece(int64_t n) { return n <= 8192 ? 8 : n <= 32768 ? 16 : n <= 65536 ? 32 : 64; }

constexpr int64_t kFwdManyRows = 16384;

template <typename TW, typename TO, int NOISE, int VEC>
static int embedding_fwd_launch(const EmbedArgs& a, hipStream_t s) {
  const int vecs = (a.D + VEC - 1) / VEC;
  int log_lanes = 3;
  while (log_lanes < 6 && (1 << log_lanes) < vecs) ++log_lanes;
  auto go = [&](auto kernel, int rows) {
    const int64_t blocks = ((((a.N + rows - 1) / rows) << log_lanes) + kBlock - 1) / kBlock;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, a, log_lanes);
    return to_err(hipGetLastError());
  };
  if (a.N >= kFwdManyRows) return go(&embedding_fwd_kernel<TW, TO, NOISE, VEC, 4>, 4);
  return go(&embedding_fwd_kernel<TW, TO, NOISE, VEC, 1>, 1);
}
constexpr int kJoinsPerLaunch = 1 << 19;       // (a launch holds fewer than 2^32 threads)
template <typename TW, typename TG, int NOISE, int VEC>
static int embedding_bwd_launch(EmbedArgs a, hipStream_t s) {
  const dim3 groups(1u << a.log_groups);
  if (embedding_small(a.N, a.D)) {
    hipLaunchKernelGGL((embedding_small_kernel<TW, TG, NOISE, VEC>), groups, dim3(kSmallThreads), 0, s, a, a.log_groups);
    return to_err(hipGetLastError());
  }
  const size_t lds = sizeof(int) * kSortWaves * a.bucket;
  if (a.chunk > 0) {
    const int chunks = static_cast<int>((a.N + a.chunk - 1) / a.chunk);
    hipLaunchKernelGGL(embedding_count_kernel, dim3(chunks), dim3(kSortThreads), 0, s, a, a.log_deal);
    if (const int rc = to_err(hipGetLastError())) return rc;
    hipLaunchKernelGGL(embedding_deal_kernel, dim3(chunks), dim3(kSortThreads), 0, s, a, a.log_deal, chunks);
    if (const int rc = to_err(hipGetLastError())) return rc;
    hipLaunchKernelGGL((embedding_sort_kernel<TW, true>), groups, dim3(kSortThreads), lds, s, a, a.log_groups);
  } else {
    hipLaunchKernelGGL((embedding_sort_kernel<TW, false>), groups, dim3(kSortThreads), lds, s, a, a.log_groups);
  }
  if (const int rc = to_err(hipGetLastError())) return rc;
  const int tiles = (a.D + 64 * VEC - 1) / (64 * VEC), pieces = static_cast<int>((a.N + a.piece - 1) / a.piece);
  const int64_t all = static_cast<int64_t>(pieces) * tiles;
  hipLaunchKernelGGL((embedding_sum_kernel<TW, TG, NOISE, VEC>), dim3(static_cast<unsigned>((all + kBlock / 64 - 1) / (kBlock / 64))), dim3(kBlock), 0, s,
                     a, tiles);
  if (const int rc = to_err(hipGetLastError())) return rc;
  for (int64_t first = 0; pieces > 1 && first < all; first += kJoinsPerLaunch) {
    a.join0 = static_cast<int>(first);
    const unsigned joins = static_cast<unsigned>(std::min<int64_t>(kJoinsPerLaunch, all - first));
    hipLaunchKernelGGL((embedding_join_kernel<TW, NOISE, VEC>), dim3(joins), dim3(kJoinBlock), 0, s, a, tiles);
    if (const int rc = to_err(hipGetLastError())) return rc;
  }
  return 0;
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

constexpr int64_t kDealBytes = 4 * (256 * kMaxDealGroups + kMaxDealGroups + 64);      // counts and group starts

extern "C" size_t bde_embedding_bwd_ws_bytes(int64_t N, int64_t D, int noise) {
  if (N < 0 || N > BDE_EMBEDDING_MAX_TOKENS || D < 1 || D > BDE_EMBEDDING_MAX_DIM) return 0;
  if (embedding_small(N, D)) return 256;      // (not used)
  const int64_t list = (4 * N + 255) / 256 * 256;
  const int64_t lists = 256 + 2 * list + (embedding_chunk(N) > 0 ? 2 * list + kDealBytes : 0);
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
  // 256 workgroups (one per CU), or as many as keep a workgroup's counts in LDS; no more than tokens
  a.log_groups = 8;
  while ((V + (1 << a.log_groups) - 1) >> a.log_groups > kMaxBucket) ++a.log_groups;
  while (a.log_groups > 0 && (int64_t{1} << (a.log_groups - 1)) >= V) --a.log_groups;
  a.bucket = static_cast<int>((V + (1 << a.log_groups) - 1) >> a.log_groups);
  char* rest = base + 256 + 2 * list;
  if (embedding_chunk(N) > 0) {
    a.chunk = embedding_chunk(N);
    while (a.log_deal < a.log_groups && (2 << a.log_deal) <= kMaxDealGroups) ++a.log_deal;
    a.counts = reinterpret_cast<int*>(rest);
    a.group_start = a.counts + 256 * kMaxDealGroups;
    a.dealt_p = reinterpret_cast<int*>(rest + kDealBytes);
    a.dealt_t = reinterpret_cast<int*>(rest + kDealBytes + list);
    rest += kDealBytes + 2 * list;
  }
  a.part = reinterpret_cast<float*>(rest);
  a.piece = embedding_piece(N);
  a.stream_zeros = V * D * static_cast<int64_t>(dtype_bytes(weight_dtype) + (g_rho ? 4 : 0)) +
                       N * D * static_cast<int64_t>(dtype_bytes(g_dtype) + (noise == kNoisePosition && eps ? 4 : 0)) > kStreamZeros;
  return embedding_dispatch<true>(a, weight_dtype, g_dtype, noise, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("hidden"))) int bde_internal_load_embedding(void) {
  hipFuncAttributes attr;
  return to_err(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&embedding_sort_kernel<float, false>)));
}
