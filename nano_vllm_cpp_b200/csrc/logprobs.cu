// Log probabilities of given tokens, with the distribution's entropy, the tokens' ranks and the best alternatives.
//
//   m = max x,  Z = sum e^(x - m),  logprob(t) = x_t - m - log Z,  entropy = log Z - sum e^(x - m) (x - m) / Z
//
// What bounds it: the logits, read once.  2,048 rows of 151,936 float32 take 184 us, 6.8 TB/s, in a run of calls with the same logits
// and 216, 5.8 TB/s, with others in between (226 with five alternatives each, in a run); a handful of rows takes the latency of a launch, of a tile or two and of the cluster's exchange: one row 5.3 us, with five
// alternatives 9.4.
//
// One pass keeps m, n1 (how many logits equal m), s (the sum of the others' e^(x - m)) and e (the sum of e^(x - m) (x - m)):
// log Z = log n1 + log1p(s / n1).  The largest term is never added to the small ones, so the logarithm of an all but certain
// token's probability, -s, keeps its bits instead of being what 1 + s rounds to.
//
// The order of the alternatives and of the ranks is that of (logit descending, id ascending), the greedy choice first; a NaN
// comes after everything else.  A row that holds a NaN or plus infinity, or nothing above minus infinity, has no softmax: its
// numbers are NaN, its order is defined all the same.
#include "common.cuh"

#include <cfloat>

namespace {

// A float as an integer of the same order: NaN lowest, minus zero equal to zero.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// ... and with the id as the second criterion, lower ids first.  (No key is zero.)
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int id) { return ((Key)order_of(x) << 32) | (uint32_t)(0x7fffffff - id); }
__device__ __forceinline__ int id_of(Key key) { return 0x7fffffff - (int)(uint32_t)key; }
__device__ __forceinline__ float float_of(uint32_t order) {
  return order == 0u ? NAN : __uint_as_float((order & 0x80000000u) ? (order & 0x7fffffffu) : ~order);
}
// The next number below (minus zero, which equals zero, is none of its own).
__device__ __forceinline__ float below_of(uint32_t order) { return float_of(order == 0x80000000u ? 0x7ffffffeu : order - 1); }
__device__ __forceinline__ float max_nan(float a, float b) {       // (fmaxf drops a NaN)
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Stats {
  float m, n1, s, e;
};
// The sums of a warp's lanes, each against its own maximum, against the largest of them; every lane gets them.
__device__ __forceinline__ Stats join(const Stats& a) {
  Stats r;
  r.m = warp_max(a.m);
  const bool mine = a.m == r.m;
  const float d = a.m - r.m, c = mine ? 1.f : expf(d), all = a.n1 + a.s;
  r.n1 = warp_sum(mine ? a.n1 : 0.f);
  r.s = warp_sum(mine ? a.s : c * all);                      // (c is zero where nothing was there; a NaN in `all` stays)
  r.e = warp_sum(mine ? a.e : c > 0.f ? c * (a.e + d * all) : 0.f);
  return r;
}

struct LpArgs {
  const void* logits;
  long long stride;
  const int* tokens;
  float* logprob;
  float* entropy;
  int* rank;
  int* top_ids;
  float* top_logprobs;
  int* err;
  int R, V, K;
};

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int LP_E = 16;               // elements a thread takes at a time: four (bfloat16: two) 16-byte pieces
constexpr int LP_STAGES = 4;           // tiles under way: a thread copies its own pieces into shared memory, three tiles ahead
constexpr int MAX_CLUSTER = 16;        // blocks a row
constexpr int LP_LIST = 512;           // candidates a block has room for
constexpr int LP_LONG = 256;           // ... and from how many on they are thinned out to the best K
constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
struct Vec;                            // a 16-byte piece as floats
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void read(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
};
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void read(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// The blocks of a cluster leave what they have with the first one: its copy of a shared variable, as they address it.
__device__ __forceinline__ uint32_t of_first(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)));
  return a;
}
__device__ __forceinline__ void put_first(uint32_t a, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ void put_first(uint32_t a, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void put_first(uint32_t a, Key v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }

// The K largest of the n keys in list[] come to its front and to best[], in descending order (fewer keys: zeros behind them); every
// thread of the block calls, between two barriers.  A key's place is the number of larger ones.
__device__ void keep_best(Key* list, int n, int K, Key* best) {
  const int tid = threadIdx.x;
  if (tid < K) best[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += THREADS) {
    const Key k = list[i];
    int place = 0, j = 0;
    for (; j + 8 <= n; j += 8) {
      Key other[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) other[u] = list[j + u];
#pragma unroll
      for (int u = 0; u < 8; ++u) place += other[u] > k;
    }
    for (; j < n; ++j) place += list[j] > k;
    if (place < K) best[place] = k;
  }
  __syncthreads();
  if (tid < K) list[tid] = best[tid];
  __syncthreads();
}

// One after the other in runs of a warp's width, whatever the logits are: for rows whose bound let too many candidates through
// (rising ones) or too few (fewer than K logits above minus infinity).
template <typename T>
__device__ void collect_slowly(const T* x, int i0, int i1, int K, Key* list, Key* best, int* n_s) {
  constexpr int RUN = THREADS < LP_LIST - LP_LONG ? THREADS : LP_LIST - LP_LONG;
  Key bound = 0;
  __syncthreads();
  if (threadIdx.x == 0) *n_s = 0;
  __syncthreads();
  for (int i = i0; i < i1; i += RUN) {
    if (threadIdx.x < RUN && i + (int)threadIdx.x < i1) {
      const Key k = key_of(to_f32(x[i + threadIdx.x]), i + threadIdx.x);
      if (k > bound) list[atomicAdd(n_s, 1)] = k;
    }
    __syncthreads();
    const int n = *n_s;
    if (n > LP_LONG) {
      keep_best(list, n, K, best);
      bound = list[K - 1];
      if (threadIdx.x == 0) *n_s = K;
    }
    __syncthreads();
  }
}

// A cluster of blocks takes a row, each block a run of its 16-byte pieces; a warp has a maximum, its threads their sums, which are
// rescaled when it moves.  Alternatives: the first tile gives a bound that at least K of its logits reach (the K-th largest among
// every full warp's few largest thread maxima), what lies above it goes into a list, and behind 2, 4, 8 ... tiles the list is thinned
// out to its K best, which raises the bound.  Every block leaves its
// warps' sums and its list with the first one of the cluster, which joins them.
// TOP: with alternatives (K > 0).
template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 3 : 4) token_logprobs_kernel(LpArgs a) {
  constexpr int N = Vec<T>::N, NV = LP_E / N, TILE = THREADS * NV;     // (a tile in pieces)
  extern __shared__ __align__(16) uint4 ring[];                       // [LP_STAGES][NV][THREADS], and behind them:
  __shared__ Key list_s[LP_LIST];
  __shared__ Key best_s[32];
  __shared__ uint32_t most_s[64];
  __shared__ int n_s;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int cluster = (int)gridDim.x / a.R, row = blockIdx.x / cluster, part = blockIdx.x % cluster;
  // what every warp and block of the cluster has, in the first one (join_bytes)
  Stats* const all_s = (Stats*)(ring + LP_STAGES * TILE);             // [cluster * WARPS]
  Key* const join_s = (Key*)(all_s + cluster * WARPS);                // [cluster * K]
  int* const ahead_s = (int*)(join_s + cluster * a.K);                // [cluster * WARPS]
  if (tid == 0) n_s = 0;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");        // (this block runs)
  grid_dep_wait();
  grid_dep_launch();
  const T* x = (const T*)a.logits + (long long)row * a.stride;
  const int token = a.tokens ? a.tokens[row] : -1;
  const int off = (int)(((uintptr_t)x / sizeof(T)) % N);              // elements between the 16-byte boundary below and the row
  const int pieces = (int)(((long long)a.V + off + N - 1) / N), per = (pieces + cluster - 1) / cluster;
  const int q0 = min(pieces, part * per), q1 = min(pieces, q0 + per);
  Stats st = {-INFINITY, 0.f, 0.f, 0.f};
  uint32_t m_order = 0x007fffffu;                                     // st.m's (minus infinity's)
  int ahead = 0, tile = 0;
  float above = -INFINITY;                                            // candidates are above it
  bool bounded = false, lost = false;
  auto fetch = [&](int t) {                                            // tile t's whole pieces
    const int q = q0 + t * TILE;
    uint4* to = ring + (t % LP_STAGES) * TILE + tid;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int p = q + j * THREADS + tid, i0 = p * N - off;
      if (p < q1 && i0 >= 0 && i0 + N <= a.V)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to + j * THREADS)), "l"(x + i0) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < LP_STAGES - 1; ++t) fetch(t);
  // the given token: its logit arrives while the first tile does
  const bool known = token >= 0 && token < a.V, ranked = known && a.rank;
  const float xt = known ? to_f32(x[token]) : 0.f;
  const bool by_key = !(xt > -INFINITY);
  const uint32_t xt_order = order_of(xt);
  const float xt_below = below_of(xt_order);
  for (int q = q0; q < q1; q += TILE, ++tile) {
    asm volatile("cp.async.wait_group %0;" ::"n"(LP_STAGES - 2) : "memory");
    float v[LP_E];
    const uint4* from = ring + (tile % LP_STAGES) * TILE + tid;
    const bool whole = q * N >= off && q + TILE <= q1 && (long long)(q + TILE) * N - off <= a.V;
#pragma unroll
    for (int j = 0; j < NV; ++j) Vec<T>::read(from[j * THREADS], v + j * N);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int p = q + j * THREADS + tid, i0 = p * N - off;
        if (!(p < q1 && i0 >= 0 && i0 + N <= a.V)) {                  // a piece that the row covers a part of, or nothing
#pragma unroll
          for (int u = 0; u < N; ++u) v[j * N + u] = (p < q1 && i0 + u >= 0 && i0 + u < a.V) ? to_f32(x[i0 + u]) : -INFINITY;
        }
      }
    }
    fetch(tile + LP_STAGES - 1);                                      // (into the stage that was read a tile ago)
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < LP_E; ++i) mx = fmaxf(mx, v[i]);
    const uint32_t top = order_of(mx), tile_top = __reduce_max_sync(0xffffffffu, top);
    if (ranked && (by_key || tile_top >= xt_order)) {                  // (else nothing of the tile is ahead of the token)
      const int lowest = q * N - off;
      if (by_key || (lowest <= token && lowest + TILE * N > token)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int p = q + j * THREADS + tid, i0 = p * N - off;
#pragma unroll
          for (int u = 0; u < N; ++u)
            ahead += i0 + u >= 0 && i0 + u < a.V && p < q1 && key_of(v[j * N + u], i0 + u) > key_of(xt, token);
        }
      } else {
        const float over = lowest < token ? xt_below : xt;            // equal logits of lower ids are ahead
#pragma unroll
        for (int i = 0; i < LP_E; ++i) ahead += v[i] > over;
      }
    }
    if (TOP && !lost) {
      const int full = min(WARPS, (q1 - q) / 32);                     // warps all of whose threads have elements
      if (!bounded && full > 0) {
        const int each = min(32, min((a.K + full - 1) / full + 1, 64 / full));       // (K <= 32: enough, with one to spare where there is room)
        uint32_t o = mx > -INFINITY ? top : 0u;
        for (int j = 0; j < each; ++j) {
          const uint32_t most = __reduce_max_sync(0xffffffffu, o);
          const uint32_t who = __ballot_sync(0xffffffffu, o == most);
          if (lane == __ffs(who) - 1) o = 0u;
          if (lane == 0 && warp < full) most_s[warp * each + j] = most;
        }
        __syncthreads();
        // the K-th largest of these (at least K: `each` from every full warp); equal ones in their order
        const int n = full * each;
        uint32_t kth = 0u;
        for (int i = lane; i < n; i += 32) {
          const uint32_t w = most_s[i];
          int place = 0;
          for (int j = 0; j < n; ++j) place += most_s[j] > w || (most_s[j] == w && j < i);
          if (place == a.K - 1) kth = w;
        }
        kth = __reduce_max_sync(0xffffffffu, kth);
        if (kth > 0u) {
          above = below_of(kth);
          bounded = true;
        }
        __syncthreads();
      }
      if (float_of(tile_top) > above) {
        if (mx > above) {
#pragma unroll
          for (int i = 0; i < LP_E; ++i)
            if (v[i] > above) {
              const int at = atomicAdd(&n_s, 1);
              if (at < LP_LIST) list_s[at] = key_of(v[i], (q + i / N * THREADS + tid) * N - off + i % N);
            }
        }
      }
      if (tile > 0 && (tile & (tile + 1)) == 0) {                     // behind 2, 4, 8 ... tiles: as many again add some K
        __syncthreads();
        const int n = n_s;
        __syncthreads();
        lost = n > LP_LIST;                                           // (collected again at the end)
        if (n > a.K && !lost) {
          keep_best(list_s, n, a.K, best_s);
          above = float_of((uint32_t)(list_s[a.K - 1] >> 32));        // (equal logits from here on have higher ids)
          bounded = true;
          if (tid == 0) n_s = a.K;
          __syncthreads();
        }
      }
    }
    // all threads of a warp keep their sums against one m; most tiles do not reach it
    if (tile_top >= m_order) {
      if (tile_top > m_order) {
        m_order = tile_top;
        const float m = float_of(tile_top), d = st.m - m, c = ex2_fast(d * LOG2E), all = st.n1 + st.s;
        st.e = c > 0.f ? c * fmaf(d, all, st.e) : 0.f;
        st.s = c * all;                                               // (zero where nothing was there; a NaN stays)
        st.n1 = 0.f;
        st.m = m;
      }
#pragma unroll
      for (int i = 0; i < LP_E; ++i) {                                // the largest are counted and leave the sums
        const bool largest = v[i] == st.m;
        st.n1 += largest ? 1.f : 0.f;
        v[i] = largest ? -INFINITY : v[i];
      }
    }
    const float m = fmaxf(st.m, -FLT_MAX);                            // (nothing but NaN and minus infinity so far)
    float2 sum = make_float2(st.s, 0.f), by = make_float2(st.e, 0.f);
    const float2 m2 = make_float2(-m, -m), scale = make_float2(LOG2E, LOG2E);
#pragma unroll
    for (int i = 0; i < LP_E; i += 2) {                               // two elements an instruction
      float2 d = add2(make_float2(v[i], v[i + 1]), m2);
      d.x = max_nan(d.x, -150.f);
      d.y = max_nan(d.y, -150.f);
      const float2 t = mul2(d, scale), e = make_float2(ex2_fast(t.x), ex2_fast(t.y));
      sum = add2(sum, e);
      by = fma2(e, d, by);
    }
    st.s = sum.x + sum.y;
    st.e = by.x + by.y;
  }
  const int first = max(0, q0 * N - off), last = min(a.V, q1 * N - off);          // this block's elements
  if (TOP) {
    __syncthreads();
    const int n = n_s;
    if (n > LP_LIST || n < min(a.K, last - first)) collect_slowly<T>(x, first, last, a.K, list_s, best_s, &n_s);
    keep_best(list_s, n_s, a.K, best_s);
  }
  st.n1 = warp_sum(st.n1);
  st.s = warp_sum(st.s);
  st.e = warp_sum(st.e);
  if (ranked) ahead = __reduce_add_sync(0xffffffffu, ahead);
  if (cluster > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");                 // (the first block runs)
  if (cluster > 1) {
    if (lane == 0) {
      const uint32_t to = of_first(&all_s[part * WARPS + warp]);
      put_first(to, st.m);
      put_first(to + 4, st.n1);
      put_first(to + 8, st.s);
      put_first(to + 12, st.e);
      put_first(of_first(&ahead_s[part * WARPS + warp]), ahead);
    }
    if (TOP && tid < a.K) put_first(of_first(&join_s[part * a.K + tid]), best_s[tid]);
  } else if (lane == 0) {
    all_s[warp] = st;
    ahead_s[warp] = ahead;
  }
  if (cluster > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (part != 0) return;                                            // (nobody reads from this block)
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (TOP && cluster > 1) keep_best(join_s, cluster * a.K, a.K, best_s);
  if (warp != 0) return;
  const Stats none = {-INFINITY, 0.f, 0.f, 0.f};
  st = none;
  ahead = 0;
  for (int i = lane; i < cluster * WARPS; i += 32) {                  // at most four of a lane's own, then the lanes'
    const Stats other = all_s[i], hi = st.m >= other.m ? st : other, lo = st.m >= other.m ? other : st;
    const bool same = hi.m == lo.m;
    const float d = lo.m - hi.m, c = same ? 1.f : expf(d), all = lo.n1 + lo.s;
    st.m = hi.m;
    st.n1 = hi.n1 + (same ? lo.n1 : 0.f);
    st.s = hi.s + (same ? lo.s : c * all);
    st.e = hi.e + (same ? lo.e : c > 0.f ? c * (lo.e + d * all) : 0.f);
    ahead += ahead_s[i];
  }
  st = join(st);
  ahead = __reduce_add_sync(0xffffffffu, ahead);
  const bool proper = fabsf(st.m) < INFINITY;
  const float log_z = proper ? logf(st.n1) + log1pf(st.s / st.n1) : NAN;
  if (lane == 0) {
    if (a.tokens) {
      if (!known && a.err) atomicExch(a.err, 1 + row);
      if (a.logprob) a.logprob[row] = known ? (xt - st.m) - log_z : NAN;
      if (a.rank) a.rank[row] = known ? ahead : -1;
    }
    if (a.entropy) a.entropy[row] = log_z - st.e / (st.n1 + st.s);
  }
  if (TOP && lane < a.K) {
    const Key k = best_s[lane];
    a.top_ids[(long long)row * a.K + lane] = id_of(k);
    a.top_logprobs[(long long)row * a.K + lane] = (float_of((uint32_t)(k >> 32)) - st.m) - log_z;
  }
}

constexpr size_t join_bytes(int cluster, int K) { return (size_t)cluster * (WARPS * (sizeof(Stats) + sizeof(int)) + K * sizeof(Key)); }

// Blocks a row: a cluster of them while that leaves two or so a multiprocessor, each with half a tile at least.  On 1 / 2 / 4 / 8 /
// 16 blocks: one row of 151,936 logits, five alternatives, 29.8 / 19.7 / 15.0 / 11.1 / 9.4 us; 32 rows 31.5 / 21.9 / 17.0 / 16.9 /
// 20.6; 64 rows, twenty, 37.9 / 26.7 / 22.6 / 33.6; 150 rows, five, 39.2 / 34.2 / 40.2; 2,048 rows 226 / 276 / 380.
template <typename T, bool TOP>
int run_logprobs(const LpArgs& a, cudaStream_t s) {
  constexpr size_t ring = (size_t)LP_STAGES * THREADS * LP_E * sizeof(T), most = ring + join_bytes(MAX_CLUSTER, 32) > 80 * 1024 ? ring + join_bytes(MAX_CLUSTER, 32) : 80 * 1024;
  static bool attr_done = false;
  if (!attr_done) {
    NV_RETURN_IF(cudaFuncSetAttribute(token_logprobs_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    NV_RETURN_IF(cudaFuncSetAttribute(token_logprobs_kernel<T, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_done = true;
  }
  const long long sms = num_multiprocessors();
  unsigned cluster = 1;
  while (cluster < MAX_CLUSTER && a.R * (long long)cluster * 8 <= sms * 9 && a.V / (int)(2 * cluster) >= THREADS * LP_E / 2) cluster *= 2;
  // Two blocks a multiprocessor at most ask for more than a third of its memory, so that three do not share one while others
  // have none (64 rows, twenty alternatives: 27.5 and 22.6 us).  Larger clusters have too few places then (32 rows: 16.9 and 19.0).
  size_t smem = ring + join_bytes(cluster, a.K);
  if (cluster <= 4 && a.R * (long long)cluster <= 2 * sms && smem < 80 * 1024) smem = 80 * 1024;
  NV_RETURN_IF(launch_dep_clusters(cluster, token_logprobs_kernel<T, TOP>, dim3(a.R * cluster), dim3(THREADS), smem, s, a));
  NV_RETURN_LAST();
}

}  // namespace

NV_API int nv_token_logprobs_max_top(void) { return 32; }

// logits: R rows of V, `stride` elements apart.  tokens [R] or nullptr (then no logprob and no rank); logprob, entropy
// [R] float32, rank [R] int32: any may be nullptr; top_ids, top_logprobs [R, K] (K = 0: neither).  A token outside the vocabulary
// sets the error flag to 1 + its row and gets NaN and the rank -1.
NV_API int nv_token_logprobs(const void* logits, int dt, long long stride, int R, int V, const int* tokens, float* logprob,
                             float* entropy, int* rank, int K, int* top_ids, float* top_logprobs, int* err, cudaStream_t s) {
  if (!dt_ok(dt)) return NV_ERR_BAD_DTYPE;
  if (R < 0 || V < 1 || V > 1 << 30 || stride < V || K < 0 || K > V || K > nv_token_logprobs_max_top()) return NV_ERR_BAD_SIZE;
  if (K > 0 && (!top_ids || !top_logprobs)) return NV_ERR_BAD_SIZE;
  if (R == 0) return NV_OK;
  const LpArgs a = {logits, stride, tokens, logprob, entropy, rank, top_ids, top_logprobs, err, R, V, K};
  if (K > 0) return dt == NV_DT_F32 ? run_logprobs<float, true>(a, s) : run_logprobs<bf16, true>(a, s);
  return dt == NV_DT_F32 ? run_logprobs<float, false>(a, s) : run_logprobs<bf16, false>(a, s);
}
