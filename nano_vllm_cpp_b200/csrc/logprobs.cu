// Log probabilities of given tokens, with the distribution's entropy, the tokens' ranks and the best alternatives.
//
//   m = max x,  Z = sum e^(x - m),  logprob(t) = x_t - m - log Z,  entropy = log Z - sum e^(x - m) (x - m) / Z
//
// One pass keeps m, n1 (how many logits equal m), s (the sum of the others' e^(x - m)) and e (the sum of e^(x - m) (x - m)):
// log Z = log n1 + log1p(s / n1).  The largest term is never added to the small ones, so the logarithm of an all but certain
// token's probability, -s, keeps its bits instead of being what 1 + s rounds to.
//
// The order of the alternatives and of the ranks is that of (logit descending, id ascending), the greedy choice first; a NaN
// comes after everything else.  A row that holds a NaN or plus infinity, or nothing above minus infinity, has no softmax: its
// numbers are NaN, its order is defined all the same.
#include "common.cuh"

namespace {

constexpr int LP_THREADS = 512;

// A float as an integer of the same order: NaN lowest, minus zero equal to zero.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// ... and with the id as the second criterion, lower ids first.
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
  return ((unsigned long long)order_of(x) << 32) | (uint32_t)(0x7fffffff - id);
}
__device__ __forceinline__ int id_of(unsigned long long key) { return 0x7fffffff - (int)(uint32_t)key; }

struct Stats {
  float m, n1, s, e;
};
__device__ __forceinline__ void add_value(Stats& a, float x) {
  if (x > a.m) {
    if (a.m != -INFINITY) {
      const float d = a.m - x, c = expf(d);                  // (d is minus infinity where x is plus infinity: c is zero)
      a.e = c > 0.f ? c * (a.e + d * (a.n1 + a.s)) : 0.f;
      a.s = c * (a.n1 + a.s);
    } else {
      a.s *= 0.f;                                            // (nothing, or the NaN of an earlier element)
    }
    a.m = x;
    a.n1 = 1.f;
  } else if (x == a.m) {
    a.n1 += 1.f;
  } else {
    const float d = x - a.m, c = expf(d);                    // (NaN stays NaN)
    a.s += c;
    if (c > 0.f) a.e = fmaf(c, d, a.e);
  }
}
__device__ __forceinline__ Stats merge(const Stats& a, const Stats& b) {
  const Stats& hi = a.m >= b.m ? a : b;
  const Stats& lo = a.m >= b.m ? b : a;
  Stats r = hi;
  if (lo.m == hi.m) {
    r.n1 = hi.n1 + lo.n1;
    r.s = hi.s + lo.s;
    r.e = hi.e + lo.e;
  } else {
    const float d = lo.m - hi.m, c = expf(d), all = lo.n1 + lo.s;
    r.s = hi.s + c * all;
    if (c > 0.f) r.e = hi.e + c * (lo.e + d * all);
    if (lo.s != lo.s) r.s = lo.s;                            // a NaN among the lower ones
  }
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
  int V, K;
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(LpArgs a) {
  __shared__ Stats st_s[LP_THREADS / 32];
  __shared__ int rank_s[LP_THREADS / 32];
  __shared__ unsigned long long key_s[LP_THREADS / 32], best_s;
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const T* x = (const T*)a.logits + (long long)row * a.stride;
  const int token = a.tokens ? a.tokens[row] : 0;
  const bool known = a.tokens && token >= 0 && token < a.V;
  const unsigned long long mine = known ? key_of(to_f32(x[token]), token) : ~0ull;

  Stats st = {-INFINITY, 0.f, 0.f, 0.f};
  int ahead = 0;
  for (int i = tid; i < a.V; i += LP_THREADS) {
    const float v = to_f32(x[i]);
    add_value(st, v);
    ahead += key_of(v, i) > mine;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.n1 = __shfl_xor_sync(0xffffffffu, st.n1, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.e = __shfl_xor_sync(0xffffffffu, st.e, o);
    st = (lane & o) ? merge(other, st) : merge(st, other);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  }
  if (lane == 0) {
    st_s[warp] = st;
    rank_s[warp] = ahead;
  }
  __syncthreads();
  st = st_s[0];
  ahead = rank_s[0];
  for (int w = 1; w < LP_THREADS / 32; ++w) {
    st = merge(st, st_s[w]);
    ahead += rank_s[w];
  }
  const bool proper = fabsf(st.m) < INFINITY;
  const float log_z = proper ? logf(st.n1) + log1pf(st.s / st.n1) : NAN;
  if (tid == 0) {
    if (a.tokens) {
      if (!known && a.err) atomicExch(a.err, 1 + row);
      if (a.logprob) a.logprob[row] = known ? (to_f32(x[token]) - st.m) - log_z : NAN;
      if (a.rank) a.rank[row] = known ? ahead : -1;
    }
    if (a.entropy) a.entropy[row] = log_z - st.e / (st.n1 + st.s);
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < a.K; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < a.V; i += LP_THREADS) {
      const unsigned long long key = key_of(to_f32(x[i]), i);
      if (key < below && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) key_s[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < LP_THREADS / 32; ++w) best = key_s[w] > best ? key_s[w] : best;
      best_s = best;
      const int id = id_of(best);
      a.top_ids[(long long)row * a.K + k] = id;
      a.top_logprobs[(long long)row * a.K + k] = (to_f32(x[id]) - st.m) - log_z;
    }
    __syncthreads();
    below = best_s;
  }
}

}  // namespace

NV_API int nv_token_logprobs_max_top(void) { return 32; }

// logits: R rows of V, `stride` elements apart.  tokens [R] or nullptr (then no logprob and no rank); logprob, entropy
// [R] float32, rank [R] int32: any may be nullptr; top_ids, top_logprobs [R, K] (K = 0: neither).  A token outside the vocabulary
// sets the error flag to 1 + its row and gets NaN and the rank -1.
NV_API int nv_token_logprobs(const void* logits, int dt, long long stride, int R, int V, const int* tokens, float* logprob,
                             float* entropy, int* rank, int K, int* top_ids, float* top_logprobs, int* err, cudaStream_t s) {
  if (!dt_ok(dt)) return NV_ERR_BAD_DTYPE;
  if (R < 0 || V < 1 || stride < V || K < 0 || K > V || K > nv_token_logprobs_max_top()) return NV_ERR_BAD_SIZE;
  if (K > 0 && (!top_ids || !top_logprobs)) return NV_ERR_BAD_SIZE;
  if (R == 0) return NV_OK;
  LpArgs a = {logits, stride, tokens, logprob, entropy, rank, top_ids, top_logprobs, err, V, K};
  if (dt == NV_DT_F32) NV_RETURN_IF(launch_dep(token_logprobs_kernel<float>, dim3(R), dim3(LP_THREADS), 0, s, a));
  else NV_RETURN_IF(launch_dep(token_logprobs_kernel<bf16>, dim3(R), dim3(LP_THREADS), 0, s, a));
  NV_RETURN_LAST();
}
