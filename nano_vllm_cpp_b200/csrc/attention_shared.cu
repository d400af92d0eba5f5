// Decode attention for rows that share a prefix: several replies to one prompt, or requests behind one system prompt.
//
// The rows of a group hold the same keys and values at their first len[g] positions.  The whole pages of these are read once,
// through the block table of the group's first row; a page that the prefix ends in every row reads for itself.  A row's softmax
// over all its keys is put together from parts with sums of their own,
//
//   m = max over the part of s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j;      out = sum_p e^(m_p - M) o_p / sum_p e^(m_p - M) l_p
//
// so the shared part can be worked out for all rows of the group at once, its keys and values read once instead of once a
// row: per kv head it is a matrix product of the (row, query head) pairs that read it.  Three launches: the shared parts (here),
// every row's own keys, from the page on that holds position len[g] (here, or the split-key kernel of attention_decode.cu), and their join
// (here).  A row that belongs to no group has no shared part; of a group's keys a row sees those up to its own position.
//
// What bounds it (bfloat16, heads of 128): 64 rows of 28 heads on 4 behind 8,192 positions, 16 to 512 of their own, take 34 us (each
// row by itself: 221), 18 of it the shared part, 10 the rows' own keys, 5 the join of up to 18 parts.  128 rows behind 16,384 take 51
// (673), 38 of it the shared part: 64 keys of two blocks of 128 pairs in 1.1 us a multiprocessor, where its exponentials alone take
// 0.6, the products 0.8 (those of different shapes do not overlap), and the 64 KB of keys and values from L2 0.9.
#include "tcgen05.cuh"

int nv_attention_decode_rest(const void* qkv, int q_dt, int q_stride, const void* kc, const void* vc, int cache_dt,
                             const int* block_table, int max_blocks, const int* row_entry, const int* positions, const int* rows,
                             const int* first, int R, float scale, int out_dt, int Hq, int Hkv, int D, int page, int num_pages,
                             int splits, int slots, float* scratch, int* err, int float_weights, float softcap, int beside, cudaStream_t stream);

namespace {

// (Queries, keys, values, parts and their sums are read past the first cache where a kernel reads them beside the one in front or without
// a wait of its own: kernels in front may write them while a kernel here has begun.)
struct SharedArgs {
  const void* q;
  const void* kc;
  const void* vc;
  const int* block_table;
  const int* row_entry;
  const int* positions;
  const int* rows;          // batch row of row r (nullptr: r)
  const int* members;       // [M] rows, group by group
  const int* cu;            // [groups + 1] into members
  const int* len;           // [groups] shared positions
  const int* lead;          // [groups] the row whose block table is read
  float* part_o;            // [R, Hq, slots, D]
  float* part_ml;           // [R, Hq, slots, 2]
  int* err;
  float scale, softcap;
  int q_dt, q_stride, max_blocks, num_pages, Hq, Hkv, D, page, groups, splits, slots, slot0;
  int split_keys;           // a split has at least so many keys (a multiple of the page and of the kernel's block of keys)
};

// A block's tile: which group, its first pair and the number of pairs from there on in the group, its places in `members`, whole
// pages of shared positions, and the leading row.
struct Tile {
  int group, pair0, pairs, member0, len, lead;
};
// Which tile of `rows_per_tile` pairs of which group is tile number x?  A whole warp looks, 32 groups at a time; group < 0: none (a
// launch has as many tiles as there may be).  A prefix that reaches beyond the block tables is read as far as these go, and reported:
// the arrays may have been replaced since the host last looked.
__device__ __forceinline__ Tile find_tile(const SharedArgs& a, int x, int G, int rows_per_tile, int lane) {
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = min(g0 + lane, a.groups - 1);
    const int from = a.cu[g], to = a.cu[g + 1], len = a.len[g], lead = a.lead[g];
    const int pairs = g0 + lane < a.groups ? (to - from) * G : 0, tiles = (pairs + rows_per_tile - 1) / rows_per_tile;
    int end = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += before;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, x < end);
    if (who) {
      const int l = __ffs(who) - 1, pair0 = (x - __shfl_sync(0xffffffffu, end - tiles, l)) * rows_per_tile;
      if (lane == l && len / a.page > a.max_blocks && a.err) atomicExch(a.err, 1 + (a.rows ? a.rows[lead] : lead));
      return Tile{g0 + l, pair0, __shfl_sync(0xffffffffu, pairs, l) - pair0, __shfl_sync(0xffffffffu, from, l),
                  min(__shfl_sync(0xffffffffu, len, l) / a.page, a.max_blocks) * a.page, __shfl_sync(0xffffffffu, lead, l)};
    }
    x -= __shfl_sync(0xffffffffu, end, 31);
  }
  return Tile{-1, 0, 0, 0, 0, 0};
}

// The plain form: any type, any head size in steps of eight, float32 products.  A block takes 16 pairs of one kv head and one
// split of the keys, 32 keys at a time; eight threads share a pair.  The values are on their way while the scores are worked out,
// the next keys while the values are summed.  DC: elements of a head at most.
constexpr int SP_PAIRS = 16, SP_KEYS = 32, SP_THREADS = 128;

template <typename T>
struct Eight;                                    // eight elements as they lie in the cache
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = __ldcg((const float4*)p); b = __ldcg((const float4*)p + 1); }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void put(float* to) const { *(float4*)to = a; *(float4*)(to + 4) = b; }
};
template <>
struct Eight<bf16> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = __ldcg((const uint4*)p); }
  __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void put(float* to) const {
    const __nv_bfloat162* h = (const __nv_bfloat162*)&a;
    const float2 f0 = __bfloat1622float2(h[0]), f1 = __bfloat1622float2(h[1]), f2 = __bfloat1622float2(h[2]), f3 = __bfloat1622float2(h[3]);
    *(float4*)to = make_float4(f0.x, f0.y, f1.x, f1.y);
    *(float4*)(to + 4) = make_float4(f2.x, f2.y, f3.x, f3.y);
  }
};

template <typename T, int DC>
__global__ void __launch_bounds__(SP_THREADS) shared_plain_kernel(SharedArgs a) {
  constexpr int CHUNKS = SP_KEYS * (DC / 8) / SP_THREADS;        // pieces of eight elements a thread fetches of a block of keys
  extern __shared__ __align__(16) float sp_smem[];
  const int D = a.D, LD = D + 4;
  float* q_s = sp_smem;                          // [SP_PAIRS][LD]
  float* k_s = q_s + SP_PAIRS * LD;              // [SP_KEYS][LD]
  float* v_s = k_s + SP_KEYS * LD;               // [SP_KEYS][LD]
  __shared__ float p_s[SP_PAIRS][SP_KEYS + 1];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, kvh = blockIdx.y, split = blockIdx.z, G = a.Hq / a.Hkv;
  const Tile tile = find_tile(a, blockIdx.x, G, SP_PAIRS, tid % 32);
  if (tile.group < 0) return;
  const int m0 = tile.member0, pair0 = tile.pair0, pairs = pair0 + tile.pairs, len = tile.len;
  const int lead = tile.lead, lead_t = a.rows ? a.rows[lead] : lead;
  const int* bt = a.block_table + (long long)a.row_entry[lead_t] * a.max_blocks;
  const int share = max(a.split_keys, ((len + a.splits - 1) / a.splits + SP_KEYS - 1) / SP_KEYS * SP_KEYS);
  const int j_lo = min(len, split * share), j_hi = min(len, j_lo + share);

  Eight<T> part[CHUNKS];
  auto fetch = [&](const void* cache, int j0) {  // zeros behind the split
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int x = tid + c * SP_THREADS, key = x / (D / 8), at = x % (D / 8), j = j0 + key;
      part[c].zero();
      if (key < SP_KEYS && j < j_hi) {
        const int blk = bt[j / a.page];
        if (blk >= 0 && blk < a.num_pages) part[c].load((const T*)cache + (((size_t)blk * a.Hkv + kvh) * a.page + j % a.page) * D + at * 8);
        else if (a.err) atomicExch(a.err, 1 + lead_t);
      }
    }
  };
  auto put = [&](float* to) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int x = tid + c * SP_THREADS, key = x / (D / 8), at = x % (D / 8);
      if (key < SP_KEYS) part[c].put(to + key * LD + at * 8);
    }
  };
  fetch(a.kc, j_lo);

  const int i = tid / 8, sub = tid % 8;          // this thread's pair of the tile, and which of its eight threads it is
  const bool live = pair0 + i < pairs;
  const int r = live ? a.members[m0 + (pair0 + i) / G] : lead, h = kvh * G + (live ? (pair0 + i) % G : 0);
  const int t = a.rows ? a.rows[r] : r;
  const int limit = live ? min(j_hi, a.positions[t] + 1) : 0;        // the first key that this row does not see
  for (int d = sub; d < D; d += 8) q_s[i * LD + d] = live ? ld_dt(a.q, a.q_dt, (size_t)t * a.q_stride + (size_t)h * D + d) * a.scale : 0.f;

  float m = -INFINITY, l = 0.f, o[DC / 32][4];
#pragma unroll
  for (int c = 0; c < DC / 32; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
  for (int j0 = j_lo; j0 < j_hi; j0 += SP_KEYS) {
    put(k_s);                                    // (the scores before these are done: every thread has been at the barrier below)
    __syncthreads();
    fetch(a.vc, j0);
    float s[SP_KEYS / 8];
#pragma unroll
    for (int u = 0; u < SP_KEYS / 8; ++u) s[u] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 4; ++c) {
      const float4 qv = *(const float4*)&q_s[i * LD + c * 4];
#pragma unroll
      for (int u = 0; u < SP_KEYS / 8; ++u) {
        const float4 kv = *(const float4*)&k_s[(u * 8 + sub) * LD + c * 4];
        s[u] = fmaf(qv.x, kv.x, s[u]); s[u] = fmaf(qv.y, kv.y, s[u]); s[u] = fmaf(qv.z, kv.z, s[u]); s[u] = fmaf(qv.w, kv.w, s[u]);
      }
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < SP_KEYS / 8; ++u) {
      if (a.softcap > 0.f) s[u] = a.softcap * tanhf(s[u] / a.softcap);
      if (j0 + u * 8 + sub >= limit) s[u] = -INFINITY;
      mx = fmaxf(mx, s[u]);
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float ref = mx == -INFINITY ? 0.f : mx, alpha = expf(m - ref);
    m = mx;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < SP_KEYS / 8; ++u) {
      const float p = expf(s[u] - ref);
      p_s[i][u * 8 + sub] = p;
      sum += p;
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * alpha + sum;
    put(v_s);                                    // (the sums before these are done: every thread has been at the barrier above)
    __syncthreads();
    fetch(a.kc, j0 + SP_KEYS);
#pragma unroll
    for (int c = 0; c < DC / 32; ++c)
#pragma unroll
      for (int u = 0; u < 4; ++u) o[c][u] *= alpha;
#pragma unroll 4
    for (int key = 0; key < SP_KEYS; ++key) {
      const float p = p_s[i][key];
#pragma unroll
      for (int c = 0; c < DC / 32; ++c) {
        const int at = (c * 8 + sub) * 4;
        if (at < D) {
          const float4 v = *(const float4*)&v_s[key * LD + at];
          o[c][0] = fmaf(p, v.x, o[c][0]); o[c][1] = fmaf(p, v.y, o[c][1]); o[c][2] = fmaf(p, v.z, o[c][2]); o[c][3] = fmaf(p, v.w, o[c][3]);
        }
      }
    }
  }
  if (!live) return;
  const size_t at = ((size_t)r * a.Hq + h) * a.slots + a.slot0 + split;
#pragma unroll
  for (int c = 0; c < DC / 32; ++c) {
    const int d = (c * 8 + sub) * 4;
    if (d < D) *(float4*)(a.part_o + at * D + d) = make_float4(o[c][0], o[c][1], o[c][2], o[c][3]);
  }
  if (sub == 0) {
    a.part_ml[at * 2] = m == -INFINITY ? -1e30f : m;
    a.part_ml[at * 2 + 1] = l;
  }
}

// The tensor-core form, for bfloat16 and head sizes in steps of 16 from 32 on: a CTA takes 128 pairs of one kv head and one split
// of the keys, 64 keys at a time.  S = Q K^T and O += P V are tcgen05.mma with S, P (two buffers) and O in tensor memory:
//   warp 0     fetches the pages of K (two buffers) and V as TMA boxes of one page x 64 elements, a lane a box
//   warp 1     allocates tensor memory; issues the products, a lane of it elected
//   warps 2-5  gather the queries of the tile's pairs into shared memory (128-byte swizzle), then a thread owns a pair: it takes its
//              row of S into registers, whereupon the next product may write S, keeps the row's maximum and sum, writes P as bfloat16
//              to where the second product takes it (three terms: into shared memory), and at the end its row of O, undivided, with
//              maximum and sum to the scratch
// All keys of a split are seen by all pairs, but for those behind a row's own position, so there is no mask in most blocks.  TERMS =
// 3: the float32 weights enter the product with the values as three bfloat16 terms (all their bits) instead of one rounded.
// Heads between the forms' sizes: the boxes reach beyond the pages' rows and are filled with zeros.
constexpr int ST_PAIRS = 128, ST_KEYS = 64, ST_THREADS = 192;

// Shared memory to global in one copy: addresses and bytes in steps of 16; the caller waits before it leaves.
__device__ __forceinline__ void bulk_store(void* to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(from)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_store_wait() {
  asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
}

// A warp's 32 queries of a tile of `pairs` pairs (lane's: batch row t, head h) into shared memory, D / 8 lanes a row and sixteen loads of a
// lane under way; rows of nobody and columns beyond the head are zeros.  q: the warp's quarter of the tile.
template <int D>
__device__ __forceinline__ void gather_queries(const SharedArgs& a, uint8_t* Qs, int q, int lane, int pairs, int t, int h) {
  constexpr int PER = D / 8, AT_ONCE = 32 / PER, LOADS = 32 / AT_ONCE < 16 ? 32 / AT_ONCE : 16;      // (PER is 8, 16 or 32)
  const int c = lane % PER;
  const long long place = (long long)t * a.q_stride + (long long)h * a.D;
#pragma unroll
  for (int i0 = 0; i0 < 32; i0 += LOADS * AT_ONCE) {
    uint4 v[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = i0 + u * AT_ONCE + lane / PER;
      const long long from = __shfl_sync(0xffffffffu, place, i);
      v[u] = q * 32 + i < pairs && c * 8 < a.D ? *(const uint4*)((const bf16*)a.q + from + c * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int row = q * 32 + i0 + u * AT_ONCE + lane / PER;
      *(uint4*)(Qs + (c / 8) * (ST_PAIRS * 128) + row * 128 + (((c % 8) ^ (row & 7)) << 4)) = v[u];
    }
  }
  fence_async_smem();
  __syncwarp();
}

// A score's cap, in base-2 units.  capped_log2's error is some 2^-22 of the cap, however small the score.  TERMS 3, where the weights keep
// all their bits: an error of some units of the result.  Up to half the cap the tangent's series (x^15 is its last term, the next is
// 2^-27 of the sum; 1.1 units), beyond 1 - 2 / (e^2x + 1), which is no difference of like numbers there (7.5 units at most).  (64 rows of 28 heads on 4 behind 8,192 with a sink
// and a cap: 54.3 us by capped_log2, 61.9 so, 70.8 by tanhf.)  shared_map has the factor that either takes.
__device__ __forceinline__ float capped_small(const ScoreMap& map, float s) {
  const float x = s * map.cap_k, z = x * x;
  float p = -929569.f / 638512875.f;
  p = fmaf(p, z, 21844.f / 6081075.f);
  p = fmaf(p, z, -1382.f / 155925.f);
  p = fmaf(p, z, 62.f / 2835.f);
  p = fmaf(p, z, -17.f / 315.f);
  p = fmaf(p, z, 2.f / 15.f);
  p = fmaf(p, z, -1.f / 3.f);
  return map.cap1 * fmaf(x * z, p, x);
}
template <int TERMS>
__device__ __forceinline__ float capped(const ScoreMap& map, float s) {
  if (TERMS == 1) return capped_log2(map, s);
  const float x = s * map.cap_k, e = ex2_fast(fabsf(x) * 2.8853900817779268f);
  return fabsf(x) <= 0.5f ? capped_small(map, s) : map.cap1 * copysignf(fmaf(-2.f, rcp_fast(e + 1.f), 1.f), x);
}
static inline ScoreMap shared_map(float scale, float softcap, int terms) {
  ScoreMap map = score_map(scale, softcap);
  if (terms > 1 && softcap > 0.f) map.cap_k = scale / softcap;
  return map;
}

// A pair's next block of scores, from key j on, becomes weights against its reference m; returns the sum of its weights, l among them.
// The reference follows the maximum only when that has moved by more than 2^8 (weights of up to 256 cost bfloat16 and the float32
// sums nothing), so that O is rescaled, by alpha, once in a long while.
template <int TERMS, bool CAP>
__device__ __forceinline__ float softmax_step(const ScoreMap& map, float* s, int j, int limit, float& m, float& alpha, float l) {
  if (CAP && TERMS == 1 && map.cap1 > 0.f) {
#pragma unroll
    for (int c = 0; c < ST_KEYS; ++c) s[c] = capped<TERMS>(map, s[c]);
  }
  if (CAP && TERMS > 1) {
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < ST_KEYS; ++c) most = fmaxf(most, fabsf(s[c]));
    if (__all_sync(0xffffffffu, most * map.cap_k <= 0.5f)) {
#pragma unroll
      for (int c = 0; c < ST_KEYS; ++c) s[c] = capped_small(map, s[c]);
    } else {
#pragma unroll
      for (int c = 0; c < ST_KEYS; ++c) s[c] = capped<TERMS>(map, s[c]);
    }
  }
  if (j + ST_KEYS > limit) {
#pragma unroll
    for (int c = 0; c < ST_KEYS; ++c)
      if (j + c >= limit) s[c] = -INFINITY;
  }
  float mx4[4] = {s[0], s[1], s[2], s[3]};                       // four chains, three numbers a step
#pragma unroll
  for (int c = 4; c < ST_KEYS - 4; c += 8) {
#pragma unroll
    for (int u = 0; u < 4; ++u) mx4[u] = fmaxf(fmaxf(s[c + u], s[c + 4 + u]), mx4[u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) mx4[u] = fmaxf(mx4[u], s[ST_KEYS - 4 + u]);
  const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
  if (mx > m && (m == -INFINITY || (mx - m) * map.in > 8.f)) {
    alpha = m == -INFINITY ? 0.f : ex2_fast((m - mx) * map.in);
    m = mx;
  }
  const float ms = m == -INFINITY ? 0.f : m * map.in;
  // two elements an instruction where there is one
  float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  const float2 in2 = make_float2(map.in, map.in), ms2 = make_float2(-ms, -ms);
#pragma unroll
  for (int c = 0; c < ST_KEYS; c += 4) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float2 e = fma2(make_float2(s[c + 2 * u], s[c + 2 * u + 1]), in2, ms2);
      s[c + 2 * u] = ex2_fast(e.x);
      s[c + 2 * u + 1] = ex2_fast(e.y);
      sum2[u] = add2(sum2[u], make_float2(s[c + 2 * u], s[c + 2 * u + 1]));
    }
  }
  return l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
}
// A row's weights as bfloat16 into tensor memory, two in a column.
__device__ __forceinline__ void put_weights(uint32_t to, const float* s) {
  uint32_t w[ST_KEYS / 2];
#pragma unroll
  for (int c = 0; c < ST_KEYS / 2; ++c) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(s[2 * c], s[2 * c + 1]);
    w[c] = *(const uint32_t*)&b;
  }
  tmem_st32_u32(to, w);
}
// The warp's rows of O, where any of them is to be rescaled.
template <int D>
__device__ __forceinline__ void rescale(uint32_t tmem_o, float alpha) {
  if (!__any_sync(0xffffffffu, alpha != 1.f)) return;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    float o[32];
    tmem_ld32(tmem_o + c * 32, o);
#pragma unroll
    for (int j = 0; j < 32; ++j) o[j] *= alpha;
    tmem_st32(tmem_o + c * 32, o);
  }
}

// A pair's part: its row of O as it is (some: a product has written it; else zeros), relative to m, with maximum and sum.  The row
// goes through shared memory (all of it is free now; rows a chunk of 16 bytes further apart than they are long, so that a warp's
// threads write to different banks) and leaves in one copy: whole lines instead of 16 bytes in each of 32.
template <int D>
__device__ __forceinline__ void leave_part(const SharedArgs& a, uint8_t* row, uint32_t tmem_o, bool some, bool live, size_t at, float m,
                                           float l, float in) {
  if (live) {
    // (m is in the units of the raw or the capped scores: `in` takes it to base 2)
    a.part_ml[at * 2] = m == -INFINITY ? -1e30f : m * in * 0.6931471805599453f;
    a.part_ml[at * 2 + 1] = l;
  }
  constexpr int W = D < 128 ? D : 128;                  // columns whose loads are under way at once
#pragma unroll
  for (int c0 = 0; c0 < D; c0 += W) {
    float o[W];
    if (some) {
#pragma unroll
      for (int c = 0; c < W; c += 32) tmem_ld32_nowait(tmem_o + c0 + c, o + c);
      tmem_ld_wait();
      tmem_ld_fence<W>(o);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) o[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < W; j += 4) *(float4*)(row + (c0 + j) * 4) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
  }
  fence_async_smem();
  if (live) bulk_store(a.part_o + at * a.D, row, (uint32_t)a.D * 4);
  bulk_store_wait();
}

template <int D>
constexpr int st_tmem_cols() { return 2 * ST_KEYS + D <= 256 ? 256 : 512; }

// Buffers of values: two, but for the largest form, whose three tiles of P leave room for one.
template <int D, int TERMS>
constexpr int st_v_buffers() { return D > 128 && TERMS > 1 ? 1 : 2; }

// CAP: scores may be capped (TERMS 1) or are (TERMS 3, whose cap has a form of its own: in one with the other it took 2 % of its time).
template <int D, int TERMS, bool CAP>
__global__ void __launch_bounds__(ST_THREADS, D <= 128 ? 2 : 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, SharedArgs a, ScoreMap map) {
  constexpr int SL = D / 64, VB = st_v_buffers<D, TERMS>();
  constexpr uint32_t Q_SLAB = ST_PAIRS * 128, KV_SLAB = ST_KEYS * 128, P_TILE = ST_PAIRS * 128;
  extern __shared__ __align__(1024) uint8_t st_smem_raw[];
  __shared__ uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full, s_free, p_full, pv_done;
  __shared__ uint32_t tmem_base_s;

  uint8_t* smem = (uint8_t*)(((uintptr_t)st_smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* Qs = smem;
  uint8_t* Ks = Qs + SL * Q_SLAB;                  // two buffers
  uint8_t* Vs = Ks + 2 * SL * KV_SLAB;             // VB buffers
  uint8_t* Ps = Vs + VB * SL * KV_SLAB;             // TERMS > 1: so many tiles of [128 pairs][64 keys]

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int kvh = blockIdx.y, split = blockIdx.z, G = a.Hq / a.Hkv;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tm_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tm_v) : "memory");
    mbar_init(&q_full, 4);                         // one arrival per softmax warp
    for (int b = 0; b < 2; ++b) {
      mbar_init(&k_full[b], 1);
      mbar_init(&k_empty[b], 1);
      mbar_init(&v_full[b], 1);
      mbar_init(&v_empty[b], 1);
    }
    mbar_init(&s_full, 1);
    mbar_init(&s_free, 4);
    mbar_init(&p_full, 4);
    mbar_init(&pv_done, 1);
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&tmem_base_s, st_tmem_cols<D>());
  // The groups, the tables and the positions are inputs of the whole step (as in attention_decode.cu): they are read before the
  // kernel in front has ended, every warp for itself; queries, keys and values come after the wait.
  const Tile tile = find_tile(a, blockIdx.x, G, ST_PAIRS, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  if (tile.group >= 0) {
    const int pair0 = tile.pair0, pairs = min(ST_PAIRS, tile.pairs), len = tile.len;
    const int share = max(a.split_keys, ((len + a.splits - 1) / a.splits + ST_KEYS - 1) / ST_KEYS * ST_KEYS);
    const int j_lo = min(len, split * share), j_hi = min(len, j_lo + share);
    const int n_blocks = (j_hi - j_lo + ST_KEYS - 1) / ST_KEYS;
    const uint32_t tmem_s = tmem_base, tmem_p = tmem_base + ST_KEYS, tmem_o = tmem_base + 2 * ST_KEYS;      // (P: two buffers)
    const int lead_t = a.rows ? a.rows[tile.lead] : tile.lead;
    // A block's keys behind the split's end are not loaded; their weights are zero, their values must be finite numbers.  Only the
    // first VB blocks meet what the shared memory held before.
    if (n_blocks <= VB && (j_hi - j_lo) % ST_KEYS) {
      for (int i = tid; i < (int)(VB * SL * KV_SLAB / 16); i += ST_THREADS) ((uint4*)Vs)[i] = make_uint4(0, 0, 0, 0);
      fence_async_smem();
      __syncthreads();
    }

    if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer
      const int page_shift = 31 - __clz(a.page);     // pages are 16, 32 or 64 keys
      const int pages = ST_KEYS >> page_shift;
      const uint32_t box = (uint32_t)a.page * 128;
      const int my_p = lane / SL, my_s = lane % SL;
      const int* bt = a.block_table + (long long)a.row_entry[lead_t] * a.max_blocks + (j_lo >> page_shift);
      const int n_pages = my_p < pages ? (j_hi - j_lo) >> page_shift : 0;      // (a lane without a box has none)
      auto page_of = [&](int i) { return i * pages + my_p < n_pages ? bt[i * pages + my_p] : -2; };
      int blk_k = page_of(0), blk_v = blk_k, blk_next = page_of(1);            // read two blocks ahead
      grid_dep_wait();
      grid_dep_launch();
      auto load = [&](int i, bool values, int blk) {
        if (blk != -2 && (blk < 0 || blk >= a.num_pages)) {                    // it should be there and is not
          if (a.err) atomicExch(a.err, 1 + lead_t);
          blk = -1;
        }
        const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, blk >= 0));
        const int vb = i % VB;
        uint64_t* full = values ? &v_full[vb] : &k_full[i & 1];
        if (lane == 0) {
          if (values) mbar_wait(&v_empty[vb], ((i / VB) & 1) ^ 1, a.err, 0x7302);
          else mbar_wait(&k_empty[i & 1], ((i >> 1) & 1) ^ 1, a.err, 0x7301);
          mbar_expect_tx(full, boxes * box);
        }
        __syncwarp();
        if (blk >= 0) {
          uint8_t* dst = (values ? Vs + vb * SL * KV_SLAB : Ks + (i & 1) * SL * KV_SLAB) + my_s * KV_SLAB + my_p * box;
          tma_load_2d(dst, values ? &tm_v : &tm_k, full, my_s * 64, (blk * a.Hkv + kvh) * a.page);
        }
      };
      if (n_blocks > 0) load(0, false, blk_k);
      for (int i = 0; i < n_blocks; ++i) {         // the next keys go out before these values: they are free earlier
        blk_v = blk_k;
        blk_k = blk_next;
        blk_next = page_of(i + 2);
        if (i + 1 < n_blocks) load(i + 1, false, blk_k);
        load(i, true, blk_v);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer
      grid_dep_wait();
      grid_dep_launch();
      const int n = __shfl_sync(0xffffffffu, n_blocks, 0);
      const uint32_t tmem_s = __shfl_sync(0xffffffffu, tmem_base, 0), tmem_p = tmem_s + ST_KEYS, tmem_o = tmem_s + 2 * ST_KEYS;
      if (n > 0) {
        const uint32_t idesc_s = instr_desc(ST_KEYS), idesc_o = instr_desc_b_mn(D);
        const uint32_t q_addr = smem_u32(Qs), k_addr = smem_u32(Ks), v_addr = smem_u32(Vs), p_addr = smem_u32(Ps);
        uint64_t dq[SL], dk[2][SL], dp[TERMS];
#pragma unroll
        for (int s = 0; s < SL; ++s) {
          dq[s] = smem_desc_sw128(q_addr + s * Q_SLAB);
          dk[0][s] = smem_desc_sw128(k_addr + s * KV_SLAB);
          dk[1][s] = smem_desc_sw128(k_addr + (SL + s) * KV_SLAB);
        }
        const uint64_t dv[2] = {smem_desc_sw128_mn(v_addr, KV_SLAB, 1024), smem_desc_sw128_mn(v_addr + SL * KV_SLAB, KV_SLAB, 1024)};
#pragma unroll
        for (int t = 0; t < TERMS; ++t) dp[t] = smem_desc_sw128(p_addr + t * P_TILE);
        auto issue_s = [&](int i) {
          const int b = i & 1;
          mbar_wait(&k_full[b], (i >> 1) & 1, a.err, 0x7303);
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < SL; ++s)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16_warp(tmem_s, dq[s] + k * 2, (b ? dk[1][s] : dk[0][s]) + k * 2, idesc_s, (s || k) ? 1u : 0u);
          umma_commit_warp(&k_empty[b]);
          umma_commit_warp(&s_full);
        };
        mbar_wait(&q_full, 0, a.err, 0x7304);
        tc_fence_after();
        issue_s(0);
        for (int i = 0; i < n; ++i) {
          if (i + 1 < n) {                             // S(i) is in the threads' registers
            mbar_wait(&s_free, i & 1, a.err, 0x7310);
            issue_s(i + 1);
          }
          mbar_wait(&p_full, i & 1, a.err, 0x7305);    // P(i) is written, O is rescaled
          mbar_wait(&v_full[i % VB], (i / VB) & 1, a.err, 0x7306);
          tc_fence_after();
          // 16 keys per product: eight columns of P in tensor memory, or 32 bytes (2 units) along its rows in shared memory, and two
          // 8-key groups (2,048 bytes = 128 units) of V
          const uint64_t v = i % VB ? dv[1] : dv[0];
          if (TERMS == 1) {
#pragma unroll
            for (int k = 0; k < ST_KEYS / 16; ++k)
              umma_bf16_ts_warp(tmem_o, tmem_p + (i & 1) * (ST_KEYS / 2) + k * 8, v + k * 128, idesc_o, (i || k) ? 1u : 0u);
          } else {
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
              for (int k = 0; k < ST_KEYS / 16; ++k) umma_bf16_warp(tmem_o, dp[t] + k * 2, v + k * 128, idesc_o, (i || t || k) ? 1u : 0u);
          }
          umma_commit_warp(&v_empty[i % VB]);
          umma_commit_warp(&pv_done);
        }
      }
    } else {
      // ---------------------------------------------------------------- a thread a pair
      const int q = warp % 4;                        // a warp may touch tensor-memory lanes [32q, 32q + 32) only
      const int p = q * 32 + lane;
      const bool live = p < pairs, some = q * 32 < pairs;       // (a warp without pairs only arrives where it is waited for)
      const int r = live ? a.members[tile.member0 + (pair0 + p) / G] : tile.lead, h = kvh * G + (live ? (pair0 + p) % G : 0);
      const int t = a.rows ? a.rows[r] : r;
      const uint32_t lane_off = (uint32_t)(q * 32) << 16;
      const int position = a.positions[t];
      grid_dep_wait();
      grid_dep_launch();
      // (A split without keys has no products: nobody waits for its queries, and nothing would order one warp's gathering before
      // another's results, which take the same shared memory.)
      if (n_blocks > 0) {
        gather_queries<D>(a, Qs, q, lane, pairs, t, h);
        if (lane == 0) mbar_arrive(&q_full);
      }
      const int limit = live ? min(j_hi, position + 1) : j_hi;                  // the first key that this row does not see
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < n_blocks; ++i) {
        const int j0 = j_lo + i * ST_KEYS;
        mbar_wait(&s_full, i & 1, a.err, 0x7307);
        float s[ST_KEYS];
        float alpha = 1.f;
        if (some) {
          tc_fence_after();
          tmem_ld32_nowait(tmem_s + lane_off, s);
          tmem_ld32_nowait(tmem_s + lane_off + 32, s + 32);
          tmem_ld_wait();
          tmem_ld_fence<64>(s);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free);
        if (some) {
          l = softmax_step<TERMS, CAP>(map, s, j0, limit, m, alpha, l);
        }
        // O += P(i-1) V(i-1) must have ended before O is rescaled and P is overwritten (a warp without pairs waits too: its
        // arrival is one for this block)
        if (i > 0) {
          mbar_wait(&pv_done, (i - 1) & 1, a.err, 0x7309);
          tc_fence_after();
        }
        if (some) {
          if (i > 0) rescale<D>(tmem_o + lane_off, alpha);
          if (TERMS == 1) {
            put_weights(tmem_p + (i & 1) * (ST_KEYS / 2) + lane_off, s);
          } else {
            uint8_t* prow = Ps + (size_t)p * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float w[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) w[u] = s[c * 8 + u];
#pragma unroll
              for (int x = 0; x < TERMS; ++x) {
                __nv_bfloat162 b[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) b[u] = __floats2bfloat162_rn(w[2 * u], w[2 * u + 1]);
                *(uint4*)(prow + x * P_TILE + ((c ^ (p & 7)) << 4)) = *(uint4*)b;
                if (x + 1 < TERMS) {
#pragma unroll
                  for (int u = 0; u < 4; ++u) {
                    const float2 f = __bfloat1622float2(b[u]);
                    w[2 * u] -= f.x;
                    w[2 * u + 1] -= f.y;
                  }
                }
              }
            }
            fence_async_smem();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full);
      }
      // ---- this split's part: O as it is, relative to m
      if (n_blocks > 0) {
        mbar_wait(&pv_done, (n_blocks - 1) & 1, a.err, 0x7308);
        tc_fence_after();
      }
      if (some)
        leave_part<D>(a, smem + (size_t)p * (D * 4 + 16), tmem_o + lane_off, n_blocks > 0, live, ((size_t)r * a.Hq + h) * a.slots + a.slot0 + split, m, l, map.in);
    }
  } else {                       // no tile: a block waits all the same, since the kernel of the own keys relies on it (and there may be none with one)
    grid_dep_wait();
    grid_dep_launch();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, st_tmem_cols<D>());
}

// Every row's own keys, from the page on that the prefix ends in, for bfloat16, heads of 64, 80, 96, 128 or 256 elements: eight query heads
// of a kv head and one split of the keys a block, whose four warps take 16 keys in turn.  A row has few keys of its own, so that a
// block's time is its latency; there is no ring of pages, no copy into shared memory and no order among the warps until their sums are
// joined: keys and values come as 16-byte loads to where the products want them.  S^T = K Q^T and O^T = V^T P^T (mma.sync, 16 keys or
// dimensions by 8 heads): a product does not care which of the head's elements it calls its k-th, so a lane's piece of eight elements is
// four of its places in two products of S^T; row g of product 8 i + j of O^T is element 128 i + 8 g + j, row g + 8 the same of the 64
// behind.  (Whole calls with this kernel and with the split-key kernel, whose ring has eight pages of 16 and two of 32 x 256: 64 rows of 28
// heads on 4 behind 8,192 positions 33.9 and 38.4 us, 44 of 16 heads of 256 on 1 in pages of 32 27.8 and 92.9.  Four blocks a
// multiprocessor, for which registers are spilled, 58.6 us where three take 55.7.)
constexpr int OW_WARPS = 4, OW_HEADS = 8;

// Where a row's keys are all in one part, its result needs no join (out: nullptr where it does).
struct OwnResult {
  void* out;
  int out_dt, has_sink;
  float sink;
  HeadGate gate;
};

__device__ __forceinline__ void mma_16x8(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {        // 8 x 8 elements over a warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D, int TERMS>
__global__ void __launch_bounds__(OW_WARPS * 32, D <= 128 ? 3 : 2) own_keys_kernel(SharedArgs a, const int* __restrict__ first, int own_splits, ScoreMap map,
                                                                int beside, OwnResult result) {
  // 16-byte pieces of a key a lane; runs of 128 elements; registers of a value behind a run's first 64
  constexpr int KC = (D + 31) / 32, RUNS = (D + 127) / 128, MORE = D < 128 ? (D - 64) / 16 : 4;
  __shared__ float o_s[OW_WARPS][OW_HEADS][D + 4], m_s[OW_WARPS][OW_HEADS], l_s[OW_WARPS][OW_HEADS];
  const int r = blockIdx.x, t = a.rows ? a.rows[r] : r, G = a.Hq / a.Hkv, parts = (G + OW_HEADS - 1) / OW_HEADS;
  const int kvh = blockIdx.y / parts, h0 = kvh * G + blockIdx.y % parts * OW_HEADS, heads = min(OW_HEADS, (kvh + 1) * G - h0), split = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, tq = lane % 4;
  const int n = a.positions[t] + 1, lo = first ? first[r] / a.page * a.page : 0;
  const int units = max(0, (n - lo + 15) / 16), per = (units + own_splits - 1) / own_splits;
  const int u0 = split * per, u1 = min(units, u0 + per);
  const int* bt = a.block_table + (long long)a.row_entry[t] * a.max_blocks;
  // (beside the shared part, which has waited for what wrote the queries and the newest page, and whose results are not read here)
  if (!beside) grid_dep_wait();
  grid_dep_launch();
  uint4 q[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c)
    q[c] = g < heads && c * 32 + tq * 8 < D
               ? __ldcg((const uint4*)((const bf16*)a.q + (long long)t * a.q_stride + (long long)(h0 + g) * D + c * 32 + tq * 8))
               : make_uint4(0, 0, 0, 0);

  float o[8 * RUNS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8 * RUNS; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  uint4 ka[KC], kb[KC], v[RUNS][4];                                  // keys g and g + 8; values of keys 2 tq, 2 tq + 1, and 8 behind
  uint32_t w[RUNS][4][MORE > 0 ? MORE : 1];
  int pages = -2;                                                    // lane i: where this warp's unit i of 32 lies
  auto place_of = [&](int i) {                                       // the unit's first key, in rows of the cache; -1: not there
    const int u = u0 + warp + i * OW_WARPS;
    if (i % 32 == 0) {
      const int mine = u + lane * OW_WARPS;
      pages = mine < u1 ? bt[(lo + mine * 16) / a.page] : -2;
    }
    const int blk = __shfl_sync(0xffffffffu, pages, i % 32);
    if (blk == -2) return -1LL;
    if (blk < 0 || blk >= a.num_pages) {
      if (lane == 0 && a.err) atomicExch(a.err, 1 + t);
      return -1LL;
    }
    return ((long long)blk * a.Hkv + kvh) * a.page + (lo + u * 16) % a.page;
  };
  auto fetch_keys = [&](long long at) {
    if (at < 0) return;
    const bf16* x = (const bf16*)a.kc + (at + g) * D + tq * 8;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const bool in = c * 32 + tq * 8 < D;
      ka[c] = in ? __ldcg((const uint4*)(x + c * 32)) : make_uint4(0, 0, 0, 0);
      kb[c] = in ? __ldcg((const uint4*)(x + 8 * D + c * 32)) : make_uint4(0, 0, 0, 0);
    }
  };
  auto fetch_values = [&](long long at, int left) {                  // zeros behind the row's position
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 2 * tq + (i & 1) + (i >> 1) * 8;
      const bf16* x = (const bf16*)a.vc + (at + key) * D;
      const bool there = at >= 0 && key < left;
#pragma unroll
      for (int u = 0; u < RUNS; ++u) {
        v[u][i] = there ? __ldcg((const uint4*)(x + u * 128 + g * 8)) : make_uint4(0, 0, 0, 0);
        if (MORE == 4) {
          const uint4 y = there ? __ldcg((const uint4*)(x + u * 128 + 64 + g * 8)) : make_uint4(0, 0, 0, 0);
          w[u][i][0] = y.x; w[u][i][MORE > 1 ? 1 : 0] = y.y; w[u][i][MORE > 2 ? 2 : 0] = y.z; w[u][i][MORE > 3 ? 3 : 0] = y.w;
        }
        if (MORE == 2) {
          const uint2 y = there ? __ldcg((const uint2*)(x + 64 + g * 4)) : make_uint2(0, 0);
          w[u][i][0] = y.x; w[u][i][MORE > 1 ? 1 : 0] = y.y;
        }
        if (MORE == 1) w[u][i][0] = there ? __ldcg((const uint32_t*)(x + 64 + g * 2)) : 0u;
      }
    }
  };
  const int rounds = u0 + warp < u1 ? (u1 - u0 - warp + OW_WARPS - 1) / OW_WARPS : 0;
  long long at = rounds > 0 ? place_of(0) : -1;
  fetch_keys(at);
  fetch_values(at, n - lo - (u0 + warp) * 16);
  for (int i = 0; i < rounds; ++i) {
    const int left = n - lo - (u0 + warp + i * OW_WARPS) * 16;       // keys from the unit's first on
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      mma_16x8(s, ka[c].x, kb[c].x, ka[c].y, kb[c].y, q[c].x, q[c].y);
      mma_16x8(s, ka[c].z, kb[c].z, ka[c].w, kb[c].w, q[c].z, q[c].w);
    }
    const bool here = at >= 0;
    at = i + 1 < rounds ? place_of(i + 1) : -1;
    fetch_keys(at);
    // s: keys g (heads 2 tq, 2 tq + 1) and g + 8, in base-2 units from here on
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      s[x] = map.cap1 > 0.f ? capped<TERMS>(map, s[x]) : s[x] * map.in;
      if (!here || g + (x >> 1) * 8 >= left) s[x] = -INFINITY;
    }
    float alpha[2], ref[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float mx = fmaxf(s[x], s[x + 2]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      mx = fmaxf(mx, m[x]);
      ref[x] = mx == -INFINITY ? 0.f : mx;
      alpha[x] = ex2_fast(m[x] - ref[x]);
      m[x] = mx;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) s[x] = ex2_fast(s[x] - ref[x & 1]);
    l[0] = l[0] * alpha[0] + (s[0] + s[2]);
    l[1] = l[1] * alpha[1] + (s[1] + s[3]);
#pragma unroll
    for (int j = 0; j < 8 * RUNS; ++j) {
      o[j][0] *= alpha[0]; o[j][1] *= alpha[1]; o[j][2] *= alpha[0]; o[j][3] *= alpha[1];
    }
    uint32_t b[TERMS][2];                                            // the weights: rounded once, or as three terms with all their bits
#pragma unroll
    for (int x = 0; x < TERMS; ++x) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(s[2 * k], s[2 * k + 1]);
        b[x][k] = transposed(*(const uint32_t*)&p);
        if (x + 1 < TERMS) {
          const float2 f = __bfloat1622float2(p);
          s[2 * k] -= f.x;
          s[2 * k + 1] -= f.y;
        }
      }
    }
#pragma unroll
    for (int jj = 0; jj < 8 * RUNS; ++jj) {
      const int u = jj / 8, j = jj % 8, k = j / 2 < MORE ? j / 2 : 0;
      const uint32_t sel = j % 2 ? 0x7632 : 0x5410;
      auto word = [&](const uint4& x) { return j / 2 == 0 ? x.x : j / 2 == 1 ? x.y : j / 2 == 2 ? x.z : x.w; };
      const uint32_t a0 = __byte_perm(word(v[u][0]), word(v[u][1]), sel), a2 = __byte_perm(word(v[u][2]), word(v[u][3]), sel);
      const uint32_t a1 = j / 2 < MORE ? __byte_perm(w[u][0][k], w[u][1][k], sel) : 0u;
      const uint32_t a3 = j / 2 < MORE ? __byte_perm(w[u][2][k], w[u][3][k], sel) : 0u;
#pragma unroll
      for (int x = 0; x < TERMS; ++x) mma_16x8(o[jj], a0, a1, a2, a3, b[x][0], b[x][1]);
    }
    fetch_values(at, left - 16 * OW_WARPS);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
    if (g == 0) {
      m_s[warp][2 * tq + x] = m[x];
      l_s[warp][2 * tq + x] = l[x];
    }
#pragma unroll
    for (int jj = 0; jj < 8 * RUNS; ++jj) {
      const int u = jj / 8, j = jj % 8;
      o_s[warp][2 * tq + x][u * 128 + g * 8 + j] = o[jj][x];
      if (j / 2 < MORE) o_s[warp][2 * tq + x][u * 128 + 64 + g * (MORE * 2) + j] = o[jj][2 + x];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (D / 4); i += OW_WARPS * 32) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float mm = m_s[0][h];
#pragma unroll
    for (int x = 1; x < OW_WARPS; ++x) mm = fmaxf(mm, m_s[x][h]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < OW_WARPS; ++x) {
      const float c = ex2_fast(m_s[x][h] - ref);
      const float4 y = *(const float4*)&o_s[x][h][d];
      ll = fmaf(l_s[x][h], c, ll);
      sum.x = fmaf(y.x, c, sum.x); sum.y = fmaf(y.y, c, sum.y); sum.z = fmaf(y.z, c, sum.z); sum.w = fmaf(y.w, c, sum.w);
    }
    if (result.out) {
      if (result.has_sink) ll += ex2_fast(result.sink * 1.4426950408889634f - ref);
      const float by = (ll > 0.f ? 1.f / ll : 0.f) * head_gate_of(result.gate, t, h0 + h);
      const float z[4] = {sum.x * by, sum.y * by, sum.z * by, sum.w * by};
#pragma unroll
      for (int x = 0; x < 4; ++x) st_dt(result.out, result.out_dt, ((size_t)t * a.Hq + h0 + h) * D + d + x, z[x]);
      continue;
    }
    const size_t at_p = ((size_t)r * a.Hq + h0 + h) * a.slots + split;
    *(float4*)(a.part_o + at_p * D + d) = sum;
    if (d == 0) {
      a.part_ml[at_p * 2] = mm == -INFINITY ? -1e30f : mm * 0.6931471805599453f;
      a.part_ml[at_p * 2 + 1] = ll;
    }
  }
  if (beside) grid_dep_wait();
}

// The parts of one (row, head): its own keys' splits, then the shared ones'.  W warps of a block take it, each every W-th part, eight
// loads of a lane under way, and add their sums in their order.  WIDE: heads of more than 128 elements.
constexpr int MAX_PARTS = 64, JOIN_WARPS = 4;

template <int W, bool WIDE>
__global__ void __launch_bounds__(JOIN_WARPS * 32) shared_join_kernel(const float* part_o, const float* part_ml,
                                                                      const int* __restrict__ rows, const int* __restrict__ group,
                                                                      void* out, int out_dt, int pairs, int Hq, int D, int own, int slots,
                                                                      int has_sink, float sink, HeadGate gate, int whole) {
  constexpr int C = WIDE ? 2 : 1, AT_ONCE = 8;
  __shared__ float4 sum_s[W > 1 ? JOIN_WARPS : 1][C * 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, sub = warp % W;
  const int pair = min((int)blockIdx.x * (JOIN_WARPS / W) + warp / W, pairs - 1), r = pair / Hq, h = pair % Hq, t = rows ? rows[r] : r;
  const int n = group && group[r] >= 0 ? slots : own;
  const size_t at = (size_t)pair * slots;
  grid_dep_wait();
  grid_dep_launch();
  const float2 none = make_float2(-1e30f, 0.f);
  const float2* ml = (const float2*)part_ml + at;
  const float2 x = lane < n ? __ldcg(ml + lane) : none, y = lane + 32 < n ? __ldcg(ml + lane + 32) : none;
  float4 o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  float wx = 0.f, wy = 0.f, by = 0.f;
  bool weighed = false;
  for (int s0 = sub; s0 < n || !weighed; s0 += AT_ONCE * W) {
    float4 v[AT_ONCE][C];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int s = s0 + i * W, d = (c * 32 + lane) * 4;
        v[i][c] = s < n && d < D ? __ldcg((const float4*)(part_o + (at + s) * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    if (!weighed) {                                  // (behind the loads, which need not wait for it)
      const float mm = warp_max(fmaxf(x.x, y.x));
      wx = expf(x.x - mm);
      wy = expf(y.x - mm);
      float ll = warp_sum(x.y * wx + y.y * wy);
      if (has_sink) ll += expf(sink - mm);
      by = (ll > 0.f ? 1.f / ll : 0.f) * head_gate_of(gate, t, h);
      weighed = true;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int s = s0 + i * W;
      const float w = __shfl_sync(0xffffffffu, s < 32 ? wx : wy, s % 32);
      if (s < n) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          o[c].x = fmaf(v[i][c].x, w, o[c].x); o[c].y = fmaf(v[i][c].y, w, o[c].y);
          o[c].z = fmaf(v[i][c].z, w, o[c].z); o[c].w = fmaf(v[i][c].w, w, o[c].w);
        }
      }
    }
  }
  if (W > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) sum_s[warp][c * 32 + lane] = o[c];
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int u = 1; u < W; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float4 p = sum_s[warp + u][c * 32 + lane];
        o[c].x += p.x; o[c].y += p.y; o[c].z += p.z; o[c].w += p.w;
      }
  }
  if ((int)blockIdx.x * (JOIN_WARPS / W) + warp / W >= pairs) return;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int d = (c * 32 + lane) * 4;
    if (d >= D) continue;
    const size_t to = ((size_t)t * Hq + h) * D + d;
    const float z[4] = {o[c].x * by, o[c].y * by, o[c].z * by, o[c].w * by};
    if (whole && out_dt == NV_DT_BF16) {
      const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(z[0], z[1]), __floats2bfloat162_rn(z[2], z[3])};
      *(uint2*)((bf16*)out + to) = *(const uint2*)b;
    } else if (whole) {
      *(float4*)((float*)out + to) = make_float4(z[0], z[1], z[2], z[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) st_dt(out, out_dt, to + i, z[i]);
    }
  }
}

template <typename T, int DC>
int launch_plain_d(const SharedArgs& a, int tiles, cudaStream_t s) {
  const size_t smem = (size_t)(SP_PAIRS + 2 * SP_KEYS) * (a.D + 4) * sizeof(float);
  static bool attr_done = false;
  if (!attr_done) {
    NV_RETURN_IF(cudaFuncSetAttribute(shared_plain_kernel<T, DC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (SP_PAIRS + 2 * SP_KEYS) * (DC + 4) * (int)sizeof(float)));
    attr_done = true;
  }
  NV_RETURN_IF(launch_dep(shared_plain_kernel<T, DC>, dim3(tiles, a.Hkv, a.splits), dim3(SP_THREADS), smem, s, a));
  NV_RETURN_LAST();
}
template <typename T>
int launch_plain(const SharedArgs& a, int tiles, cudaStream_t s) {
  return a.D <= 128 ? launch_plain_d<T, 128>(a, tiles, s) : launch_plain_d<T, 256>(a, tiles, s);
}

template <int D, int TERMS>
int launch_tc(const SharedArgs& a, int tiles, cudaStream_t s) {
  CUtensorMap tm_k, tm_v;
  const long long rows = (long long)a.num_pages * a.Hkv * a.page;
  int rc = nv_tensor_map_bf16(a.kc, rows, a.D, a.D, a.page, &tm_k);
  if (rc) return rc;
  rc = nv_tensor_map_bf16(a.vc, rows, a.D, a.D, a.page, &tm_v);
  if (rc) return rc;
  constexpr int SL = D / 64;
  constexpr size_t tiles_bytes = (size_t)SL * ST_PAIRS * 128 + (2 + st_v_buffers<D, TERMS>()) * (size_t)SL * ST_KEYS * 128 +
                                 (TERMS > 1 ? (size_t)TERMS * ST_PAIRS * 128 : 0);
  constexpr size_t smem = tiles_bytes + 1024;
  static_assert(tiles_bytes >= (size_t)ST_PAIRS * (D * 4 + 16), "a row of results has its place");
  constexpr auto capped_kernel = shared_tc_kernel<D, TERMS, true>, plain_kernel = shared_tc_kernel<D, TERMS, TERMS == 1>;
  static bool attr_done = false;
  if (!attr_done) {
    NV_RETURN_IF(cudaFuncSetAttribute(capped_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    NV_RETURN_IF(cudaFuncSetAttribute(plain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    attr_done = true;
  }
  // scores go to base-2 units by map.in; capped ones are there already
  ScoreMap map = shared_map(a.scale, a.softcap, TERMS);
  if (a.softcap > 0.f) map.in = 1.f;
  NV_RETURN_IF(launch_dep(a.softcap > 0.f ? capped_kernel : plain_kernel, dim3(tiles, a.Hkv, a.splits), dim3(ST_THREADS), smem, s, tm_k, tm_v, a, map));
  NV_RETURN_LAST();
}

template <int D, int TERMS>
int launch_own(const SharedArgs& a, const int* first, int R, int own_splits, int beside, const OwnResult& result, cudaStream_t s) {
  const int parts = (a.Hq / a.Hkv + OW_HEADS - 1) / OW_HEADS;
  NV_RETURN_IF(launch_dep(own_keys_kernel<D, TERMS>, dim3(R, a.Hkv * parts, own_splits), dim3(OW_WARPS * 32), 0, s, a, first, own_splits,
                          shared_map(a.scale, a.softcap, TERMS), beside, result));
  NV_RETURN_LAST();
}

template <int TERMS>
int launch_own_d(const SharedArgs& a, const int* first, int R, int own_splits, int beside, const OwnResult& result, cudaStream_t s) {
  return a.D == 64   ? launch_own<64, TERMS>(a, first, R, own_splits, beside, result, s)
         : a.D == 80 ? launch_own<80, TERMS>(a, first, R, own_splits, beside, result, s)
         : a.D == 96 ? launch_own<96, TERMS>(a, first, R, own_splits, beside, result, s)
         : a.D == 128 ? launch_own<128, TERMS>(a, first, R, own_splits, beside, result, s)
                      : launch_own<256, TERMS>(a, first, R, own_splits, beside, result, s);
}
template <int TERMS>
int launch_tc_d(const SharedArgs& a, int tiles, cudaStream_t s) {
  return a.D <= 64 ? launch_tc<64, TERMS>(a, tiles, s) : a.D <= 128 ? launch_tc<128, TERMS>(a, tiles, s) : launch_tc<256, TERMS>(a, tiles, s);
}

// Keys of a split at least.
constexpr int TC_SPLIT_KEYS = 256, PLAIN_SPLIT_KEYS = 64;

// Whether the tensor-core form takes these sizes (and, with pointers, these addresses).
bool tc_takes(int cache_dt, int D, int page) {
  return cache_dt == NV_DT_BF16 && D >= 32 && D % 16 == 0 && (page == 16 || page == 32 || page == 64);
}
// (The head sizes of the models here and of the measured range.  Others, such as the 112, 160 and 192 that heads can be padded to, take the
// split-key kernel.)
bool own_takes(int D) { return D == 64 || D == 80 || D == 96 || D == 128 || D == 256; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Tiles of pairs that M rows in `groups` groups make at most.
long long shared_tiles(int M, int groups, int Hq, int Hkv, int per_tile) {
  return ((long long)M * (Hq / Hkv) + per_tile - 1) / per_tile + groups - 1;
}
}  // namespace

namespace {
template <int W>
int launch_join(const float* part_o, const float* part_ml, const int* rows, const int* group, void* out, int out_dt, int R, int Hq, int D,
                int own, int slots, int has_sink, float sink, const HeadGate& gate, cudaStream_t s) {
  const long long pairs = (long long)R * Hq, blocks = (pairs * W + JOIN_WARPS - 1) / JOIN_WARPS;
  if (pairs > 0x7fffffffLL) return NV_ERR_BAD_SIZE;
  const int whole = ((uintptr_t)out & 15) == 0;                      // (four elements in one store)
  NV_RETURN_IF(D > 128 ? launch_dep(shared_join_kernel<W, true>, dim3((unsigned)blocks), dim3(JOIN_WARPS * 32), 0, s, part_o, part_ml, rows, group,
                                    out, out_dt, (int)pairs, Hq, D, own, slots, has_sink, sink, gate, whole)
                       : launch_dep(shared_join_kernel<W, false>, dim3((unsigned)blocks), dim3(JOIN_WARPS * 32), 0, s, part_o, part_ml, rows, group,
                                    out, out_dt, (int)pairs, Hq, D, own, slots, has_sink, sink, gate, whole));
  NV_RETURN_LAST();
}
}  // namespace

// Splits of the shared keys for M rows in `groups` groups whose longest prefix has `longest` positions: as many blocks as live on
// the GPU at once (two a multiprocessor, one of the larger forms), 256 keys a split or more.  (64 rows of 28 heads on 4 behind 8,192
// positions, 16 splits: 38.4 us; 9: 44.0, 32: 46.3.  128 behind 16,384, 10: 61; 6: 74, 18: 70.)
NV_API int nv_attention_shared_splits(int M, int groups, int Hq, int Hkv, int D, int page, int cache_dt, int float_weights, int longest) {
  if (M <= 0 || groups <= 0 || longest <= 0 || Hkv <= 0) return 0;
  const bool tc = tc_takes(cache_dt, D, page);
  const int each = tc ? (D <= 128 && !float_weights ? 2 : 1) : 4, least = tc ? TC_SPLIT_KEYS : PLAIN_SPLIT_KEYS;
  const long long tiles = shared_tiles(M, groups, Hq, Hkv, tc ? ST_PAIRS : SP_PAIRS);
  const long long want = (long long)each * num_multiprocessors() / (tiles * Hkv), most = (longest + least - 1) / least;
  long long n = want < most ? want : most;
  n = n < 1 ? 1 : n > 32 ? 32 : n;
  const long long block = tc ? ST_KEYS : SP_KEYS, share = ((longest + n - 1) / n + block - 1) / block * block;
  return (int)((longest + share - 1) / share);                       // (no split without keys)
}

// Splits of the rows' own keys, of which no row has more than `most`, beside shared_splits of the above.  Where the shared part leaves
// room, they run beside it, one block on its multiprocessors and three on the others, 128 keys a split or more, and a second wave
// would come after it (eight rows of 16 heads behind 2,048: 11.8 us in one wave, 15.3 in two); where it fills the GPU they come
// after it anyway, 256 keys a split or more unless 128 make one wave (64 rows of 28 heads on 4 behind 8,192, up to 512 of their own:
// one split 38.5, two 34.1, four 36.2; up to 1,000: 49.1, 39.0, 38.1; four of 16 behind 16,384, up to 200: 33.2, two 31.1).  A block takes
// eight heads of the own-key kernel, 16 of the split-key kernel (44 rows of 32 heads on 2 behind 1,000, up to 300 of their own: 13.1 in one
// wave, 18.7 in three splits; 40 rows of 64 heads of 64 on 4 that share nothing, up to 700: 11.4 and 14.8 in two).  Heads of more than 128
// elements: 384 keys a split at most, whose time is beyond that of a second wave (64 rows of 16 heads of 256 on 1 behind 8,192, up to 512 of
// their own: one split 44.6, two 37.7; up to 1,000: 59.5, 46.0, three 45.1; 44 behind 1,000, up to 300: 16.3 and 16.0).
NV_API int nv_attention_shared_own_splits(int R, int M, int groups, int Hq, int Hkv, int D, int page, int cache_dt, int shared_splits,
                                          int most) {
  if (R <= 0 || Hkv <= 0 || most <= 0) return 1;
  const int G = Hq / Hkv, heads = tc_takes(cache_dt, D, page) && own_takes(D) ? OW_HEADS : 16;      // of a block
  const long long sms = num_multiprocessors(), blocks = (long long)R * Hkv * ((G + heads - 1) / heads);
  const long long shared = shared_splits <= 0 ? 0 : shared_tiles(M, groups, Hq, Hkv, tc_takes(cache_dt, D, page) ? ST_PAIRS : SP_PAIRS) * Hkv * shared_splits;
  const long long room = shared <= sms ? shared + (D > 128 ? 2 : 3) * (sms - shared) : 7 * sms;
  long long n = room / blocks;
  const long long least = shared <= sms || blocks * ((most + 127) / 128) <= 3 * sms ? 128 : 256;
  if (n > (most + least - 1) / least) n = (most + least - 1) / least;
  if (D > 128 && shared > 0 && n < (most + 383) / 384) n = (most + 383) / 384;
  return (int)(n < 1 ? 1 : n > 32 ? 32 : n);
}

// Whether `repeated` positions that need not be read again are worth a kernel more and a join (1) or not (0), in bytes of keys and
// values.  Tensor-core form: 24 MB, and 32 KB for every row and kv head, whose parts are joined.  (Calls behind one another would have
// it pay about as soon: shared and not, four rows of 16 kv heads behind 1,000 positions, 24 MB, 10.5 and 11.2 us, behind 1,500, 37 MB,
// 10.5 and 12.8; eight of 4 behind 1,500, 22 MB, 11.7 and 10.9, behind 2,048, 29 MB, 11.6 and 12.3, behind 4,000, 57 MB, 12.6 and 15.5;
// 64 of 16 behind 64, 33 MB, 17.1 and 16.2, behind 128, 66 MB, 18.0 and 20.5; 16 rows of 16 heads of 256 on 1 behind 1,000, 15 MB,
// 14.9 and 13.6, behind 2,000, 31 MB, 15.3 and 23.1.  In a model's step the kernel without groups begins beside the one in front, and the step
// has to look for groups: 16 layers with eight rows of 4 behind 1,500 take 2.26 and 2.27 ms without and with groups, behind 2,048 2.28
// either way, 32 rows behind 1,024, 65 MB, 2.74 and 2.65.)  Plain form: 192 KB
// for every row and kv head, since the kernel without groups is slow at few rows of these
// types (four float32 rows of 8 heads on 2 behind 500, 3 MB, 15.6 and 21.5; 32 of 28 on 4 behind 128, 16 MB, 30.1 and 25.9, behind
// 256, 33 MB, 34.8 and 44.6), and half a tile of pairs a group (four rows of 16 on 16 behind 1,000, 49 MB, 21.1 and 15.1).
NV_API int nv_attention_shared_pays(int R, int M, int groups, int Hq, int Hkv, int D, int page, int cache_dt, long long repeated) {
  if (groups <= 0 || Hkv <= 0) return 0;
  const long long saved = repeated * Hkv * D * 2 * (cache_dt == NV_DT_BF16 ? 2 : 4), parts = (long long)R * Hkv;
  if (tc_takes(cache_dt, D, page)) return saved >= (24LL << 20) + 32768 * parts;
  return saved >= 196608 * parts && 2LL * M * (Hq / Hkv) >= (long long)SP_PAIRS * groups;
}

// Whether rows that share nothing take the own-key kernel and, from two parts on, the join instead of the split-key kernel: its types
// and sizes (both: 40 rows of 28 heads on 4, 400 to 700 positions, 16.8 and 21.4 us, in pages of 32 16.8 and 21.1; two behind 4,000 9.1 and
// 13.1; four of 16 on 16 behind 496 9.4 and 9.6; eight of 16 heads of 256 on 1 behind 300, pages of 32, 9.5 and 32.7).
NV_API int nv_attention_shared_alone(int D, int page, int cache_dt) {
  return tc_takes(cache_dt, D, page) && own_takes(D) ? 1 : 0;
}

NV_API int nv_attention_shared_usable(int D, int page) { return D >= 8 && D <= 256 && D % 8 == 0 && page >= 16 && page % 16 == 0; }

// R rows (rows: their batch rows, nullptr: all); first [R]: positions of the row that are shared (0 without a group), group [R]: its
// group or -1 (both nullptr: none shares, see nv_attention_shared_alone), members [M], cu [groups + 1], len and lead [groups]: see
// SharedArgs.  own_splits and shared_splits parts a (row, head);
// scratch: R * Hq * (own_splits + shared_splits) * (D + 2) floats.
NV_API int nv_attention_decode_shared(const void* qkv, int q_dt, int q_stride, const void* kc, const void* vc, int cache_dt,
                                      const int* block_table, int max_blocks, const int* row_entry, const int* positions,
                                      const int* rows, int R, const int* first, const int* group, const int* members, int M,
                                      const int* cu, const int* len, const int* lead, int groups, float scale, void* out, int out_dt, int Hq, int Hkv,
                                      int D, int page, int num_pages, int own_splits, int shared_splits, float* scratch, int* err,
                                      int has_sink, float sink_score, int float_weights, float softcap, const float* gate,
                                      long long gate_ld, cudaStream_t stream) {
  if (!dt_ok(q_dt) || !dt_ok(cache_dt) || !dt_ok(out_dt)) return NV_ERR_BAD_DTYPE;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || !nv_attention_shared_usable(D, page) || !(scale > 0.f)) return NV_ERR_UNSUPPORTED;
  if (R < 0 || M < 0 || groups < 0 || own_splits < 1 || shared_splits < 0 || own_splits + shared_splits > MAX_PARTS || num_pages < 1)
    return NV_ERR_BAD_SIZE;
  if (R == 0) return NV_OK;
  if (!aligned16(kc) || !aligned16(vc)) return NV_ERR_UNSUPPORTED;
  if (!scratch || ((uintptr_t)scratch & 15)) return NV_ERR_BAD_SIZE;
  const int slots = own_splits + shared_splits;
  const bool tc = tc_takes(cache_dt, D, page) && q_dt == NV_DT_BF16 && q_stride % 8 == 0 && aligned16(qkv) && aligned16(kc) && aligned16(vc);
  const int exact = (float_weights || has_sink) ? 1 : 0, beside = shared_splits > 0 && groups > 0 ? 1 : 0;
  SharedArgs a;
  a.q = qkv; a.kc = kc; a.vc = vc; a.block_table = block_table; a.row_entry = row_entry; a.positions = positions; a.rows = rows;
  a.members = members; a.cu = cu; a.len = len; a.lead = lead; a.part_o = scratch; a.part_ml = scratch + (size_t)R * Hq * slots * D; a.err = err;
  a.scale = scale; a.softcap = softcap > 0.f ? softcap : 0.f; a.q_dt = q_dt; a.q_stride = q_stride; a.max_blocks = max_blocks;
  a.num_pages = num_pages; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.page = page; a.groups = groups; a.splits = shared_splits;
  a.slots = slots; a.slot0 = own_splits; a.split_keys = tc ? TC_SPLIT_KEYS : PLAIN_SPLIT_KEYS;
  if (beside) {
    const int tiles = (int)shared_tiles(M, groups, Hq, Hkv, tc ? ST_PAIRS : SP_PAIRS);
    const int rc = !tc ? (cache_dt == NV_DT_BF16 ? launch_plain<bf16>(a, tiles, stream) : launch_plain<float>(a, tiles, stream))
                   : exact ? launch_tc_d<3>(a, tiles, stream) : launch_tc_d<1>(a, tiles, stream);
    if (rc) return rc;
  }
  const HeadGate gated{gate, gate_ld};
  const bool direct = tc && own_takes(D) && slots == 1 && !beside;
  const OwnResult result{direct ? out : nullptr, out_dt, has_sink, sink_score, gated};
  const int rc = tc && own_takes(D) ? (exact ? launch_own_d<3>(a, first, R, own_splits, beside, result, stream)
                                             : launch_own_d<1>(a, first, R, own_splits, beside, result, stream))
                 : !first ? NV_ERR_UNSUPPORTED
                 : nv_attention_decode_rest(qkv, q_dt, q_stride, kc, vc, cache_dt, block_table, max_blocks, row_entry, positions, rows,
                                            first, R, scale, out_dt, Hq, Hkv, D, page, num_pages, own_splits, slots, scratch, err, exact,
                                            softcap, beside, stream);
  if (rc || direct) return rc;
  // A warp a pair where there are many with few parts, else two (128 rows of 28 heads, 11 parts: 51.4 and 52.2 us; 64 rows, 18: 35.1 and
  // 34.0; 50 of 24, three terms, 9: 17.9 and 16.9).
  return slots <= 12 && (long long)R * Hq >= 2048
             ? launch_join<1>(a.part_o, a.part_ml, rows, group, out, out_dt, R, Hq, D, own_splits, slots, has_sink, sink_score, gated, stream)
             : launch_join<2>(a.part_o, a.part_ml, rows, group, out, out_dt, R, Hq, D, own_splits, slots, has_sink, sink_score, gated, stream);
}

// The same with what a step's layers have in common in one array on the host (fewer arguments to convert a call): type of queries,
// cache and result; Hq, Hkv, D, page; R, first, group, members, M, cu, len, lead, groups; own_splits, shared_splits, float_weights.
NV_API int nv_attention_decode_shared_plan(const long long* plan, const void* qkv, int q_stride, const void* kc, const void* vc,
                                           const int* block_table, int max_blocks, const int* row_entry, const int* positions,
                                           const int* rows, float scale, void* out, int num_pages, float* scratch, int* err,
                                           int has_sink, float sink_score, float softcap, const float* gate, long long gate_ld,
                                           cudaStream_t stream) {
  const int dt = (int)plan[0];
  return nv_attention_decode_shared(qkv, dt, q_stride, kc, vc, dt, block_table, max_blocks, row_entry, positions, rows, (int)plan[5],
                                    (const int*)plan[6], (const int*)plan[7], (const int*)plan[8], (int)plan[9], (const int*)plan[10],
                                    (const int*)plan[11], (const int*)plan[12], (int)plan[13], scale, out, dt, (int)plan[1],
                                    (int)plan[2], (int)plan[3], (int)plan[4], num_pages, (int)plan[14], (int)plan[15], scratch, err,
                                    has_sink, sink_score, (int)plan[16], softcap, gate, gate_ld, stream);
}
