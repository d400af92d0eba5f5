// Decode attention for rows that share a prefix: several replies to one prompt, or requests behind one system prompt.
//
// The rows of a group hold the same keys and values at their first len[g] positions.  The whole pages of these are read once,
// through the block table of the group's first row; a page that the prefix ends in every row reads for itself.  A row's softmax over all its keys is put together from parts with sums of their own,
//
//   m = max over the part of s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j;      out = sum_p e^(m_p - M) o_p / sum_p e^(m_p - M) l_p
//
// so the shared part can be worked out for all rows of the group at once, its keys and values read once instead of once a
// row: per kv head it is a matrix product of the (row, query head) pairs that read it.  Three launches: the shared parts (here),
// every row's own keys, from the page on that holds position len[g] (the split-key kernel of attention_decode.cu), and their join (here).  A row that
// belongs to no group has no shared part; of a group's keys a row sees those up to its own position.
#include "pipeline.cuh"

int nv_attention_decode_rest(const void* qkv, int q_dt, int q_stride, const void* kc, const void* vc, int cache_dt,
                             const int* block_table, int max_blocks, const int* row_entry, const int* positions, const int* rows,
                             const int* first, int R, float scale, int out_dt, int Hq, int Hkv, int D, int page, int num_pages,
                             int splits, int slots, float* scratch, int* err, int float_weights, float softcap, cudaStream_t stream);

namespace {

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
  float* part_o;            // [R, Hq, slots, D]
  float* part_ml;           // [R, Hq, slots, 2]
  int* err;
  float scale, softcap;
  int q_dt, q_stride, max_blocks, num_pages, Hq, Hkv, D, page, groups, splits, slots, slot0;
  int split_keys;           // a split has at least so many keys (a multiple of the page and of the kernel's block of keys)
};

// Which tile of `rows_per_tile` pairs of which group is tile number x?  Found by one thread; tile.x < 0: none (a launch has as many
// tiles as there may be).
__device__ __forceinline__ int2 find_tile(const SharedArgs& a, int x, int G, int rows_per_tile) {
  for (int g = 0; g < a.groups; ++g) {
    const int pairs = (a.cu[g + 1] - a.cu[g]) * G, tiles = (pairs + rows_per_tile - 1) / rows_per_tile;
    if (x < tiles) return make_int2(g, x * rows_per_tile);
    x -= tiles;
  }
  return make_int2(-1, 0);
}

// The plain form: any type, any head size in steps of eight, float32 products.  A block takes 16 pairs of one kv head and one
// split of the keys, 32 keys at a time; eight threads share a pair.
constexpr int SP_PAIRS = 16, SP_KEYS = 32, SP_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(SP_THREADS) shared_plain_kernel(SharedArgs a) {
  extern __shared__ __align__(16) float sp_smem[];
  const int D = a.D, LD = D + 4;
  float* q_s = sp_smem;                          // [SP_PAIRS][LD]
  float* kv_s = q_s + SP_PAIRS * LD;             // [SP_KEYS][LD]
  __shared__ float p_s[SP_PAIRS][SP_KEYS + 1];
  __shared__ int2 tile_s;
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, kvh = blockIdx.y, split = blockIdx.z, G = a.Hq / a.Hkv;
  if (tid == 0) tile_s = find_tile(a, blockIdx.x, G, SP_PAIRS);
  __syncthreads();
  const int g = tile_s.x, pair0 = tile_s.y;
  if (g < 0) return;
  const int m0 = a.cu[g], pairs = (a.cu[g + 1] - m0) * G, len = a.len[g] / a.page * a.page;
  const int lead = a.members[m0], lead_t = a.rows ? a.rows[lead] : lead;
  const int* bt = a.block_table + (long long)a.row_entry[lead_t] * a.max_blocks;
  const int share = max(a.split_keys, ((len + a.splits - 1) / a.splits + SP_KEYS - 1) / SP_KEYS * SP_KEYS);
  const int j_lo = min(len, split * share), j_hi = min(len, j_lo + share);

  const int i = tid / 8, sub = tid % 8;          // this thread's pair of the tile, and which of its eight threads it is
  const bool live = pair0 + i < pairs;
  const int r = live ? a.members[m0 + (pair0 + i) / G] : lead, h = kvh * G + (live ? (pair0 + i) % G : 0);
  const int t = a.rows ? a.rows[r] : r;
  const int limit = live ? min(j_hi, a.positions[t] + 1) : 0;        // the first key that this row does not see
  for (int d = sub; d < D; d += 8) q_s[i * LD + d] = live ? ld_dt(a.q, a.q_dt, (size_t)t * a.q_stride + (size_t)h * D + d) * a.scale : 0.f;

  float m = -INFINITY, l = 0.f, o[8][4];
#pragma unroll
  for (int c = 0; c < 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
  const int chunks = D / 4;
  auto load = [&](const void* cache, int j0) {   // SP_KEYS keys (or values) as floats, zeros beyond the split
    for (int x = tid; x < SP_KEYS * (D / 8); x += SP_THREADS) {
      const int key = x / (D / 8), c = x % (D / 8), j = j0 + key;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (j < j_hi) {
        const int blk = bt[j / a.page];
        if (blk >= 0 && blk < a.num_pages) {
          const T* p = (const T*)cache + (((size_t)blk * a.Hkv + kvh) * a.page + j % a.page) * D + c * 8;
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = to_f32(p[u]);
        } else if (a.err) {
          atomicExch(a.err, 1 + lead_t);
        }
      }
      *(float4*)&kv_s[key * LD + c * 8] = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)&kv_s[key * LD + c * 8 + 4] = make_float4(v[4], v[5], v[6], v[7]);
    }
  };
  for (int j0 = j_lo; j0 < j_hi; j0 += SP_KEYS) {
    __syncthreads();
    load(a.kc, j0);
    __syncthreads();
    float s[SP_KEYS / 8];
#pragma unroll
    for (int u = 0; u < SP_KEYS / 8; ++u) s[u] = 0.f;
    for (int c = 0; c < chunks; ++c) {
      const float4 qv = *(const float4*)&q_s[i * LD + c * 4];
#pragma unroll
      for (int u = 0; u < SP_KEYS / 8; ++u) {
        const float4 kv = *(const float4*)&kv_s[(u * 8 + sub) * LD + c * 4];
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
    __syncthreads();
    load(a.vc, j0);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int at = (c * 8 + sub) * 4;
      if (at < D) {
        float4 acc = make_float4(o[c][0] * alpha, o[c][1] * alpha, o[c][2] * alpha, o[c][3] * alpha);
        for (int key = 0; key < SP_KEYS; ++key) {
          const float p = p_s[i][key];
          const float4 v = *(const float4*)&kv_s[key * LD + at];
          acc.x = fmaf(p, v.x, acc.x); acc.y = fmaf(p, v.y, acc.y); acc.z = fmaf(p, v.z, acc.z); acc.w = fmaf(p, v.w, acc.w);
        }
        o[c][0] = acc.x; o[c][1] = acc.y; o[c][2] = acc.z; o[c][3] = acc.w;
      }
    }
  }
  if (!live) return;
  const size_t at = ((size_t)r * a.Hq + h) * a.slots + a.slot0 + split;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int d = (c * 8 + sub) * 4;
    if (d < D)
#pragma unroll
      for (int u = 0; u < 4; ++u) a.part_o[at * D + d + u] = o[c][u];
  }
  if (sub == 0) {
    a.part_ml[at * 2] = m == -INFINITY ? -1e30f : m;
    a.part_ml[at * 2 + 1] = l;
  }
}

// The parts of one (row, head), in the order of their slots: its own keys' splits, then the shared ones'.
__global__ void __launch_bounds__(128) shared_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                          const int* __restrict__ rows, const int* __restrict__ group, void* out,
                                                          int out_dt, int Hq, int D, int own, int slots, int has_sink, float sink,
                                                          HeadGate gate) {
  grid_dep_wait();
  grid_dep_launch();
  const int r = blockIdx.x, h = blockIdx.y, t = rows ? rows[r] : r;
  const int n = group[r] >= 0 ? slots : own;
  const size_t at = ((size_t)r * Hq + h) * slots;
  float mm = -1e30f, ll = 0.f;
  for (int s = 0; s < n; ++s) mm = fmaxf(mm, part_ml[(at + s) * 2]);
  for (int s = 0; s < n; ++s) ll = fmaf(part_ml[(at + s) * 2 + 1], expf(part_ml[(at + s) * 2] - mm), ll);
  if (has_sink) ll += expf(sink - mm);
  const float by = (ll > 0.f ? 1.f / ll : 0.f) * head_gate_of(gate, t, h);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float o = 0.f;
    for (int s = 0; s < n; ++s) o = fmaf(part_o[(at + s) * D + d], expf(part_ml[(at + s) * 2] - mm), o);
    st_dt(out, out_dt, ((size_t)t * Hq + h) * D + d, o * by);
  }
}

template <typename T>
int launch_plain(const SharedArgs& a, int tiles, cudaStream_t s) {
  const size_t smem = (size_t)(SP_PAIRS + SP_KEYS) * (a.D + 4) * sizeof(float);
  static bool attr_done = false;
  if (!attr_done) {
    NV_RETURN_IF(cudaFuncSetAttribute(shared_plain_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
    attr_done = true;
  }
  NV_RETURN_IF(launch_dep(shared_plain_kernel<T>, dim3(tiles, a.Hkv, a.splits), dim3(SP_THREADS), smem, s, a));
  NV_RETURN_LAST();
}

}  // namespace

// Splits of the shared keys for M rows in `groups` groups whose longest prefix has `longest` positions.
NV_API int nv_attention_shared_splits(int M, int groups, int Hq, int Hkv, int longest) {
  if (M <= 0 || groups <= 0 || longest <= 0 || Hkv <= 0) return 0;
  const int G = Hq / Hkv;
  const long long tiles = ((long long)M * G + SP_PAIRS - 1) / SP_PAIRS + groups;
  const long long blocks = tiles * Hkv, want = (4LL * num_multiprocessors() + blocks - 1) / blocks;
  const long long most = (longest + 255) / 256;
  const long long n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 32 ? 32 : n);
}

NV_API int nv_attention_shared_usable(int D, int page) { return D >= 8 && D <= 256 && D % 8 == 0 && page >= 16 && page % 16 == 0; }

// R rows (rows: their batch rows, nullptr: all); first [R]: positions of the row that are shared (0 without a group), group [R]: its
// group or -1, members [M], cu [groups + 1], len [groups]: see SharedArgs.  own_splits and shared_splits parts a (row, head);
// scratch: R * Hq * (own_splits + shared_splits) * (D + 2) floats.
NV_API int nv_attention_decode_shared(const void* qkv, int q_dt, int q_stride, const void* kc, const void* vc, int cache_dt,
                                      const int* block_table, int max_blocks, const int* row_entry, const int* positions,
                                      const int* rows, int R, const int* first, const int* group, const int* members, int M,
                                      const int* cu, const int* len, int groups, float scale, void* out, int out_dt, int Hq, int Hkv,
                                      int D, int page, int num_pages, int own_splits, int shared_splits, float* scratch, int* err,
                                      int has_sink, float sink_score, int float_weights, float softcap, const float* gate,
                                      long long gate_ld, cudaStream_t stream) {
  if (!dt_ok(q_dt) || !dt_ok(cache_dt) || !dt_ok(out_dt)) return NV_ERR_BAD_DTYPE;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || !nv_attention_shared_usable(D, page) || !(scale > 0.f)) return NV_ERR_UNSUPPORTED;
  if (R < 0 || M < 0 || groups < 0 || own_splits < 1 || shared_splits < 0 || num_pages < 1) return NV_ERR_BAD_SIZE;
  if (R == 0) return NV_OK;
  if (!scratch) return NV_ERR_BAD_SIZE;
  const int slots = own_splits + shared_splits;
  const long long tiles = ((long long)M * (Hq / Hkv) + SP_PAIRS - 1) / SP_PAIRS + groups;
  if (shared_splits > 0 && groups > 0) {
    SharedArgs a;
    a.q = qkv; a.kc = kc; a.vc = vc; a.block_table = block_table; a.row_entry = row_entry; a.positions = positions; a.rows = rows;
    a.members = members; a.cu = cu; a.len = len; a.part_o = scratch; a.part_ml = scratch + (size_t)R * Hq * slots * D; a.err = err;
    a.scale = scale; a.softcap = softcap > 0.f ? softcap : 0.f; a.q_dt = q_dt; a.q_stride = q_stride; a.max_blocks = max_blocks;
    a.num_pages = num_pages; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.page = page; a.groups = groups; a.splits = shared_splits;
    a.slots = slots; a.slot0 = own_splits; a.split_keys = 256;
    const int rc = cache_dt == NV_DT_BF16 ? launch_plain<bf16>(a, (int)tiles, stream) : launch_plain<float>(a, (int)tiles, stream);
    if (rc) return rc;
  }
  const int rc = nv_attention_decode_rest(qkv, q_dt, q_stride, kc, vc, cache_dt, block_table, max_blocks, row_entry, positions, rows,
                                          first, R, scale, out_dt, Hq, Hkv, D, page, num_pages, own_splits, slots, scratch, err,
                                          (float_weights || has_sink) ? 1 : 0, softcap, stream);
  if (rc) return rc;
  NV_RETURN_IF(launch_dep(shared_join_kernel, dim3(R, Hq), dim3(128), 0, stream, (const float*)scratch,
                          (const float*)scratch + (size_t)R * Hq * slots * D, rows, group, out, out_dt, Hq, D, own_splits, slots,
                          has_sink, sink_score, HeadGate{gate, gate_ld}));
  NV_RETURN_LAST();
}
