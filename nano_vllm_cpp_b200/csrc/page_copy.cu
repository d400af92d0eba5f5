// Copies of pages between places of a cache, in all of its arrays at once: what a fork of a request needs (the page that is
// part full, or a state slot, once per reply), in one launch for a model's keys and values of every layer.
//
// An array is [pages][heads][slots][bytes]; copy i takes the first slots[i] slots of every head of page src[i] to page dst[i]
// and leaves the others as they were.  The destinations are distinct and none of them is a source, so that the order of the
// copies does not matter.  The kernel is launched the ordinary way and lets no dependent start early: the attention kernels
// read the older pages of their rows before the kernel in front of them has ended.
//
// What bounds it: the bytes.  Four sequences of 128 pages, 48 arrays, 3.2 GB read and written: 481 us, 6.7 TB/s; eight copies of a
// state of 25 MB (225 MB, most of them written) 46 us, 4.9 TB/s; a fork's part-full pages the latency of a launch and two
// loads in turn (the array's description beside the copy's places, then the source) and a store.
#include "common.cuh"

namespace {

struct PageArray {              // what the host puts into the table of arrays, eight 8-byte words an array
  unsigned long long base;
  long long page_bytes, heads, head_bytes, slot_bytes, slots, pages, unit;
};

constexpr int PC_WARPS = 8;              // warps of a block
constexpr int PC_SHARE = 4096, PC_LEAST = 1024;      // bytes of a page a warp: the former, or less where there are few copies
constexpr int PC_RUN = 8;                // copies of one source that a warp writes at most
constexpr int PC_AT_ONCE = 4;            // loads of a lane under way

// A warp's share of `all` units, of which every head has per_head one after the other: runs of 32 units, `share` warps in turn.
template <typename U>
__device__ __forceinline__ void copy_units(const PageArray& a, const char* from, char* const* to, int copies, long long n, int c,
                                           int share, int lane) {
  const long long per = n * a.slot_bytes / (long long)sizeof(U);
  const bool flat = n == a.slots;                                    // whole heads lie one after the other
  const unsigned per_head = (unsigned)(flat ? 1 : per);
  const long long all = per * a.heads, step = 32LL * share;
  for (long long i0 = 32LL * c + lane; i0 < all; i0 += PC_AT_ONCE * step) {
    U v[PC_AT_ONCE];
    long long at[PC_AT_ONCE];
#pragma unroll
    for (int k = 0; k < PC_AT_ONCE; ++k) {
      const long long i = i0 + k * step;
      at[k] = i * (long long)sizeof(U);
      if (!flat) {                                                   // (a page is far below 2^32 units, or is copied whole)
        const unsigned h = (unsigned)i / per_head;
        at[k] = h * a.head_bytes + (long long)((unsigned)i - h * per_head) * (long long)sizeof(U);
      }
      if (i < all) v[k] = *(const U*)(from + at[k]);
    }
    for (int j = 0; j < copies; ++j) {
      char* const dst = to[j];
#pragma unroll
      for (int k = 0; k < PC_AT_ONCE; ++k)
        if (i0 + k * step < all) *(U*)(dst + at[k]) = v[k];
    }
  }
}

// A block row per array, `share` warps per copy.  Copies of one source that stand beside one another (a fork's) are made by the first
// one's warps, up to PC_RUN of them, so that the source is read once.
__global__ void __launch_bounds__(PC_WARPS * 32) copy_pages_kernel(const PageArray* __restrict__ arrays, const int* __restrict__ src,
                                                                   const int* __restrict__ dst, const int* __restrict__ slots, int N,
                                                                   int share, int* err) {
  __shared__ char* to_s[PC_WARPS][PC_RUN];
  const PageArray a = arrays[blockIdx.y];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long w = (long long)blockIdx.x * PC_WARPS + warp;
  const int i = (int)(w / share), c = (int)(w % share);
  if (i >= N) return;
  // the copies i .. i + 7 as far as they lie in one window of eight: a lane looks at one of them
  const int j = i + lane;
  const bool there = lane < PC_RUN - i % PC_RUN && j < N;
  const int s = there ? src[j] : -1, d = there ? dst[j] : -1, n_here = there && slots ? slots[j] : -1;
  const int s0 = __shfl_sync(0xffffffffu, s, 0), n0 = __shfl_sync(0xffffffffu, n_here, 0);
  if (i % PC_RUN && src[i - 1] == s0 && (!slots || slots[i - 1] == n0)) return;      // (an earlier copy's warps make this one)
  const uint32_t same = __ballot_sync(0xffffffffu, there && s == s0 && n_here == n0);
  const int run = __ffs(~same) - 1;
  const bool fine = lane < run && s >= 0 && s < a.pages && d >= 0 && d < a.pages;
  if (lane < run && !fine && err) atomicExch(err, 1 + j);
  const uint32_t good = __ballot_sync(0xffffffffu, fine && d != s);
  if (good >> lane & 1u) to_s[warp][__popc(good & ((1u << lane) - 1u))] = (char*)a.base + d * a.page_bytes;
  __syncwarp();
  if (!good) return;
  const long long n = slots ? min(max((long long)n0, 0LL), a.slots) : a.slots;
  const char* from = (const char*)a.base + s0 * a.page_bytes;
  char* const* to = to_s[warp];
  switch ((int)a.unit) {
    case 16: copy_units<uint4>(a, from, to, __popc(good), n, c, share, lane); break;
    case 8: copy_units<uint2>(a, from, to, __popc(good), n, c, share, lane); break;
    case 4: copy_units<uint32_t>(a, from, to, __popc(good), n, c, share, lane); break;
    default: copy_units<uint16_t>(a, from, to, __popc(good), n, c, share, lane);
  }
}

}  // namespace

// arrays: [A][8] 64-bit words on the device (address, bytes of a page, heads, bytes of a head, bytes of a slot, slots of a page,
// pages, bytes of the widest access that address and sizes allow); src, dst, slots [N] on the device (slots may be
// nullptr: whole pages).  A page outside an array sets the error flag to 1 + the copy and is not copied.
NV_API int nv_copy_pages(const void* arrays, int A, long long page_bytes, const int* src, const int* dst, const int* slots, int N,
                         int* err, cudaStream_t s) {
  if (A < 0 || N < 0 || A > 65535 || page_bytes < 0) return NV_ERR_BAD_SIZE;
  if (A == 0 || N == 0) return NV_OK;
  // (one request's page forked into seven, 48 arrays, 45 of 64 KB: 4 KB a warp 12.4 us, 2 KB 10.0; 64 forked into four, 56 arrays,
  // 5 of 16 KB: 20.6 and 30.4)
  long long share = (page_bytes + PC_SHARE - 1) / PC_SHARE;
  const long long fill = 4LL * 64 * num_multiprocessors() / ((long long)A * N), most = (page_bytes + PC_LEAST - 1) / PC_LEAST;
  if (share < fill) share = fill < most ? fill : most;
  share = share < 1 ? 1 : share > 16384 ? 16384 : share;
  const long long blocks = (N * share + PC_WARPS - 1) / PC_WARPS;
  if (blocks > 0x7fffffffLL) return NV_ERR_BAD_SIZE;
  copy_pages_kernel<<<dim3((unsigned)blocks, (unsigned)A), PC_WARPS * 32, 0, s>>>((const PageArray*)arrays, src, dst, slots, N, (int)share, err);
  NV_RETURN_LAST();
}
