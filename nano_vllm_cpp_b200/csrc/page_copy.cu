// Copies of pages between places of a cache, in all of its arrays at once: what a fork of a request needs (the page that is
// part full, or a state slot, once per reply), in one launch for a model's keys and values of every layer.
//
// An array is [pages][heads][slots][bytes]; copy i takes the first slots[i] slots of every head of page src[i] to page dst[i]
// and leaves the others as they were.  The destinations are distinct and none of them is a source, so that the order of the
// copies does not matter.  The kernel is launched the ordinary way and lets no dependent start early: the attention kernels
// read the older pages of their rows before the kernel in front of them has ended.
#include "common.cuh"

namespace {

struct PageArray {              // what the host puts into the table of arrays, eight 8-byte words an array
  unsigned long long base;
  long long page_bytes, heads, head_bytes, slot_bytes, slots, pages, unit;
};

constexpr int PC_THREADS = 256;

template <typename U>
__device__ __forceinline__ void copy_rows(const PageArray& a, long long src, long long dst, long long n) {
  const long long per_head = n * a.slot_bytes / (long long)sizeof(U), all = per_head * a.heads;
  const char* from = (const char*)a.base + src * a.page_bytes;
  char* to = (char*)a.base + dst * a.page_bytes;
  for (long long i = (long long)blockIdx.x * PC_THREADS + threadIdx.x; i < all; i += (long long)gridDim.x * PC_THREADS) {
    const long long h = i / per_head, at = h * a.head_bytes + (i - h * per_head) * (long long)sizeof(U);
    *(U*)(to + at) = *(const U*)(from + at);
  }
}

__global__ void __launch_bounds__(PC_THREADS) copy_pages_kernel(const PageArray* __restrict__ arrays, const int* __restrict__ src,
                                                                const int* __restrict__ dst, const int* __restrict__ slots,
                                                                int* err) {
  const PageArray a = arrays[blockIdx.z];
  const int i = blockIdx.y;
  const int s = src[i], d = dst[i];
  if (s < 0 || s >= a.pages || d < 0 || d >= a.pages) {
    if (threadIdx.x == 0 && err) atomicExch(err, 1 + i);
    return;
  }
  const long long n = slots ? min(max((long long)slots[i], 0LL), a.slots) : a.slots;
  if (s == d || n == 0) return;
  switch ((int)a.unit) {
    case 16: copy_rows<uint4>(a, s, d, n); break;
    case 8: copy_rows<uint2>(a, s, d, n); break;
    case 4: copy_rows<uint32_t>(a, s, d, n); break;
    default: copy_rows<uint16_t>(a, s, d, n);
  }
}

}  // namespace

// arrays: [A][8] 64-bit words on the device (address, bytes of a page, heads, bytes of a head, bytes of a slot, slots of a page,
// pages, bytes of the widest access that address and sizes allow); src, dst, slots [N] on the device (slots may be
// nullptr: whole pages).  A page outside an array sets the error flag to 1 + the copy and is not copied.
NV_API int nv_copy_pages(const void* arrays, int A, long long page_bytes, const int* src, const int* dst, const int* slots, int N,
                         int* err, cudaStream_t s) {
  if (A < 0 || N < 0 || A > 65535 || N > 65535 || page_bytes < 0) return NV_ERR_BAD_SIZE;
  if (A == 0 || N == 0) return NV_OK;
  long long share = (page_bytes + 16383) / 16384;
  share = share < 1 ? 1 : share > 1024 ? 1024 : share;
  copy_pages_kernel<<<dim3((unsigned)share, (unsigned)N, (unsigned)A), PC_THREADS, 0, s>>>((const PageArray*)arrays, src, dst, slots, err);
  NV_RETURN_LAST();
}
