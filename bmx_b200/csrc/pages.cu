// Slots of page pools and rows of windows copied to other slots: what forking a sequence, closing the holes of a pool and taking a pool
// over into a larger one come down to.  bmx keeps a page as a Python dict of tensors and never moves one; a pool of slots does.
//
// dst_a[d_i] = src_a[s_i] for all pairs i and up to eight arrays a at once (pages and coefficients, or the three windows), in one
// launch.  The pairs travel as kernel parameters: there is no staging buffer that would have to outlive the call, and a captured launch
// keeps its own copy.  The host checks every index and refuses what would race.
#include <cstdlib>
#include <cstring>

#include "common.cuh"

namespace bmxk {

namespace {

constexpr int COPY_ARRAYS = 8, COPY_THREADS = 256, COPY_UNROLL = 4;
constexpr int COPY_CHUNK = COPY_THREADS * COPY_UNROLL * 16;  // bytes per block

struct CopyArray {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_stride, dst_stride, bytes;
  int chunk0;  // chunks of the arrays before this one
};
template <int N>
struct CopyParams {
  CopyArray a[COPY_ARRAYS];
  int n_arrays, chunks;  // chunks of one pair over all arrays
  int32_t from[N], to[N];
};

}  // namespace

// One block per chunk of 16 KB of one pair and array: four 16-byte loads per thread in flight, no reuse and no sharing.  Bound by memory: 640
// slots of 8 heads at rank 32 (109 MB read and written) in 35.3 us, 3000 in 155.5 us, 6.2 and 6.6 TB/s, the rate of a plain copy.
template <int N>
__global__ void __launch_bounds__(COPY_THREADS) copy_slots_kernel(const __grid_constant__ CopyParams<N> p) {
  const int pair = blockIdx.x / p.chunks, c = blockIdx.x % p.chunks;
  int k = 0;
  while (k + 1 < p.n_arrays && c >= p.a[k + 1].chunk0) ++k;
  const CopyArray& a = p.a[k];
  const int64_t off = (int64_t)(c - a.chunk0) * COPY_CHUNK;
  const uint4* s = reinterpret_cast<const uint4*>(a.src + p.from[pair] * a.src_stride + off);
  uint4* d = reinterpret_cast<uint4*>(a.dst + p.to[pair] * a.dst_stride + off);
  const int n = (int)(min((int64_t)COPY_CHUNK, a.bytes - off) >> 4);
  uint4 v[COPY_UNROLL];
#pragma unroll
  for (int i = 0; i < COPY_UNROLL; ++i) {
    const int o = i * COPY_THREADS + threadIdx.x;
    if (o < n) v[i] = __ldcs(s + o);
  }
#pragma unroll
  for (int i = 0; i < COPY_UNROLL; ++i) {
    const int o = i * COPY_THREADS + threadIdx.x;
    if (o < n) __stcs(d + o, v[i]);
  }
}

template <int N>
static int launch_copy(CopyParams<N>& p, const int32_t* from, const int32_t* to, int n, cudaStream_t s) {
  memcpy(p.from, from, sizeof(int32_t) * n);
  memcpy(p.to, to, sizeof(int32_t) * n);
  copy_slots_kernel<N><<<(unsigned)(p.chunks * n), COPY_THREADS, 0, s>>>(p);
  return check_launch("bmxk_copy_slots");
}

}  // namespace bmxk

using namespace bmxk;

extern "C" int bmxk_copy_slots(int n_arrays, const void* const* src, void* const* dst, const int64_t* src_stride, const int64_t* dst_stride,
                               const int64_t* bytes, const int32_t* src_slots, const int32_t* dst_slots, int n, int64_t n_src_slots,
                               int64_t n_dst_slots, void* stream) {
  BMXK_REQUIRE(n_arrays >= 1 && n_arrays <= COPY_ARRAYS, "bmxk_copy_slots: n_arrays=%d must be 1..%d", n_arrays, COPY_ARRAYS);
  BMXK_REQUIRE(n >= 0, "bmxk_copy_slots: n=%d", n);
  BMXK_REQUIRE(n_src_slots >= 0 && n_dst_slots >= 0 && n_src_slots < (1LL << 31) && n_dst_slots < (1LL << 31), "bmxk_copy_slots: slot counts out of range");
  BMXK_REQUIRE(src && dst && src_stride && dst_stride && bytes && (n == 0 || (src_slots && dst_slots)), "bmxk_copy_slots: null pointer");
  if (n == 0) return BMXK_OK;
  CopyArray arr[COPY_ARRAYS];
  int64_t chunks = 0;
  bool in_place = false;
  for (int a = 0; a < n_arrays; ++a) {
    BMXK_REQUIRE(src[a] && dst[a], "bmxk_copy_slots: array %d is null", a);
    BMXK_REQUIRE(bytes[a] >= 16 && src_stride[a] >= bytes[a] && dst_stride[a] >= bytes[a],
                 "bmxk_copy_slots: array %d: %lld bytes of slots that lie %lld / %lld apart", a, (long long)bytes[a], (long long)src_stride[a],
                 (long long)dst_stride[a]);
    BMXK_REQUIRE((((uintptr_t)src[a] | (uintptr_t)dst[a] | (uintptr_t)bytes[a] | (uintptr_t)src_stride[a] | (uintptr_t)dst_stride[a]) & 15) == 0,
                 "bmxk_copy_slots: array %d: pointers, strides and sizes must be multiples of 16 bytes", a);
    BMXK_REQUIRE(src_stride[a] <= (1LL << 32) && dst_stride[a] <= (1LL << 32), "bmxk_copy_slots: array %d: slots more than 4 GiB apart", a);
    arr[a] = CopyArray{(const uint8_t*)src[a], (uint8_t*)dst[a], src_stride[a], dst_stride[a], bytes[a], (int)chunks};
    chunks += (bytes[a] + COPY_CHUNK - 1) / COPY_CHUNK;
  }
  // Arrays may coincide (a copy inside one pool) but not overlap in any other way: what one pair writes another one could read.
  auto overlap = [](const uint8_t* p, int64_t pn, const uint8_t* q, int64_t qn) { return p < q + qn && q < p + pn; };
  for (int a = 0; a < n_arrays; ++a)
    for (int b = 0; b < n_arrays; ++b) {
      const int64_t da = (n_dst_slots - 1) * arr[a].dst_stride + arr[a].bytes;
      if (overlap(arr[a].dst, da, arr[b].src, (n_src_slots - 1) * arr[b].src_stride + arr[b].bytes)) {
        BMXK_REQUIRE(arr[a].dst == arr[b].src && arr[a].dst_stride == arr[b].src_stride && arr[a].bytes == arr[b].bytes,
                     "bmxk_copy_slots: destination %d overlaps source %d without being the same array", a, b);
        in_place = true;
      }
      if (a < b && overlap(arr[a].dst, da, arr[b].dst, (n_dst_slots - 1) * arr[b].dst_stride + arr[b].bytes))
        BMXK_REQUIRE(arr[a].dst == arr[b].dst && arr[a].dst_stride == arr[b].dst_stride && arr[a].bytes == arr[b].bytes && arr[a].src == arr[b].src &&
                         arr[a].src_stride == arr[b].src_stride,
                     "bmxk_copy_slots: destinations %d and %d overlap", a, b);
    }
  // Every index in range, no slot written twice, and inside one pool no slot both read and written.
  uint8_t* seen = (uint8_t*)calloc((size_t)(n_dst_slots + 7) / 8 + 1, 1);
  BMXK_REQUIRE(seen != nullptr, "bmxk_copy_slots: out of host memory");
  const char* why = nullptr;
  int at = 0;
  for (int i = 0; i < n && !why; ++i) {
    const int64_t s = src_slots[i], d = dst_slots[i];
    at = i;
    if (s < 0 || s >= n_src_slots) why = "source slot out of range";
    else if (d < 0 || d >= n_dst_slots) why = "destination slot out of range";
    else if (seen[d >> 3] >> (d & 7) & 1) why = "destination slot named twice";
    else seen[d >> 3] |= (uint8_t)(1u << (d & 7));
  }
  for (int i = 0; in_place && i < n && !why; ++i) {
    const int64_t s = src_slots[i];
    at = i;
    if (s < n_dst_slots && (seen[s >> 3] >> (s & 7) & 1)) why = "slot both read and written";
  }
  free(seen);
  BMXK_REQUIRE(why == nullptr, "bmxk_copy_slots: pair %d (%d -> %d): %s", at, src_slots[at], dst_slots[at], why);

  // A launch carries as many pairs as its parameters have room for (32 KB at most); small calls (a fork) carry few, and in between the
  // parameters of 3000 pairs would take the device longer to fetch than those of 1000.
  auto fill = [&](auto& p) {
    memcpy(p.a, arr, sizeof(arr));
    p.n_arrays = n_arrays, p.chunks = (int)chunks;
  };
  const int most = (int)((1LL << 30) / chunks);  // blocks of one launch
  for (int i = 0; i < n;) {
    const int m = n - i < most ? n - i : most;
    int rc, done;
    if (m <= 64) {
      CopyParams<64> p;
      fill(p);
      done = m, rc = launch_copy(p, src_slots + i, dst_slots + i, done, (cudaStream_t)stream);
    } else if (m <= 1000) {
      CopyParams<1000> p;
      fill(p);
      done = m, rc = launch_copy(p, src_slots + i, dst_slots + i, done, (cudaStream_t)stream);
    } else {
      CopyParams<3000> p;
      fill(p);
      done = m < 3000 ? m : 3000, rc = launch_copy(p, src_slots + i, dst_slots + i, done, (cudaStream_t)stream);
    }
    if (rc) return rc;
    i += done;
  }
  return BMXK_OK;
}
