// Page copies inside a layered pool (gfx950): page dst_ids[i] becomes a copy of page src_ids[i], every plane of it,
// payload and scale tiles, in one launch.
//
// Bound by memory: each byte is read once and written once. Measured: 450 pages of 80 layers of 8-bit KV with scales, 2.36 GB read
// and written, in 460 us (5.1 TB/s; a large torch copy in the same memory 4.7); 2 pages of 28 layers in 2.7 us. Loads and stores
// with and without the non-temporal and system-scope hints run alike. The shape is the one the pool's movers run
// fastest with: every 64 vectors of a tile are a workgroup of one wave, one vector per lane, the entry's ids and the
// plane's base by scalar loads. A page's planes follow each other in the grid, so that neighbouring
// workgroups touch planes gigabytes apart. A gather into staging and a scatter out of it would move the same bytes
// twice and need a buffer of their size.
#include "pagecopy_kernels.h"

namespace bikv {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int VW> struct MoveVec;
template <> struct MoveVec<16> { using T = u32x4; };
template <> struct MoveVec<8> { using T = u32x2; };
template <> struct MoveVec<4> { using T = uint32_t; };
template <> struct MoveVec<2> { using T = uint16_t; };
template <> struct MoveVec<1> { using T = uint8_t; };

#define BIKV_GLB __attribute__((address_space(1)))
#define BIKV_CST __attribute__((address_space(4)))

template <int VW>
__device__ __forceinline__ void move_vec(uint64_t s, uint64_t d) {
  using T = typename MoveVec<VW>::T;
  __builtin_nontemporal_store(__builtin_nontemporal_load((const BIKV_GLB T*)s), (BIKV_GLB T*)d);
}

__device__ __forceinline__ void move_by(int vw, uint64_t s, uint64_t d) {
  switch (vw) {
    case 16: move_vec<16>(s, d); break;
    case 8: move_vec<8>(s, d); break;
    case 4: move_vec<4>(s, d); break;
    case 2: move_vec<2>(s, d); break;
    default: move_vec<1>(s, d); break;
  }
}

template <int VW>
__global__ __launch_bounds__(64) void page_move_kernel(const PageMoveArgs a) {
  const uint64_t i = (uint64_t)blockIdx.y + (uint64_t)blockIdx.z * gridDim.y;
  if (i >= (uint64_t)a.n) return;
  const int64_t s = ((const BIKV_CST int64_t*)a.src_ids)[i], d = ((const BIKV_CST int64_t*)a.dst_ids)[i];
  if ((uint64_t)s >= (uint64_t)a.n_pool_pages || (uint64_t)d >= (uint64_t)a.n_pool_pages) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile uint32_t*>(a.status + ST_SLOT_PAGE) = 1u;
    return;
  }
  if (s == d) return;
  if (blockIdx.x < a.payload.n_blocks) {
    const uint32_t q = blockIdx.x / a.payload.parts, part = blockIdx.x - q * a.payload.parts;
    const uint64_t off = ((uint64_t)part * 64u + threadIdx.x) * VW;
    if (off >= (uint64_t)a.payload.tile_bytes) return;
    uint64_t at = off;
    if (a.payload.row_bytes != a.payload.tile_bytes) {            // a tile in rows, as the Worker's own tensors hold it
      const uint64_t r = a.payload.log2_row >= 0 ? off >> a.payload.log2_row : off / (uint64_t)a.payload.row_bytes;
      at = r * (uint64_t)a.payload.row_stride + (off - r * (uint64_t)a.payload.row_bytes);
    }
    const uint64_t plane = (uint64_t)((const char* const BIKV_CST*)a.payload.plane_base)[q] + at;
    move_vec<VW>(plane + (uint64_t)(s * a.payload.page_stride), plane + (uint64_t)(d * a.payload.page_stride));
  } else {
    // scale tiles: one lane per vector, the planes of the page one after the other
    const uint32_t v = (blockIdx.x - a.payload.n_blocks) * 64u + threadIdx.x;
    const uint32_t q = v / a.scale.parts, off = (v - q * a.scale.parts) * (uint32_t)a.scale.vec_width;
    if (q >= a.n_planes) return;
    const uint64_t plane = (uint64_t)a.scale.plane_base[q] + off;
    move_by(a.scale.vec_width, plane + (uint64_t)(s * a.scale.page_stride), plane + (uint64_t)(d * a.scale.page_stride));
  }
}

hipError_t launch_page_moves(PageMoveArgs& a, hipStream_t stream) {
  if (a.n <= 0) return hipSuccess;
  const int64_t vecs = a.payload.tile_bytes / a.payload.vec_width;
  const int64_t parts = (vecs + 63) / 64;
  const int64_t px = parts * a.n_planes;
  int64_t sx = 0, vpt = 0;
  if (a.scale.tile_bytes > 0) {
    vpt = a.scale.tile_bytes / a.scale.vec_width;
    sx = (vpt * a.n_planes + 63) / 64;
  }
  if (parts >= (int64_t(1) << 31) || vpt * a.n_planes >= (int64_t(1) << 31) || px + sx >= (int64_t(1) << 32) / 64) return hipErrorInvalidConfiguration;
  a.payload.parts = (uint32_t)parts;
  a.payload.n_blocks = (uint32_t)px;
  a.scale.parts = (uint32_t)vpt;
  const int64_t gy = a.n < 32768 ? a.n : 32768, gz = (a.n + gy - 1) / gy;
  if (gz > 65535) return hipErrorInvalidConfiguration;
  const dim3 grid((uint32_t)(px + sx), (uint32_t)gy, (uint32_t)gz), block(64);
  switch (a.payload.vec_width) {
    case 16: hipLaunchKernelGGL((page_move_kernel<16>), grid, block, 0, stream, a); break;
    case 8: hipLaunchKernelGGL((page_move_kernel<8>), grid, block, 0, stream, a); break;
    case 4: hipLaunchKernelGGL((page_move_kernel<4>), grid, block, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((page_move_kernel<2>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((page_move_kernel<1>), grid, block, 0, stream, a); break;
  }
  return hipGetLastError();
}

}  // namespace bikv
