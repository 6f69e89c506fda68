// Pages of the paged K/V store moved on the device: copies of whole pages (fork of a sequence, compaction of the pool) and
// the accepted path of a drafted tree written into the pages of its sequence.
//
// Both are pure data movement: every byte is read once and written once, so the floor of a call is 2 * bytes at the copy
// bandwidth of the HBM, plus one launch.  All layers and both tensors go in one launch.  Measured: 512 pages of 8 heads of 128,
// bf16, in 4 layers (1.07 GB moved) 170 us, 0.97 of the copy bandwidth; one page in 2 layers 3.0 us (9 a call, the host's time);
// paths of up to 16 of 32 sequences in 16 layers (34 MB) 11 us with cold caches, 12 a call.
#include <stdlib.h>
#include <string.h>

#include <algorithm>

#include "common.cuh"

namespace hils {

// Set when a page table holds an id outside the pool, a chunk past the table's width or a path an id that is no node.
static __device__ int g_pages_status = 0;

// ---- whole pages -----------------------------------------------------------------------------------------------
// The page ids are host data (the free list and the tables of the store live there), so they travel with the launch as
// kernel arguments: no upload, nothing to keep alive until the copy has run.
constexpr int kPairsPerLaunch = 480;

struct PagePairs {
  int32_t src[kPairsPerLaunch], dst[kPairsPerLaunch];
};

constexpr int kCopyThreads = 256, kCopyVecs = 4;
constexpr int kCopySlice = kCopyThreads * kCopyVecs * 16;      // bytes of a page one CTA moves

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ PagePairs ids, unsigned char* k_pages,
                                                                  unsigned char* v_pages, int64_t layer_bytes, int64_t page_bytes) {
  unsigned char* pool = ((blockIdx.z & 1) ? v_pages : k_pages) + (int64_t)(blockIdx.z >> 1) * layer_bytes;
  const uint4* src = reinterpret_cast<const uint4*>(pool + (int64_t)ids.src[blockIdx.y] * page_bytes);
  uint4* dst = reinterpret_cast<uint4*>(pool + (int64_t)ids.dst[blockIdx.y] * page_bytes);
  const int64_t n = page_bytes >> 4, i0 = (int64_t)blockIdx.x * (kCopySlice / 16) + threadIdx.x;
  uint4 x[kCopyVecs];
#pragma unroll
  for (int u = 0; u < kCopyVecs; ++u)
    if (i0 + u * kCopyThreads < n) x[u] = src[i0 + u * kCopyThreads];
#pragma unroll
  for (int u = 0; u < kCopyVecs; ++u)
    if (i0 + u * kCopyThreads < n) dst[i0 + u * kCopyThreads] = x[u];
}

// ---- accepted path of a drafted tree ---------------------------------------------------------------------------
struct CommitParams {
  const unsigned char* k_draft; const unsigned char* v_draft;
  unsigned char* k_pages; unsigned char* v_pages;
  const int32_t* pages; const int32_t* lens; const int32_t* path;
  int n_layers, B, n, m, h_kv, row_vecs, page_stride, num_pages;   // row_vecs: 16-byte pieces of one head's row
  int64_t layer_bytes;
};

constexpr int kCommitThreads = 128;

// One CTA per (sequence, place of the path, layer): a token's K and V rows, 16 bytes per thread and step.  Rows of a page are
// written in D x 2 or 4 byte pieces, one per head; the path is short, so each CTA reads it up to its own place.
__global__ void __launch_bounds__(kCommitThreads) commit_drafts_kernel(CommitParams p) {
  const int b = blockIdx.x / p.m, i = blockIdx.x - b * p.m, layer = blockIdx.y;
  const int32_t* path = p.path + (int64_t)b * p.m;
  // the path ends at its first entry that is no node; an entry past the nodes is reported as well
  int node = 0;
  for (int e = 0; e <= i; ++e) {
    node = path[e];
    if ((unsigned)node >= (unsigned)p.n) {
      if (node >= 0 && e == i && threadIdx.x == 0) atomicExch(&g_pages_status, 8100001);
      return;
    }
  }
  const int64_t tok = (int64_t)p.lens[b] + i;
  const int64_t c = tok >> 6;
  const int pg = (p.lens[b] >= 0 && c < p.page_stride) ? p.pages[(int64_t)b * p.page_stride + c] : -1;
  if ((unsigned)pg >= (unsigned)p.num_pages) {
    if (threadIdx.x == 0) atomicExch(&g_pages_status, 8100002);
    return;
  }
  const int row = (int)(tok & 63), per = p.h_kv * p.row_vecs;
  const int64_t src0 = (((int64_t)layer * p.B + b) * p.n + node) * per * 16;
  const int64_t dst0 = (int64_t)layer * p.layer_bytes + (int64_t)pg * per * 64 * 16;
  for (int x = threadIdx.x; x < per; x += kCommitThreads) {
    const int h = x / p.row_vecs, e = x - h * p.row_vecs;
    const int64_t d = dst0 + (((int64_t)h * 64 + row) * p.row_vecs + e) * 16;
    const uint4 kx = *reinterpret_cast<const uint4*>(p.k_draft + src0 + (int64_t)x * 16);
    const uint4 vx = *reinterpret_cast<const uint4*>(p.v_draft + src0 + (int64_t)x * 16);
    *reinterpret_cast<uint4*>(p.k_pages + d) = kx;
    *reinterpret_cast<uint4*>(p.v_pages + d) = vx;
  }
}

int take_status_pages() {
  int v = 0, zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v, g_pages_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_pages_status, &zero, sizeof(int));
  return v;
}

}  // namespace hils

using namespace hils;

// every id in the pool, no page written twice, no page both read and written (the copies run in no order)
static int check_pairs(const int32_t* src, const int32_t* dst, int n_pairs, int num_pages) {
  const size_t words = ((size_t)num_pages + 31) / 32;
  uint32_t* written = static_cast<uint32_t*>(calloc(words, sizeof(uint32_t)));
  if (!written) {
    set_error("copy_pages: no host memory for a bitmap of %d pages", num_pages);
    return HILS_ERR_BAD_ARG;
  }
  int rc = HILS_OK;
  for (int i = 0; i < n_pairs && rc == HILS_OK; ++i) {
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) {
      set_error("copy_pages: pair %d (%d -> %d) is outside the pool of %d pages", i, src[i], dst[i], num_pages);
      rc = HILS_ERR_BAD_ARG;
    } else if (written[dst[i] >> 5] >> (dst[i] & 31) & 1u) {
      set_error("copy_pages: page %d is written twice", dst[i]);
      rc = HILS_ERR_BAD_ARG;
    } else {
      written[dst[i] >> 5] |= 1u << (dst[i] & 31);
    }
  }
  for (int i = 0; i < n_pairs && rc == HILS_OK; ++i)
    if (written[src[i] >> 5] >> (src[i] & 31) & 1u) {
      set_error("copy_pages: page %d is read and written by one call", src[i]);
      rc = HILS_ERR_BAD_ARG;
    }
  free(written);
  return rc;
}

extern "C" int hils_copy_pages(void* k_pages, void* v_pages, const int32_t* src, const int32_t* dst, int n_pairs, int n_layers,
                               int num_pages, int64_t layer_bytes, int64_t page_bytes, void* stream) {
  HILS_REQUIRE(n_pairs >= 0 && n_layers >= 0 && num_pages >= 0, "copy_pages: negative size");
  if (n_pairs == 0 || n_layers == 0) return HILS_OK;
  HILS_REQUIRE(k_pages && v_pages && src && dst, "copy_pages: null pointer");
  HILS_REQUIRE(num_pages > 0, "copy_pages: the pool has no pages");
  HILS_REQUIRE(page_bytes > 0 && page_bytes % 16 == 0, "copy_pages: a page of %lld bytes is not a multiple of 16", (long long)page_bytes);
  HILS_REQUIRE(layer_bytes % 16 == 0 && (n_layers == 1 || layer_bytes / page_bytes >= num_pages),
               "copy_pages: layers %lld bytes apart do not hold %d pages", (long long)layer_bytes, num_pages);
  HILS_REQUIRE(((((uintptr_t)k_pages) | ((uintptr_t)v_pages)) & 15) == 0, "copy_pages: tensors must be 16-byte aligned");
  HILS_REQUIRE(n_layers <= 32767, "copy_pages: at most 32767 layers");
  const int64_t slices = (page_bytes + kCopySlice - 1) / kCopySlice;
  HILS_REQUIRE(slices <= 0x7fffffff, "copy_pages: a page of %lld bytes is too large", (long long)page_bytes);
  if (int rc = check_pairs(src, dst, n_pairs, num_pages)) return rc;
  PagePairs ids;
  for (int i0 = 0; i0 < n_pairs; i0 += kPairsPerLaunch) {
    const int m = std::min(kPairsPerLaunch, n_pairs - i0);
    memcpy(ids.src, src + i0, sizeof(int32_t) * m);
    memcpy(ids.dst, dst + i0, sizeof(int32_t) * m);
    const dim3 grid((unsigned)slices, (unsigned)m, (unsigned)n_layers * 2);
    copy_pages_kernel<<<grid, kCopyThreads, 0, (cudaStream_t)stream>>>(ids, static_cast<unsigned char*>(k_pages),
                                                                      static_cast<unsigned char*>(v_pages), layer_bytes, page_bytes);
    HILS_LAUNCH_CHECK("copy_pages");
  }
  return HILS_OK;
}

extern "C" int hils_commit_drafts(const void* k_draft, const void* v_draft, void* k_pages, void* v_pages, const int32_t* page_table,
                                  int page_stride, int num_pages, const int32_t* lens, const int32_t* path, int n_layers, int B,
                                  int n, int m, int h_kv, int D, int64_t layer_bytes, int dtype, void* stream) {
  HILS_REQUIRE(dtype == HILS_BF16 || dtype == HILS_F32, "commit_drafts: dtype must be bf16 or fp32");
  HILS_REQUIRE(n_layers >= 0 && B >= 0 && n >= 0 && m >= 0 && m <= n, "commit_drafts: a path of %d places over %d nodes", m, n);
  HILS_REQUIRE(h_kv > 0 && D > 0 && page_stride > 0 && num_pages > 0, "commit_drafts: non-positive size");
  const int64_t es = dtype == HILS_BF16 ? 2 : 4, row_bytes = D * es;
  HILS_REQUIRE(row_bytes % 16 == 0, "commit_drafts: rows of %lld bytes are not a multiple of 16", (long long)row_bytes);
  HILS_REQUIRE((int64_t)h_kv * row_bytes / 16 <= 0x7fffffff / 64, "commit_drafts: %d heads of %d are too many", h_kv, D);
  HILS_REQUIRE(layer_bytes % 16 == 0 && (n_layers <= 1 || layer_bytes / (h_kv * row_bytes * 64) >= num_pages),
               "commit_drafts: layers %lld bytes apart do not hold %d pages", (long long)layer_bytes, num_pages);
  if (n_layers == 0 || B == 0 || m == 0) return HILS_OK;
  HILS_REQUIRE((int64_t)B * m <= 0x7fffffff && n_layers <= 65535, "commit_drafts: too many rows");
  HILS_REQUIRE(k_draft && v_draft && k_pages && v_pages && page_table && lens && path, "commit_drafts: null pointer");
  HILS_REQUIRE(((((uintptr_t)k_draft) | ((uintptr_t)v_draft) | ((uintptr_t)k_pages) | ((uintptr_t)v_pages)) & 15) == 0,
               "commit_drafts: tensors must be 16-byte aligned");
  CommitParams p = {};
  p.k_draft = static_cast<const unsigned char*>(k_draft); p.v_draft = static_cast<const unsigned char*>(v_draft);
  p.k_pages = static_cast<unsigned char*>(k_pages); p.v_pages = static_cast<unsigned char*>(v_pages);
  p.pages = page_table; p.lens = lens; p.path = path;
  p.n_layers = n_layers; p.B = B; p.n = n; p.m = m; p.h_kv = h_kv; p.row_vecs = (int)(row_bytes / 16);
  p.page_stride = page_stride; p.num_pages = num_pages; p.layer_bytes = layer_bytes;
  commit_drafts_kernel<<<dim3((unsigned)(B * m), (unsigned)n_layers), kCommitThreads, 0, (cudaStream_t)stream>>>(p);
  HILS_LAUNCH_CHECK("commit_drafts");
  return HILS_OK;
}
