// Host side of the serving calls (include/fmha_i8_c.h): rotary positions and the write into the cache, attention over packed prompts
// and over the paged cache.  Argument checks, tensor maps, the choice of a kernel and the launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <mutex>
#include <utility>

#include "../../include/fmha_i8_c.h"
#include "fmha_chunk_sm100.cuh"
#include "fmha_grouped_sm100.cuh"
#include "fmha_internal.h"
#include "fmha_rope_sm100.cuh"
#include "fmha_rows_sm100.cuh"

namespace {

using namespace fmha;
using fmha_host::Device;
using fmha_host::finish;

constexpr int kMaxDevices = 64;
constexpr long long kMostRows = 0x7FFFFFFFLL;

// n rows (or pages) `stride` elements apart lie in no memory: a stride that a tensor map cannot hold, or a span beyond all addresses.
bool too_far(long long n, long long stride, int bytes) {
  constexpr long long kMostStride = 1LL << 40, kMostSpan = 1LL << 47;
  return stride >= kMostStride / bytes || (n > 0 && stride * bytes > kMostSpan / n);
}
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool power_of_two(long long n) { return n > 0 && (n & (n - 1)) == 0; }
int log2_of(long long n) { int s = 0; while ((1LL << s) < n) ++s; return s; }
int type_bytes(int type) { return type == FMHA_I8_TYPE_I8 ? 1 : type == FMHA_I8_TYPE_FP32 ? 4 : 2; }

// What is asked of and set on a device once, before the first launch there.
struct Once {
  std::atomic<bool> done{false};
  int clusters16_d64 = 0, clusters16_d128 = 0;        // clusters of 16 CTAs of the wide rows kernel that are resident at once
};
Once g_once[kMaxDevices];
std::mutex g_once_mutex;

template <typename... Params, typename... Args>
int launch(void (*fn)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  if (cluster != 0) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  fmha_host::count_launch();
  if (cudaLaunchKernelEx(&cfg, fn, std::forward<Args>(args)...) == cudaSuccess) return FMHA_I8_OK;
  cudaGetLastError();
  return FMHA_I8_ERR_LAUNCH;
}

template <int D> using RowsCfg = rows::Cfg<D>;

template <int D, int kRows> int set_up_rows() {
  constexpr int W = RowsCfg<D>::kWarps, Wide = RowsCfg<D>::kWarpsWide;
  auto set = [](const void* fn, size_t bytes) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == cudaSuccess &&
           cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
  };
  if (set(reinterpret_cast<const void*>(&rows::rows_kernel<D, W, kRows>), sizeof(rows::Smem<D, W, kRows>)) &&
      set(reinterpret_cast<const void*>(&rows::rows_kernel<D, Wide, kRows>), sizeof(rows::Smem<D, Wide, kRows>)))
    return FMHA_I8_OK;
  cudaGetLastError();
  return FMHA_I8_ERR_LAUNCH;
}
// Clusters of 16 CTAs of the wide kernel that are resident at once.
template <int D> int count_clusters() {
  constexpr int Wide = RowsCfg<D>::kWarpsWide;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 16;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(16);
  cfg.blockDim = dim3(Wide * 32);
  cfg.dynamicSmemBytes = sizeof(rows::Smem<D, Wide, 16>);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, rows::rows_kernel<D, Wide, 16>, &cfg) != cudaSuccess) n = 0;
  cudaGetLastError();
  return n;
}

template <int D> int set_up_chunk() {
  for (const void* fn : {reinterpret_cast<const void*>(&chunk::chunk_kernel<D, false, false>), reinterpret_cast<const void*>(&chunk::chunk_kernel<D, true, false>),
                         reinterpret_cast<const void*>(&chunk::chunk_kernel<D, true, true>)}) {
    cudaFuncAttributes fa{};
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(chunk::smem_bytes<D>())) != cudaSuccess ||
        cudaFuncGetAttributes(&fa, fn) != cudaSuccess) {
      cudaGetLastError();
      return FMHA_I8_ERR_LAUNCH;
    }
    // the kernel moves registers between its warps with setmaxnreg, which only terminates if the launch allocation is what the targets were sized for
    if (fa.numRegs == chunk::kLaunchRegs) continue;
    std::fprintf(stderr, "fmha_i8_sm100: chunk kernel built with %d registers per thread, expected %d; refusing to launch\n", fa.numRegs, chunk::kLaunchRegs);
    return FMHA_I8_ERR_LAUNCH;
  }
  return FMHA_I8_OK;
}

int set_up(const Device& dev) {
  Once& once = g_once[dev.index];
  if (once.done.load(std::memory_order_acquire)) return FMHA_I8_OK;
  std::lock_guard<std::mutex> lock(g_once_mutex);
  if (once.done.load(std::memory_order_relaxed)) return FMHA_I8_OK;
  int st;
  if ((st = set_up_rows<64, 4>()) != FMHA_I8_OK || (st = set_up_rows<64, 8>()) != FMHA_I8_OK || (st = set_up_rows<64, 16>()) != FMHA_I8_OK) return st;
  if ((st = set_up_rows<128, 4>()) != FMHA_I8_OK || (st = set_up_rows<128, 8>()) != FMHA_I8_OK || (st = set_up_rows<128, 16>()) != FMHA_I8_OK) return st;
  once.clusters16_d64 = count_clusters<64>();
  once.clusters16_d128 = count_clusters<128>();
  if ((st = set_up_chunk<64>()) != FMHA_I8_OK || (st = set_up_chunk<128>()) != FMHA_I8_OK) return st;
  once.done.store(true, std::memory_order_release);
  return FMHA_I8_OK;
}

// Where the keys lie: [outer, heads, rows, D] with strides in bytes; box_rows rows at a time.
struct KeyLayout {
  long long outer, heads, rows, row_stride, head_stride, outer_stride;
  int box_rows;
};
int key_map(CUtensorMap* map, const void* base, const KeyLayout& l, int D) {
  auto fn = fmha_host::encode_tiled();
  if (!fn) return FMHA_I8_ERR_DRIVER;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(l.rows), static_cast<cuuint64_t>(l.heads), static_cast<cuuint64_t>(l.outer)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(l.row_stride), static_cast<cuuint64_t>(l.head_stride), static_cast<cuuint64_t>(l.outer_stride)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(D), static_cast<cuuint32_t>(l.box_rows), 1u, 1u}, ones[4] = {1u, 1u, 1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FMHA_I8_OK : FMHA_I8_ERR_DRIVER;
}

struct Call {
  grouped::Params p{};
  const void *k = nullptr, *v = nullptr;
  KeyLayout lk{}, lv{};
  int D = 0;
  long long max_k = 0;
};

// Checks and parameters that packed and paged calls share.
int fill_call(Call* c, const float amax[5], const int desc6[6], const void* q, const void* k, const void* v, const int* cu_q, void* o, int o_type, long long total_q,
              long long q_stride, long long o_stride, unsigned flags) {
  if (!(flags & FMHA_I8_FLAG_USE_TCU)) return FMHA_I8_ERR_NO_CUDA_CORE_PATH;
  if (flags & ~(FMHA_I8_FLAG_USE_TCU | FMHA_I8_FLAG_CAUSAL)) return FMHA_I8_ERR_BAD_FLAGS;
  const int B = desc6[0], max_q = desc6[1], max_k = desc6[2], H = desc6[3], Hkv = desc6[4], D = desc6[5];
  if (B < 1 || max_q < 0 || max_k < 0 || H < 1 || Hkv < 1 || H % Hkv != 0 || (D != 64 && D != 128)) return FMHA_I8_ERR_BAD_SHAPE;
  if (o_type != FMHA_I8_TYPE_I8 && o_type != FMHA_I8_TYPE_BF16 && o_type != FMHA_I8_TYPE_FP16) return FMHA_I8_ERR_BAD_SHAPE;
  if (total_q < 0 || q_stride < static_cast<long long>(H) * D || o_stride < static_cast<long long>(H) * D) return FMHA_I8_ERR_BAD_SHAPE;
  const int G = H / Hkv;
  if (total_q > kMostRows / H || static_cast<long long>(max_q) * G > kMostRows - 256 || max_k > (1 << 30) || B > (1 << 30) || static_cast<long long>(B) * Hkv > kMostRows) return FMHA_I8_ERR_TOO_LARGE;
  if (too_far(total_q, q_stride, 1) || too_far(total_q, o_stride, type_bytes(o_type))) return FMHA_I8_ERR_TOO_LARGE;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(o, 16) || !aligned(cu_q, 4)) return FMHA_I8_ERR_MISALIGNED;
  if (q_stride % 16 != 0 || o_stride * type_bytes(o_type) % 16 != 0) return FMHA_I8_ERR_MISALIGNED;
  for (int i = 0; i < (o_type == FMHA_I8_TYPE_I8 ? 4 : 3); ++i)
    if (!(amax[i] > 0.f) || !std::isfinite(amax[i])) return FMHA_I8_ERR_BAD_AMAX;
  grouped::Params& p = c->p;
  const double c2 = static_cast<double>(amax[0]) * amax[1] / (127.0 * 127.0) / std::sqrt(static_cast<double>(D)) * 1.4426950408889634;
  // between factors at which all probabilities are 1 and at which only the largest counts (the scores are integers up to 2^21)
  p.c2 = static_cast<float>(std::min(std::max(c2, 0x1p-100), 32.0));
  p.growth = static_cast<int>(std::min(static_cast<double>(grouped::kGrowth) / p.c2, 1e9));
  const double unit = amax[2] / (o_type == FMHA_I8_TYPE_I8 ? static_cast<double>(amax[3]) : 127.0);
  p.out_down = unit < 0x1p-60 ? 0x1p-64f : 1.f;
  p.out_scale = static_cast<float>(unit / p.out_down);
  if (!std::isfinite(p.out_scale)) return FMHA_I8_ERR_BAD_AMAX;
  p.q = static_cast<const int8_t*>(q);
  p.o = o;
  p.q_stride = q_stride;
  p.o_stride = o_stride;
  p.cu_q = cu_q;
  p.B = B; p.H = H; p.Hkv = Hkv; p.G = G;
  p.total_q = static_cast<int>(total_q);
  p.max_q = max_q;
  p.o_type = o_type;
  p.o_wide = aligned(o, 32) && o_stride * type_bytes(o_type) % 32 == 0;
  p.causal = (flags & FMHA_I8_FLAG_CAUSAL) != 0u;
  c->k = k;
  c->v = v;
  c->D = D;
  c->max_k = max_k;
  return FMHA_I8_OK;
}

template <int D, int kRows> int launch_rows(cudaStream_t stream, const Device& dev, Call& c, const CUtensorMap& mk, const CUtensorMap& mv) {
  grouped::Params& p = c.p;
  constexpr int W = RowsCfg<D>::kWarps, Wide = RowsCfg<D>::kWarpsWide;
  // (one at least: a sequence with tokens where the call allows none is to be reported)
  p.row_groups = p.few_rows != 0 ? 1 : std::max(1, static_cast<int>((static_cast<long long>(p.max_q) * p.G + kRows - 1) / kRows));
  const long long units = static_cast<long long>(p.B) * p.Hkv * p.row_groups;
  const long long n_tiles = (c.max_k + grouped::kTile - 1) / grouped::kTile;
  if (units > kMostRows / rows::kMaxCluster) return FMHA_I8_ERR_TOO_LARGE;      // (B * Hkv is below 2^31, and the groups below 2^29)
  const long long resident = 3LL * dev.sm_count;
  // Few units with many keys: one CTA with all the warps of an SM on as many SMs as a cluster allows.  8 units of 131,072 keys, head_dim 128: 64 us; the CTAs of
  // two warps below in clusters of 8 74, of 16 67 to 76.
  const int clusters16 = D == 128 ? g_once[dev.index].clusters16_d128 : g_once[dev.index].clusters16_d64;
  for (const int ctas : {16, 8})
    if (units * ctas <= dev.sm_count && (ctas == 8 || units <= clusters16) && n_tiles >= 2LL * ctas * Wide)
      return launch(rows::rows_kernel<D, Wide, kRows>, static_cast<unsigned>(units * ctas), Wide * 32, sizeof(rows::Smem<D, Wide, kRows>), stream, static_cast<unsigned>(ctas), mk, mv, p);
  // Otherwise clusters as long as that fills the chip or takes a warp's tiles apart.  Against one CTA to a unit (us, head_dim 128): 8 units of 513 keys 8.0 and 10.3, of 8193
  // 16 and 72; 128 of 1025 14.6 and 17.8; 512 of 4097 104 and 115; 256 of 300 10.4 and 10.3.
  int ctas = 1;
  while (ctas < 8 && ((units * ctas < 2 * resident && n_tiles >= 4 * ctas * W) || (units * ctas * 2 <= resident && n_tiles > ctas * W))) ctas *= 2;
  return launch(rows::rows_kernel<D, W, kRows>, static_cast<unsigned>(units * ctas), W * 32, sizeof(rows::Smem<D, W, kRows>), stream, static_cast<unsigned>(ctas), mk, mv, p);
}

// Pairs of tiles of the chunk kernel: no more than the tokens make, and one more for every sequence.
long long chunk_units(const grouped::Params& p) { return std::min<long long>(p.total_q, p.total_q / (2LL * (grouped::kTile / p.G)) + p.B) * p.Hkv; }

// Which kernel.  Up to 128 heads share a key head of the chunk kernel, whose tile holds at least one token.  Otherwise by the rows of a sequence and key head
// (rows kernel against chunk kernel, us): 16 rows, head_dim 128, 4097 keys: 8 units 15.6 and 17.8, 128 units 53 and 60, 512 units 119 and 223.
// 17 to 32 rows are two groups of the rows kernel, each of which reads all keys: head_dim 64, 129 to 4097 keys, 8 to 1024 units: 0.47 to 0.87 of the chunk
// kernel's time (512 units of 1025 keys 38 and 62); head_dim 128 0.78 to 0.93 of it for 512 units and more of 1025 keys and more (4097 keys 176 and 223),
// 1.02 to 1.54 for fewer or shorter ones.  33 to 48 rows: 0.60 to 1.08 and 1.05 to 1.22.
constexpr int kMostGroup = 128;
bool few_rows(const Call& c, int sms) {
  const grouped::Params& p = c.p;
  const long long n_rows = static_cast<long long>(p.max_q) * p.G;
  if (p.G > kMostGroup || n_rows <= 16) return true;
  if (n_rows > 32) return false;
  return c.D == 64 || (chunk_units(p) >= 3LL * sms && c.max_k > 7 * grouped::kTile);
}

// CTAs that share a unit of the chunk kernel, in steps of one key tile (1.7 us): a CTA's share of them, and 4 for what a part costs besides.  Without and with, us:
// 200 tokens on 32,768 keys (B1 H32/8 D128) 469 and 147, two chunks of 103 on 88,000 (H24/12 D64) 1155 and 319, 16 on 4097 (B1 H32/8 D128) 57 and 29.
struct Split { int parts; long long steps; };
Split chunk_split(long long units, long long n_tiles, int sms) {
  Split best{1, (units + sms - 1) / sms * (n_tiles + 2)};
  for (const int c : {2, 4, 8}) {
    const long long rounds = (units * c + sms - 1) / sms, steps = rounds * ((n_tiles + c - 1) / c + 4);
    if (steps < best.steps) best = Split{c, steps};
  }
  return best;
}
// In a mixed batch, where most sequences bring a token or two: the units that there are if the others have as many tokens as they may.
long long expected_units(const grouped::Params& p) {
  return std::min(chunk_units(p), (p.total_q / (2LL * (grouped::kTile / p.G)) + (p.total_q + p.max_q - 1) / p.max_q) * p.Hkv);
}
// The rows of sequences that the rows kernel takes out of a batch of chunks, or 0.  The host does not know the lengths, but the tokens that there are in all: below a quarter of
// what the sequences may bring.  Steps of the chunk kernel with all sequences against those with the expected ones, 8 for two more launches and the rows kernel's tiles, of
// which 300 take a step.  In one launch and apart, us (H32/8 D128 where not said): one chunk of 512 among 64 sequences of up to 4096 keys 177 and 118, two of 1024 among 256 of up
// to 8192 1016 and 596, two of 2048 among 130 288 and 202, one of 480 among 33 of up to 4096 (H16/2 D64) 60 and 48; left in one launch: one of 500 among 5 of up to 1000 20 and 39, 15 of
// 256 among 64 (H12/1) 56 and 71, 8 of 300 among 33 85 and 83.
int rows_apart(const Call& c, int sms) {
  const grouped::Params& p = c.p;
  if (p.G > 16 || 4LL * p.total_q > static_cast<long long>(p.B) * p.max_q) return 0;
  const long long n_tiles = (c.max_k + grouped::kTile - 1) / grouped::kTile;
  const long long apart = chunk_split(expected_units(p), n_tiles, sms).steps + 8 + static_cast<long long>(p.B) * p.Hkv * n_tiles / 300;
  if (apart >= chunk_split(chunk_units(p), n_tiles, sms).steps) return 0;
  return p.G <= 8 ? 8 : 16;
}

template <int D> int launch_chunk(cudaStream_t stream, const Device& dev, Call& c, const CUtensorMap& mk, const CUtensorMap& mv) {
  grouped::Params& p = c.p;
  p.tq = grouped::kTile / p.G;
  auto fn = fmha_host::encode_tiled();
  CUtensorMap mq;
  const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(p.H), static_cast<cuuint64_t>(p.total_q)};
  const cuuint64_t strides[2] = {D, static_cast<cuuint64_t>(p.q_stride)};
  const cuuint32_t box[3] = {D, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(p.tq)}, ones[3] = {1u, 1u, 1u};
  if (!fn || fn(&mq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(p.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return FMHA_I8_ERR_DRIVER;
  const long long units = chunk_units(p);
  if (units > kMostRows) return FMHA_I8_ERR_TOO_LARGE;
  // In a mixed batch the expected units may be shared by clusters; what goes beyond them is left to a second launch, which mostly finds nothing.
  const long long expected = p.few_rows == 0 ? units : expected_units(p);
  const int parts = chunk_split(expected, (c.max_k + grouped::kTile - 1) / grouped::kTile, dev.sm_count).parts;
  if (parts > 1) {
    const int st = launch(chunk::chunk_kernel<D, true, true>, static_cast<unsigned>(expected * parts), chunk::kThreads, chunk::smem_bytes<D>(), stream, static_cast<unsigned>(parts), mq, mk, mv, p);
    if (st != FMHA_I8_OK || expected == units) return st;
    p.first_unit = expected;
  }
  const unsigned grid = static_cast<unsigned>(std::min<long long>(units - p.first_unit, dev.sm_count));
  return launch(p.c2 > 0.5f ? chunk::chunk_kernel<D, true, false> : chunk::chunk_kernel<D, false, false>, grid, chunk::kThreads, chunk::smem_bytes<D>(), stream, 0u, mq, mk, mv, p);
}

int run_attention(void* stream, Call& c) {
  Device dev;
  int st;
  if ((st = fmha_host::device_for_call(&dev)) != FMHA_I8_OK) return st;
  if ((st = set_up(dev)) != FMHA_I8_OK) return st;
  if (c.p.total_q == 0) return FMHA_I8_OK;
  c.p.status = dev.status;
  c.p.host_word = dev.host_word;
  const bool few = few_rows(c, dev.sm_count);
  if (!few && c.max_k > chunk::kMostKeys) return FMHA_I8_ERR_TOO_LARGE;
  CUtensorMap mk, mv;
  if ((st = key_map(&mk, c.k, c.lk, c.D)) != FMHA_I8_OK) return st;
  if ((st = key_map(&mv, c.v, c.lv, c.D)) != FMHA_I8_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!few) c.p.few_rows = rows_apart(c, dev.sm_count);
  if (few || c.p.few_rows != 0) {
    const long long rows = few ? static_cast<long long>(c.p.max_q) * c.p.G : c.p.few_rows;
    if (c.D == 128) st = rows <= 4 ? launch_rows<128, 4>(s, dev, c, mk, mv) : rows <= 8 ? launch_rows<128, 8>(s, dev, c, mk, mv) : launch_rows<128, 16>(s, dev, c, mk, mv);
    else st = rows <= 4 ? launch_rows<64, 4>(s, dev, c, mk, mv) : rows <= 8 ? launch_rows<64, 8>(s, dev, c, mk, mv) : launch_rows<64, 16>(s, dev, c, mk, mv);
    if (few || st != FMHA_I8_OK) return st;
  }
  return c.D == 128 ? launch_chunk<128>(s, dev, c, mk, mv) : launch_chunk<64>(s, dev, c, mk, mv);
}

int infer_packed_impl(void* stream, const float amax[5], const int desc6[6], const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, void* o,
                      int o_type, const long long tokens[2], const long long strides[4], unsigned flags) {
  if (!amax || !desc6 || !q || !k || !v || !cu_q || !cu_k || !o || !tokens || !strides) return FMHA_I8_ERR_NULL_POINTER;
  Call c;
  const int st = fill_call(&c, amax, desc6, q, k, v, cu_q, o, o_type, tokens[0], strides[0], strides[3], flags);
  if (st != FMHA_I8_OK) return st;
  const long long width = static_cast<long long>(c.p.Hkv) * c.D;
  if (tokens[1] < 0 || strides[1] < width || strides[2] < width) return FMHA_I8_ERR_BAD_SHAPE;
  if (tokens[1] > (1LL << 30) || too_far(tokens[1], strides[1], 1) || too_far(tokens[1], strides[2], 1)) return FMHA_I8_ERR_TOO_LARGE;
  if (strides[1] % 16 != 0 || strides[2] % 16 != 0 || !aligned(cu_k, 4)) return FMHA_I8_ERR_MISALIGNED;
  c.p.cu_k = cu_k;
  c.p.total_k = static_cast<int>(tokens[1]);
  c.max_k = std::min(c.max_k, tokens[1]);
  c.p.num_pages = 1;
  c.p.page_shift = 0;
  c.p.box_shift = log2_of(grouped::kTile);
  const long long rows = std::max(tokens[1], 1LL);
  c.lk = KeyLayout{1, c.p.Hkv, rows, strides[1], c.D, strides[1] * rows, grouped::kTile};
  c.lv = KeyLayout{1, c.p.Hkv, rows, strides[2], c.D, strides[2] * rows, grouped::kTile};
  return run_attention(stream, c);
}

int infer_paged_impl(void* stream, const float amax[5], const int desc6[6], const void* q, const void* k, const void* v, const int* page_table, const int* lens_k,
                     const int* cu_q, void* o, int o_type, long long tokens, const long long strides[2], const long long cache[5], unsigned flags) {
  if (!amax || !desc6 || !q || !k || !v || !page_table || !lens_k || !cu_q || !o || !strides || !cache) return FMHA_I8_ERR_NULL_POINTER;
  Call c;
  const int st = fill_call(&c, amax, desc6, q, k, v, cu_q, o, o_type, tokens, strides[0], strides[1], flags);
  if (st != FMHA_I8_OK) return st;
  const long long pages = cache[0], page = cache[1], page_stride = cache[2], width = cache[3], table_stride = cache[4];
  if (pages < 1 || !power_of_two(page) || page < 16 || page > 4096 || page_stride < c.p.Hkv * page * c.D || width < 1 || table_stride < width) return FMHA_I8_ERR_BAD_SHAPE;
  if (pages > 0x7FFFFFFELL || width > ((1LL << 30) / page) || too_far(pages, page_stride, 1) || too_far(c.p.B, table_stride, 4)) return FMHA_I8_ERR_TOO_LARGE;
  if (page_stride % 16 != 0 || !aligned(page_table, 4) || !aligned(lens_k, 4)) return FMHA_I8_ERR_MISALIGNED;
  c.p.lens_k = lens_k;
  c.p.page_table = page_table;
  c.p.table_stride = table_stride;
  c.p.table_width = static_cast<int>(width);
  c.p.page_shift = log2_of(page);
  c.p.num_pages = static_cast<int>(pages);
  c.p.box_shift = std::min(c.p.page_shift, log2_of(grouped::kTile));
  c.lk = KeyLayout{pages, c.p.Hkv, page, c.D, page * c.D, page_stride, 1 << c.p.box_shift};
  c.lv = c.lk;
  c.max_k = std::min(c.max_k, width * page);
  return run_attention(stream, c);
}

int rope_table_impl(void* stream, const double* inv_freq, int pairs, long long positions, double magnitude, float* table) {
  if (!inv_freq || !table) return FMHA_I8_ERR_NULL_POINTER;
  if (pairs < 1 || pairs > 64 || positions < 0) return FMHA_I8_ERR_BAD_SHAPE;
  if (positions > 0x7FFFFFFFLL) return FMHA_I8_ERR_TOO_LARGE;
  if (!std::isfinite(magnitude)) return FMHA_I8_ERR_BAD_AMAX;
  if (!aligned(inv_freq, 8) || !aligned(table, 16)) return FMHA_I8_ERR_MISALIGNED;
  Device dev;
  const int st = fmha_host::device_for_call(&dev);
  if (st != FMHA_I8_OK || positions == 0) return st;
  const long long blocks = std::min((positions * pairs + 255) / 256, 32LL * dev.sm_count);
  rope::rope_table_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(inv_freq, pairs, positions, magnitude, table);
  fmha_host::count_launch();
  return cudaGetLastError() == cudaSuccess ? FMHA_I8_OK : FMHA_I8_ERR_LAUNCH;
}

template <typename T> int launch_append(cudaStream_t stream, const rope::Params& p, int D, bool interleaved, unsigned grid) {
  auto* fn = D == 128 ? (interleaved ? rope::append_kernel<128, T, true> : rope::append_kernel<128, T, false>)
                      : (interleaved ? rope::append_kernel<64, T, true> : rope::append_kernel<64, T, false>);
  return launch(fn, grid, rope::kThreads, 0, stream, 0u, p);
}

int append_impl(void* stream, const float amax[5], const long long dims[5], const void* q, const void* k, const void* v, int in_type, const long long strides[3],
                const int* positions, const float* table, long long in_table, int interleaved, int8_t* q_out, int8_t* k_out, int8_t* v_out, const long long* slots,
                const long long cache[3]) {
  if (!amax || !dims || !q || !k || !v || !strides || !positions || !q_out || !k_out || !v_out || (slots && !cache)) return FMHA_I8_ERR_NULL_POINTER;
  const long long tokens = dims[0], H = dims[1], Hkv = dims[2], D = dims[3], rot = dims[4];
  if (tokens < 0 || H < 1 || Hkv < 1 || (D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0) return FMHA_I8_ERR_BAD_SHAPE;
  if (in_type != FMHA_I8_TYPE_BF16 && in_type != FMHA_I8_TYPE_FP16 && in_type != FMHA_I8_TYPE_FP32) return FMHA_I8_ERR_BAD_SHAPE;
  if (rot > 0 && !table) return FMHA_I8_ERR_NULL_POINTER;
  if (H > 65536 || Hkv > 65536) return FMHA_I8_ERR_TOO_LARGE;
  if (in_table < 0 || strides[0] < H * D || strides[1] < Hkv * D || strides[2] < Hkv * D) return FMHA_I8_ERR_BAD_SHAPE;
  if (tokens > kMostRows / (H + 2 * Hkv) || in_table > kMostRows) return FMHA_I8_ERR_TOO_LARGE;
  for (int i = 0; i < 3; ++i)
    if (too_far(tokens, strides[i], type_bytes(in_type))) return FMHA_I8_ERR_TOO_LARGE;
  for (int i = 0; i < 3; ++i)
    if (!(amax[i] > 0.f) || !std::isfinite(amax[i]) || !std::isfinite(127.f / amax[i])) return FMHA_I8_ERR_BAD_AMAX;
  const int bytes = type_bytes(in_type);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(table, 16) || !aligned(positions, 4) || !aligned(q_out, 16) || !aligned(k_out, 16) ||
      !aligned(v_out, 16) || !aligned(slots, 8) || strides[0] * bytes % 16 != 0 || strides[1] * bytes % 16 != 0 || strides[2] * bytes % 16 != 0)
    return FMHA_I8_ERR_MISALIGNED;
  rope::Params p{};
  if (slots) {
    if (cache[0] < 1 || !power_of_two(cache[1]) || cache[1] < 16 || cache[1] > 4096 || cache[2] < Hkv * cache[1] * D) return FMHA_I8_ERR_BAD_SHAPE;
    if (cache[0] > 0x7FFFFFFELL || too_far(cache[0], cache[2], 1)) return FMHA_I8_ERR_TOO_LARGE;
    if (cache[2] % 16 != 0) return FMHA_I8_ERR_MISALIGNED;
    p.page_shift = log2_of(cache[1]);
    p.page_stride = cache[2];
    p.num_slots = cache[0] * cache[1];
  }
  p.q = q; p.k = k; p.v = v;
  p.q_out = q_out; p.k_out = k_out; p.v_out = v_out;
  p.positions = positions;
  p.table = table;
  p.slots = slots;
  p.in_table = in_table;
  p.q_stride = strides[0]; p.k_stride = strides[1]; p.v_stride = strides[2];
  p.tokens = static_cast<int>(tokens);
  p.H = static_cast<int>(H);
  p.Hkv = static_cast<int>(Hkv);
  p.rot = static_cast<int>(rot);
  for (int i = 0; i < 3; ++i) { p.amax[i] = amax[i]; p.scale[i] = 127.f / amax[i]; }
  Device dev;
  int st = fmha_host::device_for_call(&dev);
  if (st != FMHA_I8_OK || tokens == 0) return st;
  p.status = dev.status;
  // Warps that take one round of heads each, up to 48 warps to an SM, then more rounds.  8192 tokens of 48 heads of 128: 42.9 us; with 96 warps 47.2, 160 53.4, 320 54.7 (a
  // warp's later rounds have the table's entries and the position already, and the next heads on their way).
  const int at_once = static_cast<int>(512 / D), all = static_cast<int>((H + 2 * Hkv + at_once - 1) / at_once);
  const long long most_warps = 48LL * dev.sm_count;
  p.rounds = static_cast<int>(std::min<long long>(all, std::max<long long>(1, (tokens * all + most_warps - 1) / most_warps)));
  p.parts = (all + p.rounds - 1) / p.rounds;
  const long long blocks = (tokens * p.parts + rope::kThreads / 32 - 1) / (rope::kThreads / 32);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (in_type == FMHA_I8_TYPE_BF16) return launch_append<__nv_bfloat16>(s, p, static_cast<int>(D), interleaved != 0, grid);
  if (in_type == FMHA_I8_TYPE_FP16) return launch_append<__half>(s, p, static_cast<int>(D), interleaved != 0, grid);
  return launch_append<float>(s, p, static_cast<int>(D), interleaved != 0, grid);
}

}  // namespace

extern "C" {

int fmha_i8_sm100_infer_packed(void* stream, const float amax[5], const int desc6[6], const void* q, const void* k, const void* v,
                               const int* cu_seqlens_q, const int* cu_seqlens_k, void* o, int o_type, const long long tokens[2],
                               const long long strides[4], unsigned flags) {
  return finish(infer_packed_impl(stream, amax, desc6, q, k, v, cu_seqlens_q, cu_seqlens_k, o, o_type, tokens, strides, flags));
}

int fmha_i8_sm100_infer_paged(void* stream, const float amax[5], const int desc6[6], const void* q, const void* k_cache, const void* v_cache,
                              const int* page_table, const int* seqlens_k, const int* cu_seqlens_q, void* o, int o_type, long long tokens,
                              const long long strides[2], const long long cache[5], unsigned flags) {
  return finish(infer_paged_impl(stream, amax, desc6, q, k_cache, v_cache, page_table, seqlens_k, cu_seqlens_q, o, o_type, tokens, strides, cache, flags));
}

int fmha_i8_sm100_rope_table(void* stream, const double* inv_freq, int pairs, long long positions, double magnitude, float* table) {
  return finish(rope_table_impl(stream, inv_freq, pairs, positions, magnitude, table));
}

int fmha_i8_sm100_rope_quantize_append(void* stream, const float amax[5], const long long dims[5], const void* q, const void* k, const void* v, int in_type,
                                       const long long strides[3], const int* positions, const float* table, long long positions_in_table,
                                       int interleaved, int8_t* q_out, int8_t* k_out, int8_t* v_out, const long long* slots, const long long cache[3]) {
  return finish(append_impl(stream, amax, dims, q, k, v, in_type, strides, positions, table, positions_in_table, interleaved, q_out, k_out, v_out, slots, cache));
}

}  // extern "C"
