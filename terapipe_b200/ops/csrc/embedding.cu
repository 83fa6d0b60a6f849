// Embedding rows for a batch of tokens, scaled, and the table's gradient.
//
//   y[i] = scale * W[id_i - first]                                 (zeros where id_i is in no row of this table)
//   dW[v] (+)= scale * sum over i with id_i - first = v of dy[i]   (fp32; without the padding token)
//
// The table may be one tensor-parallel rank's part of the vocabulary, rows [first, first + rows).
#include "common.cuh"
#include "granule.cuh"

namespace tp {

struct Tokens {
  const void* ids;
  OuterIndex at;
  long long first, rows, padding;   // padding: an id that gets no gradient; -1 (no id) where there is none
  int n, is64;
};

// ------------------------------------------------------------------ lookup
// A warp per row.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const Tokens t, const T* __restrict__ w, long long ldw, T* __restrict__ y, long long ldy, int H,
                     float scale) {
  constexpr int N = Granule<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  const long long i = static_cast<long long>(blockIdx.x) * 8 + warp;
  if (i >= t.n) return;
  const long long r = load_id(t.ids, t.at(i), t.is64) - t.first;
  const bool in = r >= 0 && r < t.rows;
  const T* src = w + (in ? r : 0) * ldw;
  T* dst = y + i * ldy;
  if (VEC) {
    for (int c = lane * N; c < H; c += 32 * N) {
      float f[N] = {};
      if (in) Granule<T>::unpack(*reinterpret_cast<const uint4*>(src + c), f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= scale;
      *reinterpret_cast<uint4*>(dst + c) = Granule<T>::pack(f);
    }
  } else {
    for (int c = lane; c < H; c += 32) dst[c] = Elem<T>::from_f(in ? Elem<T>::to_f(src[c]) * scale : 0.0f);
  }
}

// ------------------------------------------------------------------ tokens in the order of their rows
// A stable radix sort by one cluster of 8 CTAs, 256 warps that each own a contiguous piece of the tokens.  A pass counts
// the digits of every piece (one counter a digit and warp; lanes with the same digit are found by match_any and only the
// first of them counts), turns the counts into destinations (digits, then CTAs, then warps) and moves keys and positions.
// Equal keys keep their order, so that a row's sum does not depend on timing.  Tokens of no row get the key `rows` and
// end up behind all others.
constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBins = 512;
constexpr size_t kSortSmem = (kSortWarps * kSortBins + kSortBins + 2 * 32) * sizeof(int);

struct SortBuffers {
  uint32_t *key[2], *pos[2];   // pass p writes [p & 1]
  int passes, bits;            // digits a key, bits a digit
};

__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const Tokens t, const SortBuffers b) {
  extern __shared__ int sort_smem[];
  int* hist = sort_smem;                              // [warp][bin]
  int* total = hist + kSortWarps * kSortBins;         // [bin], read by the other CTAs
  int* scan = total + kSortBins;                      // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = cluster_ctarank();
  pdl_wait();
  const int piece = ((t.n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) / 32 * 32;
  const long long begin = static_cast<long long>(cta * kSortWarps + warp) * piece;
  const int lo = begin < t.n ? static_cast<int>(begin) : t.n;
  const int hi = begin + piece < t.n ? static_cast<int>(begin) + piece : t.n;
  int* mine = hist + warp * kSortBins;
  for (int p = 0; p < b.passes; ++p) {
    const int shift = p * b.bits, bins = 1 << b.bits, digit_mask = bins - 1;
    const uint32_t* key_in = b.key[(p + 1) & 1];
    const uint32_t* pos_in = b.pos[(p + 1) & 1];
    auto key_of = [&](int i) -> uint32_t {
      if (p > 0) return __ldcg(key_in + i);
      const long long id = load_id(t.ids, t.at(i), t.is64), r = id - t.first;
      return r >= 0 && r < t.rows && id != t.padding ? static_cast<uint32_t>(r) : static_cast<uint32_t>(t.rows);
    };
    for (int d = lane; d < bins; d += 32) mine[d] = 0;
    __syncwarp();
    for (int i = lo + lane; i - lane < hi; i += 32) {
      const bool in = i < hi;
      const int d = in ? (key_of(i) >> shift) & digit_mask : kSortBins;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (in && lane == __ffs(same) - 1) mine[d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (tid < bins) {      // counts of the warps before each, and of the CTA
      int sum = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = hist[w * kSortBins + tid];
        hist[w * kSortBins + tid] = sum;
        sum += c;
      }
      total[tid] = sum;
    }
    cluster_sync_all();
    int before = 0, all = 0;
    if (tid < bins) {
      for (int c = 0; c < kSortCtas; ++c) {
        int v;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(smem_u32(total + tid), c)) : "memory");
        before += c < cta ? v : 0;
        all += v;
      }
    }
    int incl = all;        // running sum over the digits
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (tid < bins) {
      int base = before + incl - all;
      for (int w = 0; w < warp; ++w) base += scan[w];
      for (int w = 0; w < kSortWarps; ++w) hist[w * kSortBins + tid] += base;
    }
    __syncthreads();
    for (int i = lo + lane; i - lane < hi; i += 32) {
      const bool in = i < hi;
      const uint32_t key = in ? key_of(i) : 0;
      const int d = in ? (key >> shift) & digit_mask : kSortBins;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      const int dest = in ? mine[d] + __popc(same & ((1u << lane) - 1)) : 0;
      __syncwarp();
      if (in) {
        if (lane == __ffs(same) - 1) mine[d] += __popc(same);
        __stcg(b.key[p & 1] + dest, key);
        __stcg(b.pos[p & 1] + dest, p > 0 ? __ldcg(pos_in + i) : static_cast<uint32_t>(i));
      }
      __syncwarp();
    }
    __threadfence();
    cluster_sync_all();    // keys and positions are in place; no CTA reads this pass's totals any more
  }
}

// start[v] = number of tokens of rows below v, v in [0, rows].
__global__ void __launch_bounds__(256)
embedding_bounds_kernel(const uint32_t* __restrict__ key, int n, long long rows, int* __restrict__ start) {
  pdl_wait();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i > n) return;
  const long long low = i == 0 ? 0 : static_cast<long long>(key[i - 1]) + 1, high = i == n ? rows : key[i];
  for (long long v = low; v <= high; ++v) start[v] = static_cast<int>(i);
}

// A warp per 256 columns of a row of the table.
template <typename T>
__global__ void __launch_bounds__(256)
embedding_bwd_kernel(const uint32_t* __restrict__ pos, const int* __restrict__ start, const T* __restrict__ dy,
                     long long ldy, float* __restrict__ dw, long long ldw, long long rows, int H, float scale, int accumulate) {
  pdl_wait();
  const int lane = threadIdx.x & 31, blocks = (H + 255) / 256;
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const long long v = item / blocks;
  if (v >= rows) return;
  const int c0 = static_cast<int>(item % blocks) * 256 + lane;
  const int lo = start[v], hi = start[v + 1];
  if (accumulate && lo == hi) return;
  float acc[8] = {};
  for (int i = lo; i < hi; ++i) {
    const T* src = dy + static_cast<long long>(pos[i]) * ldy;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + 32 * j < H) acc[j] += Elem<T>::to_f(src[c0 + 32 * j]);
  }
  float* dst = dw + v * ldw;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c0 + 32 * j < H) dst[c0 + 32 * j] = (accumulate ? dst[c0 + 32 * j] : 0.0f) + scale * acc[j];
}

static bool make_tokens(Tokens* t, const void* ids, int ids64, int n, int cols, long long s0, long long s1, long long first,
                        long long rows, long long padding) {
  if (n < 0 || cols < 1 || rows < 0 || rows >= 0x7fffffffll || (n > 0 && ids == nullptr)) return false;
  *t = Tokens{ids, OuterIndex{s0, s1, cols}, first, rows, padding, n, ids64};
  return true;
}

template <typename T>
static int embedding_fwd_launch(const Tokens& t, const void* w, long long ldw, void* y, long long ldy, int H, float scale,
                                cudaStream_t s) {
  const bool vec = H % Granule<T>::N == 0 && ldw % Granule<T>::N == 0 && ldy % Granule<T>::N == 0 &&
                   ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const dim3 grid((t.n + 7) / 8);
  if (vec)
    launch_pdl(embedding_fwd_kernel<T, true>, grid, dim3(256), 0, s, 1, t, static_cast<const T*>(w), ldw,
               static_cast<T*>(y), ldy, H, scale);
  else
    launch_pdl(embedding_fwd_kernel<T, false>, grid, dim3(256), 0, s, 1, t, static_cast<const T*>(w), ldw,
               static_cast<T*>(y), ldy, H, scale);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

static int key_bits(long long rows) {   // keys are 0 .. rows
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;
  return bits;
}
}  // namespace tp

using namespace tp;

// dtype: 0 fp16, 1 bf16, 2 fp32.  Token i is ids[(i / cols) * s0 + (i % cols) * s1].
extern "C" int tp_embedding_fwd(int dtype, const void* ids, int ids64, int n, int cols, long long s0, long long s1,
                                long long first, const void* w, long long ldw, long long rows, void* y, long long ldy,
                                int H, float scale, void* stream) {
  Tokens t;
  if (!make_tokens(&t, ids, ids64, n, cols, s0, s1, first, rows, -1) || H < 0 || dtype < 0 || dtype > 2) return kErrBadArgument;
  if (n == 0 || H == 0) return kOk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return embedding_fwd_launch<__half>(t, w, ldw, y, ldy, H, scale, s);
  if (dtype == 1) return embedding_fwd_launch<__nv_bfloat16>(t, w, ldw, y, ldy, H, scale, s);
  return embedding_fwd_launch<float>(t, w, ldw, y, ldy, H, scale, s);
}

// Workspace of tp_embedding_bwd in blocks of 256 bytes (base address: a multiple of 16).
extern "C" int tp_embedding_bwd_workspace_blocks(int n, long long rows, int H) {
  return static_cast<int>(((4ll * n + rows + 1) * 4 + 255) / 256);
}

extern "C" int tp_embedding_bwd(int dtype, const void* ids, int ids64, int n, int cols, long long s0, long long s1,
                                long long first, long long padding, const void* dy, long long ldy, float* dw,
                                long long ldw, long long rows, int H, float scale, int accumulate, void* workspace,
                                void* stream) {
  Tokens t;
  if (!make_tokens(&t, ids, ids64, n, cols, s0, s1, first, rows, padding) || H < 0 || dtype < 0 || dtype > 2)
    return kErrBadArgument;
  if (rows == 0 || H == 0 || (n == 0 && accumulate)) return kOk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t* ws = static_cast<uint32_t*>(workspace);
  const int bits = key_bits(rows);
  SortBuffers b;
  for (int k = 0; k < 2; ++k) {
    b.key[k] = ws + 2ll * k * n;
    b.pos[k] = ws + (2ll * k + 1) * n;
  }
  b.passes = (bits + 8) / 9;
  b.bits = (bits + b.passes - 1) / b.passes;
  int* start = reinterpret_cast<int*>(ws + 4ll * n);
  static bool ready = false;
  if (!ready) {
    if (cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) != cudaSuccess)
      return kErrLaunch;
    ready = true;
  }
  const uint32_t* key = b.key[(b.passes - 1) & 1];
  const uint32_t* pos = b.pos[(b.passes - 1) & 1];
  if (n > 0) launch_pdl(embedding_sort_kernel, dim3(kSortCtas), dim3(kSortThreads), kSortSmem, s, kSortCtas, t, b);
  launch_pdl(embedding_bounds_kernel, dim3(n / 256 + 1), dim3(256), 0, s, 1, key, n, rows, start);
  const long long items = rows * ((H + 255) / 256), grid = (items + 7) / 8;
  if (grid > 0x7fffffffll) return kErrTooLarge;
#define EMB_BWD(T)                                                                                                  \
  launch_pdl(embedding_bwd_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, 1, pos,                    \
             static_cast<const int*>(start), static_cast<const T*>(dy), ldy, dw, ldw, rows, H, scale, accumulate)
  if (dtype == 0) EMB_BWD(__half);
  else if (dtype == 1) EMB_BWD(__nv_bfloat16);
  else EMB_BWD(float);
#undef EMB_BWD
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}
