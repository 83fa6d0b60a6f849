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
// Bound by the rows read and written.  A warp takes a piece of a row, up to 2 KB of it (four loads of 16 bytes a lane, all
// under way before the first is used).
constexpr int kFwdLoads = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const Tokens t, const T* __restrict__ w, long long ldw, T* __restrict__ y, long long ldy, int H,
                     float scale, int pieces) {
  constexpr int N = VEC ? Granule<T>::N : 1, kPiece = 32 * N * kFwdLoads;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int i = static_cast<int>(item / pieces), c0 = static_cast<int>(item % pieces) * kPiece + lane * N;
  if (i >= t.n) return;
  const long long r = load_id(t.ids, t.at(i), t.is64) - t.first;
  const bool in = r >= 0 && r < t.rows;
  const T* src = w + (in ? r : 0) * ldw + c0;
  T* dst = y + i * ldy + c0;
  if constexpr (VEC) {
    uint4 u[kFwdLoads];
#pragma unroll
    for (int k = 0; k < kFwdLoads; ++k)
      u[k] = in && c0 + k * 32 * N < H ? __ldg(reinterpret_cast<const uint4*>(src + k * 32 * N)) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kFwdLoads; ++k) {
      if (c0 + k * 32 * N >= H) continue;
      float f[N];
      Granule<T>::unpack(u[k], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= scale;
      *reinterpret_cast<uint4*>(dst + k * 32 * N) = Granule<T>::pack(f);
    }
  } else {
    float f[kFwdLoads];
#pragma unroll
    for (int k = 0; k < kFwdLoads; ++k) f[k] = in && c0 + k * 32 < H ? Elem<T>::to_f(src[k * 32]) * scale : 0.0f;
#pragma unroll
    for (int k = 0; k < kFwdLoads; ++k)
      if (c0 + k * 32 < H) dst[k * 32] = Elem<T>::from_f(f[k]);
  }
}

// ------------------------------------------------------------------ tokens in the order of their rows
// A stable radix sort by one cluster of 8 CTAs (the first of the grid), 256 warps that each own a contiguous piece of the tokens.  A pass counts
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

__device__ void embedding_sort(const Tokens& t, const SortBuffers& b, int* sort_smem) {
  int* hist = sort_smem;                              // [warp][bin]
  int* total = hist + kSortWarps * kSortBins;         // [bin], read by the other CTAs
  int* scan = total + kSortBins;                      // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = cluster_ctarank();
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

// Zeros in the rows [begin, end) of the table that no token has: the CTA looks through all tokens and marks the rows that occur
// in a bit map.  It needs nothing of the sort and runs beside it.
__device__ void embedding_fill(const Tokens& t, long long begin, long long end, float* dw, long long ldw, int H, bool vec, uint32_t* map) {
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int count = static_cast<int>(end - begin);
  for (int i = tid; i < (count + 31) / 32; i += threads) map[i] = 0;
  __syncthreads();
  constexpr int kAhead = 8;
  for (int i0 = tid; i0 < t.n; i0 += threads * kAhead) {
    long long id[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * threads;
      id[k] = i < t.n ? load_id(t.ids, t.at(i), t.is64) : t.padding;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long r = id[k] - t.first - begin;
      if (i0 + k * threads < t.n && r >= 0 && r < count && id[k] != t.padding) atomicOr(map + (r >> 5), 1u << (r & 31));
    }
  }
  __syncthreads();
  for (int r = warp; r < count; r += threads / 32) {
    if (map[r >> 5] >> (r & 31) & 1) continue;
    float* dst = dw + (begin + r) * ldw;
    if (vec) {
      for (int c = lane * 4; c < H; c += 128) *reinterpret_cast<float4*>(dst + c) = make_float4(0, 0, 0, 0);
    } else {
      for (int c = lane; c < H; c += 32) dst[c] = 0.0f;
    }
  }
}

// The first cluster sorts; with FILL the CTAs of the others write the zeros of `fill_rows` rows each.
__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const Tokens t, const SortBuffers b, float* dw, long long ldw, int H, int vec, int fill_rows) {
  extern __shared__ int sort_smem[];
  pdl_wait();
  if (blockIdx.x < kSortCtas) {
    embedding_sort(t, b, sort_smem);
  } else {
    const long long begin = static_cast<long long>(blockIdx.x - kSortCtas) * fill_rows;
    const long long end = begin + fill_rows < t.rows ? begin + fill_rows : t.rows;
    if (begin < end) embedding_fill(t, begin, end, dw, ldw, H, vec, reinterpret_cast<uint32_t*>(sort_smem));
  }
}

// ------------------------------------------------------------------ sums over the sorted tokens
// Eight columns of a row's 256-column block a lane: consecutive ones with 16-byte accesses (VEC), else every 32nd.
template <typename T, bool VEC> struct Columns {
  int c0, H;
  __device__ __forceinline__ Columns(int block, int lane, int h) : c0(block * 256 + (VEC ? lane * 8 : lane)), H(h) {}
  struct Raw {
    uint4 u[VEC ? 8 * sizeof(T) / 16 : 1];
    T e[VEC ? 1 : 8];
  };
  __device__ __forceinline__ void load(const T* row, Raw& v) const {
    if constexpr (VEC) {
      constexpr int L = 8 * sizeof(T) / 16;
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (c0 < H) v.u[i] = __ldg(reinterpret_cast<const uint4*>(row + c0) + i);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + 32 * j < H) v.e[j] = row[c0 + 32 * j];
    }
  }
  __device__ __forceinline__ void add(const Raw& v, float (&acc)[8]) const {
    if constexpr (VEC) {
      constexpr int N = Granule<T>::N, L = 8 / N;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        float f[N];
        Granule<T>::unpack(v.u[i], f);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[i * N + j] += f[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += Elem<T>::to_f(v.e[j]);
    }
  }
  __device__ __forceinline__ void write(float* row, const float (&acc)[8], float scale, int accumulate) const {
    if constexpr (VEC) {
      if (c0 >= H) return;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float4* p = reinterpret_cast<float4*>(row + c0) + i;
        const float4 old = accumulate ? *p : make_float4(0, 0, 0, 0);
        *p = make_float4(fmaf(scale, acc[4 * i], old.x), fmaf(scale, acc[4 * i + 1], old.y), fmaf(scale, acc[4 * i + 2], old.z),
                         fmaf(scale, acc[4 * i + 3], old.w));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float* p = row + c0 + 32 * j;
        if (c0 + 32 * j < H) *p = fmaf(scale, acc[j], accumulate ? *p : 0.0f);
      }
    }
  }
};

struct SumArgs {
  const void* dy;
  float* dw;
  float* part;       // [chunks][2][blocks * 256]: sums of a chunk's tokens whose row began in an earlier chunk / goes on in the next
  long long ldy, ldw, rows;
  int H, blocks;     // blocks of 256 columns
  float scale;
  int accumulate;
};

enum { kHead = 1, kThrough = 2, kTail = 4 };

// One CTA's chunk [lo, hi) of n sorted tokens, a piece of PIECE of them a warp, one block of columns.  A warp runs through its
// rows of dy, eight of them under way, and stores a row's sum where the row's tokens all lie in its piece.  Of the others the
// first (began in an earlier piece) and the last (goes on in the next) go to shared memory; then the warp in whose
// piece a row began adds up the pieces in order.  Rows that cross the chunk's ends go to `part`.  So a token that
// makes up a large share of the batch is summed by many warps, and always in the same order.
template <typename T, bool VEC, int WARPS>
__device__ void embedding_sums(const uint32_t* key, const uint32_t* pos, int n, int lo, int hi, int piece, int chunk, int block,
                               const SumArgs& a, float (*slots)[2][256], int* flags) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Columns<T, VEC> cols(block, lane, a.H);
  const T* dy = static_cast<const T*>(a.dy);
  const uint32_t none = static_cast<uint32_t>(a.rows);
  const int p0 = min(lo + warp * piece, hi), p1 = min(p0 + piece, hi);
  int mark = 0;
  float acc[8] = {};
  uint32_t cur = none;
  bool began = true;      // the present row's tokens begin in this piece
  auto keep = [&](int which) {
#pragma unroll
    for (int j = 0; j < 8; ++j) slots[warp][which][j * 32 + lane] = acc[j];
  };
  auto finish = [&]() {   // no more tokens of `cur` in this piece or after it
    if (cur == none) return;
    if (began) {
      cols.write(a.dw + cur * a.ldw, acc, a.scale, a.accumulate);
    } else {
      keep(0);
      mark |= kHead;
    }
  };
  if (p0 < p1) {
    const uint32_t before = p0 > 0 ? key[p0 - 1] : none;
    constexpr int kAhead = 8;
    for (int i = p0; i < p1; i += 32) {
      const int left = min(32, p1 - i);
      const uint32_t my_key = lane < left ? key[i + lane] : none, my_pos = lane < left ? pos[i + lane] : 0;
      if (__shfl_sync(0xffffffffu, my_key, 0) == none) break;      // only tokens of no row from here on
      for (int j0 = 0; j0 < left; j0 += kAhead) {
        typename Columns<T, VEC>::Raw v[kAhead];
        uint32_t k[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          k[u] = __shfl_sync(0xffffffffu, my_key, j0 + u);
          const uint32_t p = __shfl_sync(0xffffffffu, my_pos, j0 + u);
          if (k[u] != none) cols.load(dy + p * a.ldy, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (j0 + u >= left) break;
          if (k[u] != cur || (i == p0 && j0 + u == 0)) {
            finish();
            began = i != p0 || j0 + u != 0 || p0 == 0 || before != k[u];
            cur = k[u];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
          }
          if (cur != none) cols.add(v[u], acc);
        }
      }
    }
    const bool goes_on = cur != none && p1 < n && key[p1] == cur;
    if (!goes_on) {
      finish();
    } else if (began) {
      keep(1);
      mark |= kTail;
    } else {
      keep(0);
      mark |= kHead | kThrough;
    }
  }
  if (lane == 0) flags[warp] = mark;
  __syncthreads();
  auto chain = [&](int x) {      // adds the heads from piece x on; true where the row ends in the chunk
    for (; x < WARPS; ++x) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += slots[x][0][j * 32 + lane];
      if (!(flags[x] & kThrough)) return true;
    }
    return false;
  };
  auto store_part = [&](int which) {
    float* p = a.part + ((static_cast<long long>(chunk) * 2 + which) * a.blocks + block) * 256;
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j * 32 + lane] = acc[j];
  };
  if (mark & kTail) {            // (acc is the tail)
    if (chain(warp + 1)) cols.write(a.dw + cur * a.ldw, acc, a.scale, a.accumulate);
    else store_part(1);
  }
  if (warp == 0 && (mark & kHead)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    chain(0);
    store_part(0);
  }
}

constexpr int kSumWarps = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumWarps * 32)
embedding_sums_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int n, int piece, const SumArgs a) {
  __shared__ float slots[kSumWarps][2][256];
  __shared__ int flags[kSumWarps];
  pdl_wait();
  const int chunk = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks, lo = chunk * piece * kSumWarps;
  embedding_sums<T, VEC, kSumWarps>(key, pos, n, lo, min(lo + piece * kSumWarps, n), piece, chunk, block, a, slots, flags);
}

// Rows that cross ends of chunks: a warp per chunk and block of columns adds up, in order, the row that begins in its chunk and
// goes on in the next.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
embedding_join_kernel(const uint32_t* __restrict__ key, int n, int length, int chunks, const SumArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int chunk = static_cast<int>(item / a.blocks), block = static_cast<int>(item % a.blocks);
  const long long next = static_cast<long long>(chunk + 1) * length;      // first token of the next chunk
  if (next >= n) return;
  const uint32_t k = key[next];
  if (k == static_cast<uint32_t>(a.rows) || key[next - 1] != k || (chunk > 0 && key[next - length - 1] == k)) return;
  // the last chunk of the row: the first whose own last token is another's
  int last = chunk + 1;
  while (true) {
    const long long e = static_cast<long long>(last + lane + 1) * length;      // end of chunk last + lane
    const unsigned more = __ballot_sync(0xffffffffu, e < n && key[e] == k);
    if (more != 0xffffffffu) {
      last += __ffs(~more) - 1;
      break;
    }
    last += 32;
  }
  const float* p = a.part + (static_cast<long long>(chunk) * 2 + 1) * a.blocks * 256 + block * 256 + lane;
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = p[j * 32];
  p += a.blocks * 256;      // [chunk + 1][0]
  const long long step = 2ll * a.blocks * 256;
#pragma unroll 4
  for (int c = chunk + 1; c <= last; ++c, p += step) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += p[j * 32];
  }
  const Columns<T, VEC> cols(block, lane, a.H);
  cols.write(a.dw + k * a.ldw, acc, a.scale, a.accumulate);
}

// ------------------------------------------------------------------ few tokens
// One launch: the first CTAs take a block of columns each and order the tokens by themselves (a token's place is the
// number of smaller keys and of equal ones before it), the others write the zeros.
constexpr int kFewTokens = 512, kFewWarps = 16;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kFewWarps * 32)
embedding_few_kernel(const Tokens t, const SumArgs a, int vec_fill, int fill_rows) {
  __shared__ __align__(16) uint32_t raw[kFewTokens];
  __shared__ uint32_t key[kFewTokens], pos[kFewTokens];
  __shared__ float slots[kFewWarps][2][256];
  __shared__ int flags[kFewWarps];
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= a.blocks) {
    const long long begin = static_cast<long long>(blockIdx.x - a.blocks) * fill_rows;
    embedding_fill(t, begin, min(begin + fill_rows, t.rows), a.dw, a.ldw, a.H, vec_fill, reinterpret_cast<uint32_t*>(slots));
    return;
  }
  const int i = threadIdx.x, padded = (t.n + 3) / 4 * 4;
  uint32_t mine = 0xffffffffu;
  if (i < t.n) {
    const long long id = load_id(t.ids, t.at(i), t.is64), r = id - t.first;
    mine = static_cast<uint32_t>(r >= 0 && r < t.rows && id != t.padding ? r : t.rows);
  }
  if (i < padded) raw[i] = mine;
  __syncthreads();
  if (i < t.n) {
    int place = 0;
    for (int j = 0; j < padded; j += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(raw + j);
      place += (k.x < mine || (k.x == mine && j < i)) + (k.y < mine || (k.y == mine && j + 1 < i)) +
               (k.z < mine || (k.z == mine && j + 2 < i)) + (k.w < mine || (k.w == mine && j + 3 < i));
    }
    key[place] = mine;
    pos[place] = i;
  }
  __syncthreads();
  embedding_sums<T, VEC, kFewWarps>(key, pos, t.n, 0, t.n, (t.n + kFewWarps - 1) / kFewWarps, 0, blockIdx.x, a, slots, flags);
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
  const int piece = 32 * kFwdLoads * (vec ? Granule<T>::N : 1), pieces = (H + piece - 1) / piece;
  const long long grid = (static_cast<long long>(t.n) * pieces + 7) / 8;
  if (grid > 0x7fffffffll) return kErrTooLarge;
  launch_pdl(vec ? embedding_fwd_kernel<T, true> : embedding_fwd_kernel<T, false>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s,
             1, t, static_cast<const T*>(w), ldw, static_cast<T*>(y), ldy, H, scale, pieces);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

static int key_bits(long long rows) {   // keys are 0 .. rows
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;
  return bits;
}

// Tokens a warp sums: 32 where that leaves 32 warps for every SM, else 8.  5105 tokens of 1600 columns: PIECE8 us against PIECE32.
static int sum_piece(int n, int H) { return static_cast<long long>(n) * ((H + 255) / 256) >= 32ll * 32 * num_sms() ? 32 : 8; }

// Rows a CTA of `ctas` fills, at most what its bit map (of `bits`) holds.
static int fill_rows_of(long long rows, int ctas, int bits) {
  const long long r = (rows + ctas - 1) / ctas;
  return static_cast<int>(r < bits ? r : bits);
}

template <typename T, bool VEC>
static int embedding_bwd_launch(const Tokens& t, const SumArgs& args, uint32_t* ws, cudaStream_t s) {
  SumArgs a = args;
  const int vec_fill = a.H % 4 == 0 && a.ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(a.dw) & 15) == 0;
  if (t.n <= kFewTokens) {
    const int fill_rows = fill_rows_of(t.rows, 2 * num_sms(), kFewWarps * 2 * 256 * 32);
    const long long fill = a.accumulate ? 0 : (t.rows + fill_rows - 1) / fill_rows;
    launch_pdl(embedding_few_kernel<T, VEC>, dim3(static_cast<unsigned>(a.blocks + fill)), dim3(kFewWarps * 32), 0, s, 1, t, a, vec_fill,
               fill_rows);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
  }
  const int bits = key_bits(t.rows);
  SortBuffers b;
  for (int k = 0; k < 2; ++k) {
    b.key[k] = ws + 2ll * k * t.n;
    b.pos[k] = ws + (2ll * k + 1) * t.n;
  }
  b.passes = (bits + 8) / 9;
  b.bits = (bits + b.passes - 1) / b.passes;
  a.part = reinterpret_cast<float*>(ws + 4ll * t.n);
  static unsigned long long ready = 0;      // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(ready >> dev & 1)) {
    if (cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) != cudaSuccess)
      return kErrLaunch;
    if (dev < 64) ready |= 1ull << dev;
  }
  // one CTA of the sort kernel an SM, in clusters of 8
  const int fill_rows = fill_rows_of(t.rows, (num_sms() / kSortCtas - 1) * kSortCtas, static_cast<int>(kSortSmem) * 8);
  const long long fill = a.accumulate ? 0 : (t.rows + fill_rows - 1) / fill_rows;
  launch_pdl(embedding_sort_kernel, dim3(static_cast<unsigned>((1 + (fill + kSortCtas - 1) / kSortCtas) * kSortCtas)), dim3(kSortThreads),
             kSortSmem, s, kSortCtas, t, b, a.dw, a.ldw, a.H, vec_fill, fill_rows);
  const uint32_t* key = b.key[(b.passes - 1) & 1];
  const uint32_t* pos = b.pos[(b.passes - 1) & 1];
  const int piece = sum_piece(t.n, a.H), length = piece * kSumWarps, chunks = (t.n + length - 1) / length;
  const long long grid = static_cast<long long>(chunks) * a.blocks;
  if (grid > 0x7fffffffll) return kErrTooLarge;
  launch_pdl(embedding_sums_kernel<T, VEC>, dim3(static_cast<unsigned>(grid)), dim3(kSumWarps * 32), 0, s, 1, key, pos, t.n, piece, a);
  launch_pdl(embedding_join_kernel<T, VEC>, dim3(static_cast<unsigned>((grid + 7) / 8)), dim3(256), 0, s, 1, key, t.n, length, chunks, a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
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
  if (n <= kFewTokens) return 1;
  const long long length = sum_piece(n, H) * kSumWarps, chunks = (n + length - 1) / length, blocks = (H + 255) / 256;
  const long long bytes = 16ll * n + chunks * 2 * blocks * 256 * 4;
  return static_cast<int>((bytes + 255) / 256);
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
  const SumArgs a{dy, dw, nullptr, ldy, ldw, rows, H, (H + 255) / 256, scale, accumulate};
  const int unit = dtype == 2 ? 4 : 8;      // elements of 16 bytes
  const bool vec = H % 8 == 0 && ldy % unit == 0 && ldw % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dw)) & 15) == 0;
  uint32_t* ws = static_cast<uint32_t*>(workspace);
  if (dtype == 0) return vec ? embedding_bwd_launch<__half, true>(t, a, ws, s) : embedding_bwd_launch<__half, false>(t, a, ws, s);
  if (dtype == 1)
    return vec ? embedding_bwd_launch<__nv_bfloat16, true>(t, a, ws, s) : embedding_bwd_launch<__nv_bfloat16, false>(t, a, ws, s);
  return vec ? embedding_bwd_launch<float, true>(t, a, ws, s) : embedding_bwd_launch<float, false>(t, a, ws, s);
}
