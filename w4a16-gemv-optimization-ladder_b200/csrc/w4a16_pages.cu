// Bookkeeping of a paged key-value cache on the device, so that a captured serving loop can
// grow, fork, free and compact its sequences without the host:
//   tables  int32 [sequences][width]  the pages of each sequence in order, -1 past the last
//   lengths int32 [sequences]         positions held
//   refs    int32 [pages]             number of table entries that hold the page (0: free)
// Whole pages may be shared by several sequences; a partly filled page belongs to one.
//
// extend, fork and compact first run one CTA that decides which page goes where (k_pages_plan,
// k_compact_plan); what is proportional to table widths or page contents is done by one
// grid-wide kernel after it (k_pages_apply).  Every kernel is launched with programmatic stream
// serialisation and waits for the one before it before it reads or writes anything.
#include <cuda_runtime.h>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

constexpr int kPlanThreads = kPagesMaxRequests;  // one thread per request

// Exclusive prefix sum over the CTA; *total gets the sum.  `sh` holds 33 values; callable
// again after the next __syncthreads.
__device__ __forceinline__ int block_prefix(int v, int* sh, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) sh[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int n = (int)(blockDim.x >> 5);
    int w = lane < n ? sh[lane] : 0, s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += x;
    }
    sh[lane] = s - w;
    if (lane == 31) sh[32] = s;
  }
  __syncthreads();
  *total = sh[32];
  return sh[warp] + inc - v;
}

// Serves the requests of one call in order.  extend (src == nullptr): sequence seqs[i] grows by
// counts[i] positions.  fork: seqs[i] (empty) becomes a copy of src[i]; it needs a page of its
// own for src's partly filled one.  Request i is refused (ok 0, nothing changed) when its
// arguments are out of range, when an earlier request names the same seqs[i], when the page that a fork
// would copy is none of the pool, or when the free pages do not suffice for all requests up to it.
__global__ void __launch_bounds__(kPlanThreads) k_pages_plan(const PagesState st, const int* seqs,
                                                             const int* src, const int* counts,
                                                             int n, int* ok, int2* moves) {
  __shared__ int sh[33], named[kPlanThreads], cum[kPlanThreads], first[kPlanThreads], copied[kPlanThreads];
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = threadIdx.x;
  auto free_of = [&](int p0) {  // which of this thread's 4 pages from p0 on are free
    unsigned b = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (p0 + 4 * i + k < st.pages && st.refs[p0 + 4 * i + k] == 0) b |= 1u << k;
    return b;
  };
  const int seq = i < n ? seqs[i] : -1;
  const unsigned first_bits = free_of(0);  // asked for along with the requests
  named[i] = seq;
  __syncthreads();
  const int mask = (1 << st.page_shift) - 1;
  const long long cap = (long long)st.width << st.page_shift;
  bool valid = i < n && seq >= 0 && seq < st.sequences;
  if (i < n) {
#pragma unroll 8
    for (int j = 0; j < i; ++j) valid &= named[j] != seq;
  }
  int need = 0, length = 0, from = 0, grown = 0, last = -1;
  if (valid) {
    length = st.lengths[seq];
    if (src) {
      from = src[i];
      valid = from >= 0 && from < st.sequences && from != seq && length == 0;
      if (valid) {
        grown = st.lengths[from];
        valid = grown >= 0 && grown <= cap;
        need = valid && (grown & mask) ? 1 : 0;
        length = grown & ~mask;  // the first position that needs a page of its own
        if (need) {
          last = st.tables[(size_t)from * st.table_stride + (length >> st.page_shift)];  // the page to be copied
          valid = last >= 0 && last < st.pages;
        }
      }
    } else {
      const int c = counts[i];
      valid = c >= 0 && length >= 0 && (long long)length + c <= cap;
      if (valid) {
        grown = length + c;
        need = (int)(((long long)grown + mask) >> st.page_shift) - (int)(((long long)length + mask) >> st.page_shift);
      }
    }
  }
  if (!valid) need = 0;
  int wanted;
  const int before = block_prefix(need, sh, &wanted);
  cum[i] = before + need;
  copied[i] = last;
  first[i] = (int)(((long long)length + mask) >> st.page_shift);  // table column of the request's first new page
  __syncthreads();
  // the lowest free pages, as many as are wanted, 4 for a thread at a time: rank -> request ->
  // table entry.  Which requests are served is known once the free pages are counted, so count,
  // then hand out (from the same registers where the first round has enough pages).
  constexpr int kRound = 4 * kPlanThreads;
  int found = 0, rounds = 0, rank = 0;
  unsigned bits = 0;
  auto look = [&](int p0, int have) {  // free pages of this thread's 4, and their first's rank
    bits = p0 ? free_of(p0) : first_bits;
    int got;
    __syncthreads();
    rank = have + block_prefix(__popc(bits), sh, &got);
    return got;
  };
  for (int p0 = 0; p0 < st.pages && found < wanted; p0 += kRound, ++rounds) found += look(p0, found);
  int have = 0;
  for (int r = 0; r < rounds; ++r) {
    if (rounds > 1) have += look(r * kRound, have);
    for (int k = 0; k < 4; ++k) {
      if (!(bits >> k & 1u)) continue;
      if (rank >= wanted) break;
      int lo = 0, hi = n - 1;  // the first request whose running sum exceeds rank
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] > rank) hi = mid; else lo = mid + 1;
      }
      if (cum[lo] <= found) {
        const int p = r * kRound + 4 * i + k, nth = rank - (lo ? cum[lo - 1] : 0);
        st.refs[p] = 1;
        if (moves) moves[lo] = make_int2(copied[lo], p);
        st.tables[(size_t)named[lo] * st.table_stride + first[lo] + nth] = p;
      }
      ++rank;
    }
  }
  if (i < n) {
    const bool served = valid && (need == 0 || cum[i] <= found);
    ok[i] = served ? 1 : 0;
    if (served) st.lengths[seq] = grown;
    if (moves && !(served && need)) moves[i] = make_int2(-1, -1);
  }
}

// Frees sequences: one CTA per request; the first request that names a sequence counts.
__global__ void __launch_bounds__(256) k_pages_free(const PagesState st, const int* seqs, int n, int* ok) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.x;
  const int seq = seqs[i];
  int again = 0;
  for (int j = threadIdx.x; j < i; j += blockDim.x) again |= seqs[j] == seq;
  again = __syncthreads_or(again);
  const bool valid = seq >= 0 && seq < st.sequences && !again;
  if (threadIdx.x == 0) ok[i] = valid ? 1 : 0;
  if (!valid) return;
  int* row = st.tables + (size_t)seq * st.table_stride;
  for (int c = threadIdx.x; c < st.width; c += blockDim.x) {
    const int p = row[c];
    if (p >= 0 && p < st.pages) atomicSub(st.refs + p, 1);
    row[c] = -1;
  }
  if (threadIdx.x == 0) st.lengths[seq] = 0;
}

// Compaction plan, one CTA: with L live pages, the k-th live page at or above L moves to the
// k-th free page below it.  Sources and destinations are disjoint, and no page moves that
// does not have to.  One prefix sum of the live pages is all it takes: with n live pages before
// page p and B live pages below L, a live page p >= L is the (n - B)-th to move, a free page
// p < L the (p - n)-th to be filled.
__global__ void __launch_bounds__(1024) k_compact_plan(const int* refs, int pages, int* refs_out, int* where,
                                                       int2* moves, int* moved) {
  __shared__ int sh[33], sh_below;
  grid_dependency_wait();
  grid_launch_dependents();
  const int per = (pages + 1023) / 1024, p0 = min(pages, (int)threadIdx.x * per), p1 = min(pages, p0 + per);
  int live = 0;
#pragma unroll 4
  for (int p = p0; p < p1; ++p) live += refs[p] > 0;
  int total;
  const int before = block_prefix(live, sh, &total);
  if (p0 <= total && total < p1) {  // one thread, unless every page is live
    int n = before;
    for (int p = p0; p < total; ++p) n += refs[p] > 0;
    sh_below = n;
  }
  if (total == pages && threadIdx.x == 0) sh_below = total;
  __syncthreads();
  const int below = sh_below, count = total - below;
  int n = before;
#pragma unroll 4
  for (int p = p0; p < p1; ++p) {
    const int r = refs[p];
    if (r > 0 && p >= total) {
      moves[n - below].x = p;
    } else {
      where[p] = p;
      if (r <= 0 && p < total)
        moves[p - n].y = p;
      else if (refs_out != refs)
        refs_out[p] = r;
    }
    n += r > 0;
  }
  __syncthreads();  // the moves are visible to the CTA
  for (int k = threadIdx.x; k < count; k += 1024) {
    const int2 m = moves[k];
    where[m.x] = m.y;
    refs_out[m.y] = refs[m.x];
    refs_out[m.x] = 0;
  }
  if (threadIdx.x == 0) *moved = count;
}

// The table work that goes with a set of page moves, in the first `ctas` CTAs of k_pages_apply.
struct TableWork {
  int ctas = 0;
  // fork: dst[i] shares the whole pages of src[i] if ok[i]
  PagesState st;
  const int* src = nullptr;
  const int* dst = nullptr;
  const int* ok = nullptr;
  int n = 0;
  // compact: out[e] = where[tables[e]]
  const int* tables = nullptr;
  int* out = nullptr;
  const int* where = nullptr;
  long long entries = 0;
};

// Copies whole pages of every layer, k and v: moves are pairs (src, dst), or two lists.  A pair
// with an index outside [0, pages) is skipped.  Bound by the bytes, read once and written once:
// a group of 32 to 256 threads (1 << lg) takes one page of one layer and pool at a time, a thread
// kFlight 16-byte words in flight, so that small pages do not leave threads idle (60 forks in 24
// layers with pages of 2 KB: 10.8 us with a call of free, 13.5 by 256 threads).  More CTAs than fit at once let the faster SMs
// take more (3.5 GB in all: 566 us, 0.96 of the copy rate, with 32 for each SM, 649 with 4; a fixed
// number, since only the device knows how many pages move).
constexpr int kFlight = 8;
__global__ void __launch_bounds__(256) k_pages_apply(const PageBlocks b, const int2* pairs, const int* src, const int* dst, int n,
                                                     const int* count, const int lg, const TableWork t) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < t.ctas) {
    for (long long e = (long long)blockIdx.x * 256 + tid; e < t.entries; e += (long long)t.ctas * 256) {
      const int p = t.tables[e];
      t.out[e] = p >= 0 && p < b.pages ? t.where[p] : p;
    }
    for (int i = blockIdx.x; i < t.n; i += t.ctas) {
      if (!t.ok[i]) continue;
      const int whole = t.st.lengths[t.dst[i]] >> t.st.page_shift;  // set by the plan; a source may be another request's dst
      const int* from = t.st.tables + (size_t)t.src[i] * t.st.table_stride;
      int* to = t.st.tables + (size_t)t.dst[i] * t.st.table_stride;
      for (int c = tid; c < whole; c += 256) {
        const int p = from[c];
        to[c] = p;
        if (p >= 0 && p < t.st.pages) atomicAdd(t.st.refs + p, 1);
      }
    }
    return;
  }
  if (count) n = min(n, *count);
  const long long items = 2LL * n * b.layers;
  const int words = (int)(b.page_bytes / 16);
  const int group = 1 << lg, at = tid & (group - 1), groups = 256 >> lg;  // this thread's place in its group
  const int step = (gridDim.x - t.ctas) * groups;
  for (long long e = (int)((blockIdx.x - t.ctas) * groups + (tid >> lg)); e < items; e += step) {
    const int which = (int)(e & 1), i = e >> 33 ? (int)((e >> 1) / b.layers) : (int)((uint32_t)(e >> 1) / (uint32_t)b.layers);
    const int layer = (int)((e >> 1) - (long long)i * b.layers);
    const int f = pairs ? pairs[i].x : src[i], d = pairs ? pairs[i].y : dst[i];
    if (f < 0 || f >= b.pages || d < 0 || d >= b.pages || f == d) continue;
    uint8_t* base = static_cast<uint8_t*>(which ? b.v : b.k) + (size_t)layer * b.layer_stride;
    const uint4* from = reinterpret_cast<const uint4*>(base + (size_t)f * b.page_stride);
    uint4* to = reinterpret_cast<uint4*>(base + (size_t)d * b.page_stride);
    for (int w0 = at; w0 < words; w0 += group * kFlight) {
      uint4 x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k)
        if (w0 + group * k < words) x[k] = __ldcs(from + w0 + group * k);
#pragma unroll
      for (int k = 0; k < kFlight; ++k)
        if (w0 + group * k < words) __stcs(to + w0 + group * k, x[k]);
    }
  }
}

int launched(const char* what, cudaError_t e) {
  (void)cudaGetLastError();
  if (e == cudaSuccess) return W4A16_OK;
  set_error("%s launch failed: %s", what, cudaGetErrorString(e));
  return W4A16_ERR_CUDA;
}

int launch_apply(const PageBlocks& b, const int2* pairs, const int* src, const int* dst, int n, const int* count, const TableWork& t,
                 cudaStream_t stream) {
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc != W4A16_OK) return rc;
  int group = 32;
  while (group < 256 && group * kFlight * 16LL < b.page_bytes) group *= 2;
  const long long ctas = (2LL * n * b.layers + 256 / group - 1) / (256 / group), most = (long long)sms * 32;
  return launched("k_pages_apply", launch_maybe_pdl(k_pages_apply, dim3((unsigned)(t.ctas + (ctas < most ? ctas : most))), dim3(256), 0,
                                                    stream, true, b, pairs, src, dst, n, count, __builtin_ctz(group), t));
}

}  // namespace

int launch_pages_extend(const PagesState& st, const int* seqs, const int* counts, int n, int* ok, cudaStream_t stream) {
  return launched("k_pages_plan", launch_maybe_pdl(k_pages_plan, dim3(1), dim3(kPlanThreads), 0, stream, true, st, seqs,
                                                   (const int*)nullptr, counts, n, ok, (int2*)nullptr));
}

int launch_pages_fork(const PagesState& st, const PageBlocks& b, const int* src, const int* dst, int n, int* ok, void* scratch,
                      cudaStream_t stream) {
  int2* moves = static_cast<int2*>(scratch);
  const int rc = launched("k_pages_plan", launch_maybe_pdl(k_pages_plan, dim3(1), dim3(kPlanThreads), 0, stream, true, st, dst, src,
                                                           (const int*)nullptr, n, ok, moves));
  if (rc != W4A16_OK) return rc;
  TableWork t;
  t.ctas = n < 128 ? n : 128;
  t.st = st;
  t.src = src;
  t.dst = dst;
  t.ok = ok;
  t.n = n;
  return launch_apply(b, moves, nullptr, nullptr, n, nullptr, t, stream);
}

int launch_pages_free(const PagesState& st, const int* seqs, int n, int* ok, cudaStream_t stream) {
  return launched("k_pages_free", launch_maybe_pdl(k_pages_free, dim3(n), dim3(256), 0, stream, true, st, seqs, n, ok));
}

int launch_pages_copy(const PageBlocks& b, const int* src, const int* dst, int n, cudaStream_t stream) {
  return launch_apply(b, nullptr, src, dst, n, nullptr, TableWork(), stream);
}

size_t pages_compact_scratch_bytes(int pages) { return (size_t)pages * 12; }

int launch_pages_compact(const PageBlocks& b, const int* tables, int* tables_out, long long entries, const int* refs, int* refs_out,
                         int* moved, void* scratch, cudaStream_t stream) {
  int2* moves = static_cast<int2*>(scratch);
  int* where = reinterpret_cast<int*>(moves + b.pages);
  const int rc = launched("k_compact_plan", launch_maybe_pdl(k_compact_plan, dim3(1), dim3(1024), 0, stream, true, refs, b.pages, refs_out,
                                                             where, moves, moved));
  if (rc != W4A16_OK) return rc;
  TableWork t;
  t.tables = tables;
  t.out = tables_out;
  t.where = where;
  t.entries = entries;
  t.ctas = (int)((entries + 1023) / 1024 < 128 ? (entries + 1023) / 1024 : 128);
  return launch_apply(b, moves, nullptr, nullptr, b.pages, moved, t, stream);
}

}  // namespace w4a16
