// page_plan.cuh — page table rows, slots and positions of a batch's next
// tokens, from lengths alone, in one launch with no host in between.
//
// No counterpart in the reference (dense padded caches,
// src/pallas_flash/kernels/decoding.py:86-103).  Per sequence b with held
// length L_b (0 if it is released first), N_b new tokens and page size S:
//   have_b = ceil(L_b / S), need_b = ceil((L_b + N_b) / S) - have_b
//   its new pages are ring[head + sum_{b' < b} need_b' + i], i < need_b
//   token i of the packed batch belongs to the b with start_b <= i < start_b
//   + N_b (start = exclusive sum of N), has position L_b + i - start_b and
//   slot page * S + row
// Free pages wait in a ring: they are taken at its head and returned at its
// tail, so the places read and the places written by one call never meet
// (free + returned pages never exceed the ring), and pages of a sequence
// that is released in this call are handed out from the next call on.  A
// release is refused whole where the ring has no room for the pages (they would be
// in neither table nor ring), and only entries that name a page go back.
//
// Every CTA scans all B sequences itself (block-wide sums in 64 bits;
// a second kernel would cost more than the repeated reads of a few KB from
// L2) and then takes its share of table rows and tokens.  Where the state is
// advanced in place, the CTAs form one cluster of 8 and meet at its barrier
// between the last read of the lengths and the first write; with separate
// outputs nothing is shared and the grid grows with the work.
//
// Bound by latency: one read of the lengths, two rounds of scans, the dependent reads
// of table and ring, one write.  Measured back to back in a graph: 256 sequences with
// 2048 table entries each (2 MB of table written) 9 us, 12.6 with 17 of them released
// (their rows are read ahead of the scans, by every CTA, to count the pages that come
// back; one released 9.6); 61 prompts of up to 2500 tokens 9.6; in place 64 sequences 5.9,
// one of them released 7.3.  A call's own host time is 20 us.
#pragma once

#include "paged.cuh"

namespace pu {
namespace plan {

constexpr int kThreads = 1024;
constexpr int kMaxB = 8192;
constexpr int kCluster = 8;

struct Params {
  const int32_t* table;      // [B][max_pages]
  int32_t* table_out;
  const int32_t* lens;       // [B]
  int32_t* lens_out;
  const int32_t* add;        // [B] new tokens
  const uint8_t* release;    // [B] or nullptr
  int32_t* ring;             // [num_pages] free page numbers
  const long long* cursor;   // head, tail (counts that only grow)
  long long* cursor_out;
  int32_t* slots;            // [T]
  int32_t* positions;        // [T]
  int32_t* seq_ids;          // [T]
  int32_t* cu;               // [B + 1]
  int B, max_pages, num_pages, page_shift;
  long long T;
};

// Exclusive block-wide sums of N values per thread; total[i] = the i-th's sum of all.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long (*s_warp)[32], long long (&total)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](long long x) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    return x;
  };
  long long x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = scan(v[i]);
  __syncthreads();                       // the previous scan's sums have been read
  if (lane == 31) {
#pragma unroll
    for (int i = 0; i < N; ++i) s_warp[i][warp] = x[i];
  }
  __syncthreads();
  if (warp < N) s_warp[warp][lane] = scan(s_warp[warp][lane]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    total[i] = s_warp[i][31];
    v[i] = x[i] - v[i] + (warp > 0 ? s_warp[i][warp - 1] : 0);
  }
}

template <bool kInPlace>
__global__ void __launch_bounds__(kThreads) page_plan_kernel(const Params p) {
  extern __shared__ int s_dyn[];
  int* s_start = s_dyn;                  // [B + 1] first token (at most T)
  int* s_base = s_start + p.B + 1;       // [B] tokens held before
  int* s_last = s_base + p.B;            // [B] pages held after
  int* s_new = s_last + p.B;             // [B] ring place of the first new page, from the head
  int* s_freed = s_new + p.B;            // [B] ring place of the first returned page, from the tail; -1: none;
                                         // -2 - place: the row has entries that are no pages
  __shared__ long long s_warp[2][32];
  __shared__ int s_used;                 // pages taken
  __shared__ int s_released;             // rows that return pages
  const int tid = threadIdx.x;
  if (tid == 0) s_used = s_released = 0;
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch_dependents();

  const int page = 1 << p.page_shift;
  const long long cap = (long long)p.max_pages << p.page_shift;
  const long long head = p.cursor[0], tail = p.cursor[1];
  long long avail = tail - head;
  const bool ring_ok = head >= 0 && avail >= 0 && avail <= p.num_pages;
  if (!ring_ok) avail = 0;
  const int head0 = ring_ok ? (int)(head % p.num_pages) : 0, tail0 = ring_ok ? (int)(tail % p.num_pages) : 0;

  // this thread's sequences
  const int per = (p.B + kThreads - 1) / kThreads, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  auto held_of = [&](int b) { return (int)min((long long)max(p.lens[b], 0), cap); };
  auto gone = [&](int b) { return p.release != nullptr && p.release[b] != 0; };
  long long tokens = 0, freed = 0;
  const int lane = tid & 31;
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    const bool mine = b < b1;
    int back = 0;                        // pages that the row returns
    if (mine) {
      const int held = held_of(b);
      if (gone(b)) back = (held + page - 1) >> p.page_shift;
      s_base[b] = gone(b) ? 0 : held;
      s_freed[b] = back;
      tokens += max(p.add[b], 0);
    }
    // a list of the rows that return some, in s_new for now (an atomic for each of
    // them, not each warp, took 2 us)
    const unsigned some = __ballot_sync(0xffffffffu, back > 0);
    if (some == 0) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(&s_released, __popc(some));
    at = __shfl_sync(0xffffffffu, at, 0);
    if (back > 0) {
      s_new[at + __popc(some & ((1u << lane) - 1u))] = b;
      s_last[b] = 0;                     // how many of its entries are pages
    }
  }
  constexpr int kSeg = 512;              // entries a warp takes at once
  const int segs = (p.max_pages + kSeg - 1) / kSeg;
  constexpr int kPiece = 256;            // entries a warp counts at once
  const int pieces = (p.max_pages + kPiece - 1) / kPiece;
  __syncthreads();
  if (s_released > 0) {
    // How many of the released rows' entries name a page (s_freed: -1 - the count where
    // some do not).  A warp has the loads of a piece in flight; with a row for a warp, 17
    // rows of up to 1875 entries took 5 us, pieces of 256 take 3.2, of 512 and 128 3.6, 4.2.
    const unsigned units = (unsigned)s_released * (unsigned)pieces;      // 2^13 * 2^18 at most
    for (unsigned u = tid >> 5; u < units; u += kThreads / 32) {
      const unsigned row = u / (unsigned)pieces;
      const int b = s_new[row], lo = (int)(u - row * pieces) * kPiece, n = min(s_freed[b] - lo, kPiece);
      if (n <= 0) continue;
      const int32_t* in = p.table + (size_t)b * p.max_pages + lo;
      int entry[kPiece / 32], good = 0;
#pragma unroll
      for (int i = 0; i < kPiece / 32; ++i) entry[i] = i * 32 < n ? in[min(i * 32 + lane, n - 1)] : -1;
#pragma unroll
      for (int i = 0; i < kPiece / 32; ++i) good += i * 32 + lane < n && (unsigned)entry[i] < (unsigned)p.num_pages;
      good = __reduce_add_sync(0xffffffffu, good);
      if (lane == 0 && good > 0) atomicAdd(&s_last[b], good);
    }
    __syncthreads();
    for (int b = b0; b < b1; ++b) {
      if (s_freed[b] == 0) continue;
      const int good = s_last[b];
      freed += good;
      if (good != s_freed[b]) s_freed[b] = -1 - good;
    }
  }
  long long sums[2] = {tokens, freed}, totals[2];
  block_scan(sums, s_warp, totals);
  const long long start = sums[0], total_tokens = totals[0], total_freed = totals[1];
  long long back = sums[1];
  // A release that the ring has no room for is refused with its sequence, which stays
  // as it is; a ring that holds every page has the row's too, and the row is emptied.
  const bool give = ring_ok && avail + total_freed <= p.num_pages;
  const bool keep = !give && !(ring_ok && avail == p.num_pages);
  if (tid == 0 && blockIdx.x == 0 && !give) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteFreePages);
  // what fits the table and the rows of the batch asks for pages
  long long need[1] = {0}, total_need[1], at = start;
  for (int b = b0; b < b1; ++b) {
    const bool stuck = keep && gone(b);
    if (stuck) s_base[b] = held_of(b);
    const long long n = max(p.add[b], 0), base = s_base[b];
    const int have = (int)((base + page - 1) >> p.page_shift);
    const bool fits = !stuck && base + n <= cap && at + n <= p.T;
    if (!fits && !stuck) record_device_error(PU_ERR_INVALID_ARGUMENT, kSitePagePlan);
    s_start[b] = (int)min(at, p.T);
    s_last[b] = fits ? (int)((base + n + page - 1) >> p.page_shift) : -1;
    need[0] += fits ? s_last[b] - have : 0;
    at += n;
  }
  block_scan(need, s_warp, total_need);
  long long upto = need[0];
  // Pages go to the sequences in order while they last: behind the first for which
  // they do not, only those that need none are served, so what is taken in all is the
  // furthest place that a served sequence reaches.
  int used = 0;
  for (int b = b0; b < b1; ++b) {
    const int have = (s_base[b] + page - 1) >> p.page_shift;
    const int want = s_last[b] < 0 ? 0 : s_last[b] - have;
    const bool served = s_last[b] >= 0 && (want == 0 || upto + want <= avail);
    if (s_last[b] >= 0 && !served) record_device_error(PU_ERR_WORKSPACE, kSiteFreePages);
    s_new[b] = served ? (int)min(upto, avail) : -1;        // -1: refused, the sequence stays as it is
    if (!served) s_last[b] = have;
    else if (want > 0) used = (int)upto + want;
    upto += want;
  }
  used = __reduce_max_sync(0xffffffffu, used);
  if (lane == 0 && used > 0) atomicMax(&s_used, used);
  for (int b = b0; b < b1; ++b) {
    const bool whole = s_freed[b] >= 0;
    const int f = whole ? s_freed[b] : -1 - s_freed[b];
    if (!whole) record_device_error(PU_ERR_INVALID_ARGUMENT, kSitePagePlan);
    s_freed[b] = f == 0 || !give ? -1 : whole ? (int)back : -2 - (int)back;
    back += f;
  }
  if (tid == 0) s_start[p.B] = (int)min(total_tokens, p.T);
  __syncthreads();

  // rows: pages kept, pages taken, then none
  const int warps = (int)gridDim.x * (kThreads / 32), wid = (int)blockIdx.x * (kThreads / 32) + (tid >> 5);
  auto taken = [&](int i) { int r = head0 + i; return p.ring[r >= p.num_pages ? r - p.num_pages : r]; };
  if constexpr (kInPlace) {
    // only the released rows still need their old lengths: put them where the
    // rows' owners find them before the lengths change
    for (int b = tid; b < p.B; b += kThreads)
      if (gone(b) && !keep) s_base[b] = -held_of(b) - 1;      // base is 0 for a released sequence
    __syncthreads();
    cluster_sync();
  }
  auto base_of = [&](int b) { return kInPlace && s_base[b] < 0 ? 0 : s_base[b]; };
  auto old_of = [&](int b) -> int {      // pages the row returns
    if (!gone(b) || keep) return 0;
    const int held = kInPlace ? -(s_base[b] + 1) : held_of(b);
    return (held + page - 1) >> p.page_shift;
  };
  for (long long u = wid; u < (long long)p.B * segs; u += warps) {
    const int b = (int)(u / segs), lo = (int)(u % segs) * kSeg;
    const int have = (base_of(b) + page - 1) >> p.page_shift, last = s_last[b], old = old_of(b);
    const int32_t* in = p.table + (size_t)b * p.max_pages;
    int32_t* out = p.table_out + (size_t)b * p.max_pages;
    int to = s_freed[b], hi = min(lo + kSeg, p.max_pages);
    if (to <= -2) {
      // entries that are no pages are left out: one warp takes the row, the others'
      // segments of it too, and closes the gaps
      if (lo > 0) continue;
      hi = p.max_pages;
      int put = tail0 - 2 - to;
      for (int j0 = 0; j0 < old; j0 += 32) {
        const int pg = j0 + lane < old ? in[j0 + lane] : -1;
        const bool good = (unsigned)pg < (unsigned)p.num_pages;
        const unsigned all = __ballot_sync(0xffffffffu, good);
        const int r = put + __popc(all & ((1u << lane) - 1u));
        if (good) p.ring[r >= p.num_pages ? r - p.num_pages : r] = pg;
        put += __popc(all);
      }
      to = -1;
    }
    // in place, the kept entries stay and those past both page counts are not touched
    const int from = kInPlace ? max(lo, have) : lo, end = kInPlace ? min(hi, max(last, old)) : hi;
    for (int j = from + lane; j < end; j += 32) {
      if (j < old && to >= 0) {
        int r = tail0 + to + j;
        p.ring[r >= p.num_pages ? r - p.num_pages : r] = in[j];
      }
      out[j] = j < have ? in[j] : j < last ? taken(s_new[b] + j - have) : -1;
    }
  }
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.B; b += kThreads) {
      p.cu[b] = s_start[b];
      if (b < p.B) p.lens_out[b] = base_of(b) + (s_new[b] >= 0 ? max(p.add[b], 0) : 0);
    }
    if (tid == 0) {
      p.cursor_out[0] = head + s_used;
      p.cursor_out[1] = tail + (give ? total_freed : 0);
    }
  }
  // tokens
  const long long threads = (long long)gridDim.x * kThreads;
  for (long long t = (long long)blockIdx.x * kThreads + tid; t < p.T; t += threads) {
    int seq = -1, pos = 0, slot = -1;
    if (t < s_start[p.B]) {
      int a = 0, z = p.B;                // last b with start_b <= t
      while (z - a > 1) {
        const int m = (a + z) >> 1;
        if (s_start[m] <= t) a = m;
        else z = m;
      }
      const int base = base_of(a), have = (base + page - 1) >> p.page_shift;
      seq = a;
      pos = (int)min((long long)base + (t - s_start[a]), 2147483647ll);
      if (s_new[a] >= 0) {
        const int e = pos >> p.page_shift;
        const int pg = e < have ? p.table[(size_t)a * p.max_pages + e] : taken(s_new[a] + e - have);
        if ((unsigned)pg < (unsigned)p.num_pages) slot = (pg << p.page_shift) | (pos & (page - 1));
        else record_device_error(PU_ERR_INVALID_ARGUMENT, kSitePagePlan);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.seq_ids[t] = seq;
  }
}

}  // namespace plan
}  // namespace pu

extern "C" int pu_page_plan(const int32_t* page_table, int32_t* page_table_out, int64_t max_pages_per_seq,
                            const int32_t* kv_lens, int32_t* kv_lens_out, const int32_t* new_lens,
                            const uint8_t* release, int32_t* free_ring, int64_t num_pages, const int64_t* cursor,
                            int64_t* cursor_out, int64_t page_size, int32_t* slots, int32_t* positions,
                            int32_t* seq_ids, int32_t* cu_new, int64_t B, int64_t num_tokens, void* stream) {
  using namespace pu::plan;
  if (!page_table || !page_table_out || !kv_lens || !kv_lens_out || !new_lens || !free_ring || !cursor || !cursor_out ||
      !cu_new || (num_tokens > 0 && (!slots || !positions || !seq_ids)))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page plan: null pointer");
  if (B <= 0 || B > kMaxB) return pu::set_error(PU_ERR_UNSUPPORTED, "page plan: %lld sequences (1 to %d)", (long long)B, kMaxB);
  if (num_tokens < 0 || num_tokens > 2147483647ll)
    return pu::set_error(PU_ERR_UNSUPPORTED, "page plan: %lld tokens", (long long)num_tokens);
  int shift = 0;
  int rc = pu::paged::check_pool(num_pages, page_size, &shift);
  if (rc) return rc;
  if (max_pages_per_seq <= 0 || max_pages_per_seq > (1ll << 30) / page_size)
    return pu::set_error(PU_ERR_UNSUPPORTED, "page plan: %lld pages per sequence", (long long)max_pages_per_seq);
  Params p{};
  p.table = page_table;
  p.table_out = page_table_out;
  p.lens = kv_lens;
  p.lens_out = kv_lens_out;
  p.add = new_lens;
  p.release = release;
  p.ring = free_ring;
  p.cursor = reinterpret_cast<const long long*>(cursor);
  p.cursor_out = reinterpret_cast<long long*>(cursor_out);
  p.slots = slots;
  p.positions = positions;
  p.seq_ids = seq_ids;
  p.cu = cu_new;
  p.B = (int)B;
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.page_shift = shift;
  p.T = num_tokens;
  const bool table_in = page_table == page_table_out, lens_in = kv_lens == kv_lens_out, cur_in = cursor == cursor_out;
  if (table_in != lens_in || lens_in != cur_in)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page plan: table, lengths and cursor are advanced in place together or not at all");
  // in place the lengths are written while other CTAs still read the counts
  if (lens_in && new_lens < kv_lens + B && kv_lens < new_lens + B)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page plan: new_lens overlaps the lengths that are advanced in place");
  const int smem = (int)(5 * B + 1) * (int)sizeof(int);
  const void* f = table_in ? reinterpret_cast<const void*>(page_plan_kernel<true>)
                           : reinterpret_cast<const void*>(page_plan_kernel<false>);
  rc = pu::set_max_dynamic_smem(f, (5 * kMaxB + 1) * (int)sizeof(int), "page plan shared memory");
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!table_in) {
    // 4096 entries or tokens a CTA: below that its scan is most of its time
    const long long work = B * max_pages_per_seq + num_tokens;
    const long long grid = std::max<long long>(1, std::min<long long>((work + 4095) / 4096, pu::sm_count()));
    return pu::check_cuda(pu::decode::launch_pdl(page_plan_kernel<false>, dim3((unsigned)grid), dim3(kThreads), smem, st, p),
                          "page plan launch");
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return pu::check_cuda(cudaLaunchKernelEx(&cfg, page_plan_kernel<true>, p), "page plan launch");
}
