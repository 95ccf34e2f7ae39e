// Page tables, slots and positions of a step, built on the GPU from the rows' lengths.
//
// Row r holds ceil(before / P) pages and needs ceil(after / P) for the step.  Growing rows take pages from the head
// of a ring of free pages, in row order; shrinking rows (a finished request, taken-back tokens) put theirs at its
// tail.  A row whose pages, with those of the rows before it, exceed the free ones keeps what it has and takes no
// part in the step: its count is 0 and its length stays.  Pages given back serve from the next call on.
//
// Every result is a function of the inputs and of table entries and ring places the call does not write, so calling
// it again with the same inputs gives the same results; the ring's head and tail are returned, not updated.
//
// A block takes one row and scans the demands of all (three numbers each) by itself, so no block waits for another.
// What bounds it: latency, three dependent reads (lengths; the ring or the table; nothing waits for the stores) and two
// barriers: 64 rows of one token 3.7 us, 256 rows of up to 512 tokens (2.1 MB of positions and slots) 4.9 us.
#include "kv4_device.h"
#include "launch.h"

namespace xattn {

constexpr int kReserveThreads = 256;

struct RowPages {
  int held, need, count, start, length;  // length: after the step; start: of its first new token
  bool fits;
  __device__ __forceinline__ int grow() const { return fits ? max(need - held, 0) : 0; }
  __device__ __forceinline__ int back() const { return fits ? max(held - need, 0) : 0; }
};
__device__ __forceinline__ RowPages row_pages(const ReserveArgs &a, int r) {
  const int capacity = a.width << a.page_shift, mask = (1 << a.page_shift) - 1;
  RowPages p;
  p.count = min(max(a.counts[r], 0), a.T);
  p.length = max(a.after[r], p.count);
  p.fits = p.length <= capacity;
  p.start = p.length - p.count;
  const int before = min(max(a.before[r], 0), capacity);
  p.held = (before >> a.page_shift) + ((before & mask) != 0);
  p.need = (p.length >> a.page_shift) + ((p.length & mask) != 0);
  if (!p.fits) p.length = before;
  return p;
}

__global__ void __launch_bounds__(kReserveThreads) reserve_kernel(const ReserveArgs a) {
  constexpr int WAVES = kReserveThreads / 64;
  __shared__ int wave_sum[WAVES], mine_before, sums[3][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mine = blockIdx.x;
  const int64_t head = scalar_load(a.counters, 0), tail = scalar_load(a.counters, 1);
  const int per = (a.B + kReserveThreads - 1) / kReserveThreads, first = min(tid * per, a.B), last = min(first + per, a.B);
  int demand = 0;
  for (int r = first; r < last; ++r) demand += row_pages(a, r).grow();
  const int scan = wave_scan(demand);
  if (lane == 63) wave_sum[wave] = scan;
  __syncthreads();
  int running = scan - demand;
  for (int w = 0; w < wave; ++w) running += wave_sum[w];
  // Pages taken by all granted rows, given back by those before `mine`, and by all.
  const int64_t available = min(max(tail - head, (int64_t)0), a.ring_size);
  int taken = 0, back_before = 0, back_all = 0;
  for (int r = first; r < last; ++r) {
    const RowPages p = row_pages(a, r);
    const int grow = p.grow();
    if (r == mine) mine_before = running;
    running += grow;
    if (grow > 0 && running <= available) taken += grow;
    back_all += p.back();
    if (r < mine) back_before += p.back();
  }
  const int t0 = wave_total(taken), t1 = wave_total(back_before), t2 = wave_total(back_all);
  if (lane == 0) sums[0][wave] = t0, sums[1][wave] = t1, sums[2][wave] = t2;
  __syncthreads();
  int given_before = 0, total_taken = 0, total_back = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total_taken += sums[0][w], given_before += sums[1][w], total_back += sums[2][w];
  if (mine == 0 && tid == 0) {
    a.new_counters[0] = head + total_taken;
    a.new_counters[1] = tail + total_back;
  }
  if (mine >= a.B) return;

  RowPages p = row_pages(a, mine);
  const int grow = p.grow();
  const bool granted = p.fits && (grow == 0 || (int64_t)mine_before + grow <= available);
  if (!granted) {
    const int capacity = a.width << a.page_shift;
    p.count = 0;
    p.length = min(max(a.before[mine], 0), capacity);
  }
  if (tid == 0) {
    a.lengths[mine] = p.count;
    a.lengths[a.B + mine] = p.length;
  }
  int32_t *const row = a.table + (int64_t)mine * a.width;
  const uint32_t size = (uint32_t)a.ring_size;
  // Places of the row's first new page and first page given back.
  auto place = [&](int64_t counter, int offset) {
    const uint64_t c = (uint64_t)counter;
    return (uint32_t)(((c % size) + (uint32_t)offset) % size);
  };
  if (granted && grow > 0) {
    const uint32_t from = place(head, mine_before);
    for (int i = p.held + tid; i < p.need; i += kReserveThreads) {
      const uint32_t at = from + (uint32_t)(i - p.held);
      row[i] = a.ring[at >= size ? at - size : at];
    }
  }
  if (granted && p.held > p.need) {
    const uint32_t to = place(tail, given_before);
    for (int i = p.need + tid; i < p.held; i += kReserveThreads) {
      const uint32_t at = to + (uint32_t)(i - p.need);
      a.ring[(at >= size ? at - size : at) % size] = row[i];
    }
  }
  const uint32_t from = grow > 0 ? place(head, mine_before) : 0;
  for (int t = tid; t < a.T; t += kReserveThreads) {
    int64_t position = 0, slot = -1;
    if (t < p.count) {
      position = p.start + t;
      const int i = (int)position >> a.page_shift;
      int page;
      if (i >= p.held) {
        const uint32_t at = from + (uint32_t)(i - p.held);
        page = a.ring[at >= size ? at - size : at];
      } else {
        page = row[i];
      }
      if (page >= 0) slot = ((int64_t)page << a.page_shift) + ((int)position & ((1 << a.page_shift) - 1));
    }
    a.positions[(int64_t)mine * a.T + t] = position;
    a.slots[(int64_t)mine * a.T + t] = slot;
  }
}

hipError_t launch_reserve(const ReserveArgs &a, hipStream_t stream) {
  // Without rows one block returns the counters.
  hipLaunchKernelGGL(reserve_kernel, dim3(a.B > 0 ? a.B : 1), dim3(kReserveThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace xattn
