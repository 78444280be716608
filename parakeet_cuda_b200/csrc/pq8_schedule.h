// Control flow of the scheduler warp and of the MMA issuer of the 8-bit product
// (pq8_i8.cuh). Plain C++ with the waits and the products as callables, so that a
// test on the CPU can run both warps' steps with waits that fail.
//
// The two warps meet on a named barrier that has no time limit, once per `step` K
// blocks of a tile; the meeting ORs a flag to stop. Both have to meet the same
// number of times whatever fails: a failed wait is therefore carried to the next
// meeting, never acted on before it, and after a meeting with the flag raised
// both leave.
#pragma once

#ifdef __CUDACC__
#define PQ8_SCHEDULE_FN __host__ __device__ __forceinline__
#else
#define PQ8_SCHEDULE_FN inline
#endif

namespace pq8 {

// A CTA's work: tiles first, first + stride, ... below end, K blocks [kb0, kb1) of each.
struct ScheduleRange {
  int first, end, stride, kb0, kb1;
};

// The scheduler. acc_free(i): the accumulator of this CTA's i-th tile may be
// overwritten; landed(n, ok): whether `ok` and the next n K blocks are in shared
// memory; both return false when their wait gave up, landed with one answer for the
// whole warp. meet(flag): the meeting, returns the OR of both flags.
template <typename AccFree, typename Landed, typename Meet>
PQ8_SCHEDULE_FN void schedule_products(const ScheduleRange& r, int step, AccFree&& acc_free, Landed&& landed,
                                       Meet&& meet) {
  int i = 0;
  for (int tile = r.first; tile < r.end; tile += r.stride, ++i) {
    bool ok = acc_free(i);
    for (int kb = r.kb0; kb < r.kb1; kb += step) {
      ok = landed(r.kb1 - kb < step ? r.kb1 - kb : step, ok);
      if (meet(!ok)) return;
    }
  }
}

// The MMA issuer. issue(i, kb, n): the products of K blocks [kb, kb + n) of the i-th
// tile. Returns whether it was told to stop.
template <typename Meet, typename Issue>
PQ8_SCHEDULE_FN bool issue_products(const ScheduleRange& r, int step, Meet&& meet, Issue&& issue) {
  int i = 0;
  for (int tile = r.first; tile < r.end; tile += r.stride, ++i)
    for (int kb = r.kb0; kb < r.kb1; kb += step) {
      if (meet(false)) return true;
      issue(i, kb, r.kb1 - kb < step ? r.kb1 - kb : step);
    }
  return false;
}

}  // namespace pq8
