// Self-test of the bounded wait that every pipelined kernel of this library uses (mbar_wait in
// ptx.cuh): one warp waits, with a short cycle budget, on an mbarrier that nobody ever arrives
// at.  The wait must give up and return, raise the CTA's abort flag and record its code in the
// status word; a second wait in the same CTA must then return at once.  Nothing faults or
// spins without a limit: no TMA, no tensor memory, no other CTA is involved.
#include "ptx.cuh"
#include "errors.h"
#include "row_pipe.cuh"
#include "../../include/eisen_b200.h"

namespace eisen {
namespace {

__global__ void __launch_bounds__(32) bounded_wait_selftest_kernel(int* status, long long budget, int* report) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (threadIdx.x == 0) {
    const long long t0 = clock64();
    const bool first = mbar_wait(&bar, 0, &abort_flag, status, FAULT_WAIT_SELFTEST, budget);
    const long long t1 = clock64();
    const bool second = mbar_wait(&bar, 0, &abort_flag, status, FAULT_WAIT_FULL, budget);  // abort flag is up: at once
    const long long t2 = clock64();
    if (report) {
      report[0] = first ? 1 : 0;
      report[1] = second ? 1 : 0;
      report[2] = abort_flag;
      report[3] = (t1 - t0) > budget ? 1 : 0;          // the first wait used its whole budget
      report[4] = (t2 - t1) < (t1 - t0) / 4 ? 1 : 0;   // the second one did not wait again
    }
  }
}

// The row kernels' frame (row_pipe.cuh) when a wait runs out: two groups of one warp take rows in turn, the first one is through
// its rows and gone, the second waits, with a short budget, for a row that the loading warp never sends for, and then goes on as a
// group does.  All rows must be marked in the end, those of the first group too.
__global__ void __launch_bounds__(96) row_frame_selftest_kernel(float* out, int rows, long long budget, int* fault_word) {
  __shared__ RowRing ring;
  const int g = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ring_init(ring, 2, 1);
  __syncthreads();
  if (g < 2) {
    for (int i = g; i < rows; i += 2) {
      if (g == 1) ring_wait_row(ring, i, 1, 0, budget);
      if (lane == 0) out[i] = 1.0f;
      __syncwarp();
    }
  }
  if (ring_gave_up(ring, 1, fault_word))
    for (int i = threadIdx.x; i < rows; i += blockDim.x) out[i] = NAN;
}

}  // namespace
}  // namespace eisen

extern "C" int eisen_selftest_row_frame(void* stream, float* out, int rows, long long budget_cycles) {
  if (!out || rows < 1 || rows > 4096) return eisen::fail(EISEN_ERR_INVALID, "selftest_row_frame: out is null, or rows not in [1, 4096]");
  if (budget_cycles < 1000 || budget_cycles > 200000000ll)
    return eisen::fail(EISEN_ERR_INVALID, "selftest_row_frame: budget must be between 1e3 and 2e8 cycles");
  eisen::row_frame_selftest_kernel<<<1, 96, 0, (cudaStream_t)stream>>>(out, rows, budget_cycles, eisen::fault_word());
  return eisen::check_launch("selftest_row_frame");
}

extern "C" int eisen_selftest_bounded_wait(void* stream, int* status, long long budget_cycles, int* report5) {
  if (!status) return eisen::fail(EISEN_ERR_INVALID, "selftest_bounded_wait: status is null");
  if (budget_cycles < 1000 || budget_cycles > 200000000ll)
    return eisen::fail(EISEN_ERR_INVALID, "selftest_bounded_wait: budget must be between 1e3 and 2e8 cycles");
  eisen::bounded_wait_selftest_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(status, budget_cycles, report5);
  return eisen::check_launch("selftest_bounded_wait");
}
