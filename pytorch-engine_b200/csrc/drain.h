// What a stage's barrier is still owed when two thread blocks that fill it together have given up (gemm_fp8_pair.cu).  Plain C++,
// so that it can be tried without a GPU.
#pragma once

#ifdef __CUDACC__
#define PE_BOTH __host__ __device__ __forceinline__
#else
#define PE_BOTH inline
#endif

namespace pe {

// The barrier's phase for stage `i` completes with two arrivals (the first block's producer, which announces the bytes of both blocks,
// and whoever hands the scales over) and with all bytes that were announced.  `mine` and `theirs`: stages for which the first and
// the second block started their copies (`bytes` each); `fed`: stages whose scales were handed over.  To be done in this order:
struct Owed {
  unsigned expect;      // bytes to announce: copies on their way that nobody announced
  unsigned complete;    // bytes to count as arrived: announced copies that were never started
  int arrivals;
};
PE_BOTH Owed owed_to_stage(int i, int mine, int theirs, int fed, unsigned bytes) {
  Owed o;
  o.expect = i >= mine && i < theirs ? bytes : 0u;
  o.complete = i < mine && i >= theirs ? bytes : 0u;
  o.arrivals = (i < mine ? 0 : 1) + (i < fed ? 0 : 1);
  return o;
}

}  // namespace pe
