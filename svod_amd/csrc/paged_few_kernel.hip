// Attention over a key/value cache in pages where every sequence has few query rows a KV head: tiles of 16 or 32 rows
// (paged_few.h), on places that a compute unit has for one to three workgroups.
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "launch.h"

#if !defined(__HIP_DEVICE_COMPILE__)  // the kernels' bodies are compiled for the device only: their helpers have no caller here
#pragma clang diagnostic ignored "-Wunused-function"
#pragma clang diagnostic ignored "-Wunused-const-variable"
#pragma clang diagnostic ignored "-Wunneeded-internal-declaration"
#endif
#include "paged_few.h"

namespace svodk {
namespace {

template <int D, int RT, bool F16, bool CODED, bool SHARES>
__global__ __launch_bounds__(few::kWaves * 64, (few::Few<D, RT>::kResident)) void paged_few_kernel(SVODK_DEAL_PARAMS, PagedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const Deal deal = SVODK_DEAL;
  Turn turn = turn_of<SHARES>(deal, p);
  do {
    const Work work = work_of<SHARES, false>(deal, p, turn);
    if (!work.at.found) return;
    if (work.some) few::item<D, RT, F16, CODED, true>(smem, deal, p, work);
    if (SHARES) __syncthreads();  // the states have been read
    turn.at += work.taken;
    if (SHARES) turn.first = demand_of(deal, lane_of_turn());  // asked for again: held in registers it would cost the loop five
  } while (SHARES && turn.at < turn.to);
#endif
}

template <int D, int RT, bool F16, bool CODED>
hipError_t launch(const PagedLaunch &l, hipStream_t stream) {
  constexpr int kLds = few::Few<D, RT>::kLds + 16;
  if (l.p.shares)
    return Launch<paged_few_kernel<D, RT, F16, CODED, true>>::run(l.grid, few::kWaves * 64, kLds, kLds, stream, SVODK_DEAL_ARGS(l.deal), l.p);
  return Launch<paged_few_kernel<D, RT, F16, CODED, false>>::run(l.grid, few::kWaves * 64, kLds, kLds, stream, SVODK_DEAL_ARGS(l.deal), l.p);
}
template <int D, int RT>
hipError_t launch_rows(const PagedArgs &a, const PagedLaunch &l, hipStream_t stream) {
  const bool coded = a.pages.k_scale != nullptr;
  if (a.pages.f16) return coded ? launch<D, RT, true, true>(l, stream) : launch<D, RT, true, false>(l, stream);
  return coded ? launch<D, RT, false, true>(l, stream) : launch<D, RT, false, false>(l, stream);
}

}  // namespace

hipError_t launch_paged_few(const PagedArgs &a, const PagedLaunch &l, hipStream_t stream) {
  const bool two = paged_tile_rows(a) == 32;
  switch (a.pages.d) {
    case 64: return two ? launch_rows<64, 2>(a, l, stream) : launch_rows<64, 1>(a, l, stream);
    case 128: return two ? launch_rows<128, 2>(a, l, stream) : launch_rows<128, 1>(a, l, stream);
    case 256: return launch_rows<256, 1>(a, l, stream);
    default: return hipErrorInvalidValue;
  }
}

int paged_few_resident(int d, int rows) {
  if (d == 256) return few::Few<256, 1>::kResident;
  if (d == 128) return rows == 32 ? few::Few<128, 2>::kResident : few::Few<128, 1>::kResident;
  return rows == 32 ? few::Few<64, 2>::kResident : few::Few<64, 1>::kResident;
}

}  // namespace svodk
