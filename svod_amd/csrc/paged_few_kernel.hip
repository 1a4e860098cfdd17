// Attention over a key/value cache in pages where sequences have few query rows a KV head on average, 16 or 32: tiles of as many rows
// (paged_few.h), on places that a compute unit has for one to three workgroups.  The host knows the mean alone, so a long chunk among
// many single tokens comes here too, as many tiles: it is right so, and slow (one of 449 beside 63 tokens over 4096 keys, 32 query heads
// over 8 of 128: 289 us here, 209 in tiles of 128 rows).
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

// The parameters as a turn reads them: from the launch's arguments, and not known to be what the turn before had.  (What a
// loop of turns keeps of them in registers is more than there are: 16-bit pools at D 128 spilled, and 128 sequences of 300 to 3000 keys, 8
// KV heads, took 185 us where it is 169.)
struct Arguments {
  uint64_t deal_lens, deal_starts;
  uint32_t deal_batch, deal_wide, deal_limit, deal_rows, deal_tokens, deal_tokens_rcp, deal_window_blocks, deal_kv_heads, deal_kvh_rcp;
  PagedParams p;
  __device__ Deal deal() const { return SVODK_DEAL; }
};
__device__ __forceinline__ Arguments arguments_of_turn() {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef const __attribute__((address_space(4))) Arguments *At;
  At at = (At)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *at;
#else
  return Arguments{};
#endif
}

template <int D, int RT, bool F16, bool CODED, bool SHARES>
__global__ __launch_bounds__(few::kWaves * 64, (few::Few<D, RT>::kResident)) void paged_few_kernel(SVODK_DEAL_PARAMS, PagedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const Deal deal = SVODK_DEAL;
  if constexpr (SHARES) {
    // What a wave carries from turn to turn lies behind its workgroup's LDS.
    auto kept_at = [&]() { return reinterpret_cast<volatile int *>(smem + few::Few<D, RT>::kLds + 16 + 16 * uniform((int)__builtin_amdgcn_workitem_id_x() >> 6)); };
    Turn turn = turn_of<true>(deal, p);
    kept_at()[1] = turn.parts.most, kept_at()[2] = turn.parts.run;
    do {
      const Arguments here = arguments_of_turn();
      const Work work = work_of<true, false>(here.deal(), here.p, turn);
      if (!work.at.found) return;
      kept_at()[0] = turn.at + work.taken < turn.to() ? turn.at + work.taken : -1;
      if (work.some) few::item<D, RT, F16, CODED, true>(smem, here.deal(), here.p, work);
      __syncthreads();  // the states have been read
      volatile int *const kept = kept_at();
      turn.at = uniform(kept[0]), turn.parts.most = uniform(kept[1]), turn.parts.run = uniform(kept[2]);
      const Deal again = arguments_of_turn().deal();
      turn.whose(again);
      turn.first = demand_of(again, lane_of_turn());
    } while (turn.at >= 0);
  } else {
    const Work work = work_of<false, false>(deal, p, turn_of<false>(deal, p));
    if (work.some) few::item<D, RT, F16, CODED, true>(smem, deal, p, work);
  }
#endif
}

template <int D, int RT, bool F16, bool CODED>
hipError_t launch(const PagedLaunch &l, hipStream_t stream) {
  constexpr int kLds = few::Few<D, RT>::kLds + 16 * (1 + few::kWaves);
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
