// The launch of the gated delta rule token by token.
#include "delta_step.hpp"

namespace anna {

template <int DT, int DK, int COLS>
__global__ __launch_bounds__(256) void delta_step_kernel(const anna_mi_gated_delta_args a, const SpanSeq* __restrict__ steps, int slices) {
  __shared__ StepLds<DK, COLS> lds;
  delta_step_block<DT, DK, COLS>(a, steps, slices, blockIdx.x, lds);
}

int delta_step(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream) {
  // The widest slices that leave a workgroup for every compute unit: rows of 128 columns are whole lines, and
  // fewer workgroups make the unit vectors (heads of 64 x 128, 24 sequences of up to 6 tokens: 19.2 us at 32 columns,
  // 14.8 at 128); for few sequences narrow ones are sooner done (one sequence: 4.9 us, 6.0 at 128).
  const int64_t states = s.steps * a.value_heads;
  int cols = 32;
  for (int wide = 64; wide <= 128; wide *= 2)
    if (a.value_dim % wide == 0 && states * (a.value_dim / wide) >= 256) cols = wide;
  const int slices = (int)(a.value_dim / cols);
  const int64_t grid = states * slices;
  if (grid == 0) return ANNA_MI_OK;
  ANNA_CHECK(grid <= INT32_MAX / 256, "gated delta rule: too many sequences and heads for a launch");
  ANNA_DISPATCH_DTYPE(a.dtype, DT, {
    if constexpr (DT != ANNA_MI_F32) {
      auto go = [&](auto kern) { kern<<<grid, 256, 0, stream>>>(a, span_steps(s), slices); };
      if (a.key_dim == 64) go(cols == 32 ? delta_step_kernel<DT, 64, 32> : cols == 64 ? delta_step_kernel<DT, 64, 64> : delta_step_kernel<DT, 64, 128>);
      else go(cols == 32 ? delta_step_kernel<DT, 128, 32> : cols == 64 ? delta_step_kernel<DT, 128, 64> : delta_step_kernel<DT, 128, 128>);
    }
  });
  ANNA_LAUNCH_CHECK("delta_step");
  return ANNA_MI_OK;
}

}  // namespace anna
