// attn_forms.hip -- the kernels of attn_rows.hip for the other forms of
// attention: to keys of another length that every row sees, and over a prefix
// that sequences share, where a row tile holds rows of several.
#include "attn_rows.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

template <class T, int VW, int NB, int SHARE, bool ALIGNED>
__global__ __launch_bounds__(rows_threads(SHARE), rows_waves<T>(SHARE, VW * NB)) void
k_attn_forms(const AttnArgs a) {
  attn_rows_block<T, VW, NB, SHARE, ALIGNED, ATTN_FORMS>(a);
}

template <class T, int VW, int NB>
void rows_of(hipStream_t st, const AttnArgs &a, bool aligned, int32_t share, unsigned grid) {
  if (share == 8) {
    if constexpr (16 * VW * NB <= (sizeof(T) == 4 ? 64 : 128)) {
      if (aligned)
        k_attn_forms<T, VW, NB, 8, true><<<grid, 512, 0, st>>>(a);
      else
        k_attn_forms<T, VW, NB, 8, false><<<grid, 512, 0, st>>>(a);
    }
  } else if (share == 4) {
    if (aligned)
      k_attn_forms<T, VW, NB, 4, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_forms<T, VW, NB, 4, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (aligned)
      k_attn_forms<T, VW, NB, 1, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_forms<T, VW, NB, 1, false><<<grid, 256, 0, st>>>(a);
  }
}

}  // namespace

void launch_attn_rows_forms(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t,
                            bool aligned, int32_t share) {
  const int64_t groups = share > 1 ? a.tiles : (a.tiles + 3) / 4;
  const int64_t grid = (int64_t)a.n * a.splits * groups * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  const unsigned g = (unsigned)grid;
  KernelTimer kt(ctx, "attn_forms", (double)a.tokens * a.heads, st);
  if (t == VSK_DTYPE_F32) {
    if (a.d <= 64)
      rows_of<float, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<float, 4, 2>(st, a, aligned, share, g);
    else
      rows_of<float, 4, 4>(st, a, aligned, share, g);
  } else if (t == VSK_DTYPE_F16) {
    if (a.d <= 64)
      rows_of<_Float16, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<_Float16, 8, 1>(st, a, aligned, share, g);
    else
      rows_of<_Float16, 8, 2>(st, a, aligned, share, g);
  } else {
    if (a.d <= 64)
      rows_of<__bf16, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<__bf16, 8, 1>(st, a, aligned, share, g);
    else
      rows_of<__bf16, 8, 2>(st, a, aligned, share, g);
  }
  check_launch("attn_forms");
}

}  // namespace vsk
