// Kernel instances of the grouped product with e4m3 operands.
#include "xf_grouped_gemm_kernel.cuh"

namespace xf {
namespace grouped {

const Variant g_variants_e4m3[kTilesE4m3] = {
    XF_GROUPED_VARIANT(KIND_E4M3, 256, 2, "e4m3_256x256_cta2"),
    XF_GROUPED_VARIANT(KIND_E4M3, 256, 1, "e4m3_128x256_cta1"),
    XF_GROUPED_VARIANT(KIND_E4M3, 128, 1, "e4m3_128x128_cta1"),
};

}  // namespace grouped
}  // namespace xf
