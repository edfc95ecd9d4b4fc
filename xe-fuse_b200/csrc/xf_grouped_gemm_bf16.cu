// Kernel instances of the grouped product with bf16 operands.
#include "xf_grouped_gemm_kernel.cuh"

namespace xf {
namespace grouped {

const Variant g_variants_bf16[kTilesBf16] = {
    XF_GROUPED_VARIANT(KIND_BF16, 256, 2, "bf16_256x256_cta2"),
    XF_GROUPED_VARIANT(KIND_BF16, 128, 1, "bf16_128x128_cta1"),
};

}  // namespace grouped
}  // namespace xf
