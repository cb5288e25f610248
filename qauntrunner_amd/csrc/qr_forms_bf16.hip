// qr_forms_bf16.hip -- attention in its other forms on MFMA tiles: caches of QR_DTYPE_BF16.
#include "qr_forms_mfma.hpp"

namespace qr {

hipError_t launch_forms_bf16(const FormsK& k, int units, hipStream_t s) { return form_launch_type<QR_DTYPE_BF16>(k, units, s); }

}  // namespace qr
