// qr_forms_e4m3.hip -- attention in its other forms on MFMA tiles: caches of QR_DTYPE_E4M3.
#include "qr_forms_mfma.hpp"

namespace qr {

hipError_t launch_forms_e4m3(const FormsK& k, int units, hipStream_t s) { return form_launch_type<QR_DTYPE_E4M3>(k, units, s); }

}  // namespace qr
