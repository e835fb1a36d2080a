// The kernels of w4_rows.cuh for fp16 rows, a file of their own for the sake of building in parallel.
#include "w4_rows.cuh"

namespace tb200
{
namespace ffn
{

RowsKern w4_rows_kernel_f16(int nt, int mats, bool flat)
{
    return mats == 2 ? (flat ? pick<false, 2, true>(nt) : pick<false, 2, false>(nt)) : (flat ? pick<false, 1, true>(nt) : pick<false, 1, false>(nt));
}

}    // namespace ffn
}    // namespace tb200
