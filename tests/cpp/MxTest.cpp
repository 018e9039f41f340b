// The C++ forms of the MX matrices and the token sort (Mx.hpp, TokenSort.hpp, gemm::add_rms_norm_mx),
// host only: row pitches, empty inputs, and refusals that reach no device.
#include <cstdint>

#include "Expect.hpp"
#include "litemind_b200/Gemm.hpp"
#include "litemind_b200/Mx.hpp"
#include "litemind_b200/TokenSort.hpp"

namespace mx = litemind::b200::mx;

int main() {
    Expect expect("MxTest");
    expect(mx::data_pitch(LM_MX_E2M1, 1408) == 704 && mx::data_pitch(LM_MX_E4M3, 129) == 256, "code pitches");
    expect(mx::scale_pitch(2048) == 64 && mx::scale_pitch(1) == 16, "scale pitches");
    auto* p = reinterpret_cast<std::uint8_t*>(std::uintptr_t{1} << 20);  // aligned, never read
    const mx::Matrix x{p, p, 0, 256, LM_MX_E4M3}, w{p, p, 6 * 64, 256, LM_MX_E2M1};
    expect(mx::matmul(x, w, 6, reinterpret_cast<int32_t*>(p), p, LM_DTYPE_BF16, 64) == LM_OK, "no rows: nothing to do");
    expect(mx::matmul(x, w, 5, reinterpret_cast<int32_t*>(p), p, LM_DTYPE_BF16, 64) == LM_ERR_INVALID_ARGUMENT, "rows of w that no group count divides");
    expect(mx::matmul(x, x, 1, nullptr, p, LM_DTYPE_BF16, 64) == LM_ERR_INVALID_ARGUMENT, "8-bit weights");
    mx::Matrix some = x;
    some.rows = 3;
    expect(mx::matmul(some, w, 6, nullptr, p, LM_DTYPE_BF16, 64) == LM_ERR_INVALID_ARGUMENT, "groups without offsets");
    expect(mx::quantize(nullptr, LM_DTYPE_F32, 256, some) == LM_ERR_INVALID_ARGUMENT, "null values");
    expect(mx::dequantize(some, p, LM_DTYPE_F32, 255) == LM_ERR_INVALID_ARGUMENT, "a stride below the columns");
    expect(litemind::b200::gemm::add_rms_norm_mx(nullptr, nullptr, nullptr, 0, 64, 1e-6F, nullptr, nullptr, LM_MX_E4M3, nullptr, nullptr) == LM_OK, "no rows to norm");
    const litemind::b200::SortPlan plan{reinterpret_cast<int32_t*>(p), reinterpret_cast<int32_t*>(p), 0, 6, 64};
    expect(plan.sort(p, 128, p, 0) == LM_OK && plan.unsort(p, LM_DTYPE_BF16, 0, nullptr, 64, p, LM_DTYPE_BF16) == LM_OK, "no tokens");
    litemind::b200::SortPlan wide = plan;
    wide.tokens = 4;
    wide.top_k = LM_SORT_MAX_TOP_K + 1;
    expect(wide.build(reinterpret_cast<int32_t*>(p)) == LM_ERR_INVALID_ARGUMENT, "too many slots");
    expect(wide.unsort_backward(p, p, LM_DTYPE_BF16, 4, reinterpret_cast<float*>(p), 8, p, reinterpret_cast<float*>(p)) == LM_ERR_INVALID_ARGUMENT, "too many slots");
    return expect.finish();
}
