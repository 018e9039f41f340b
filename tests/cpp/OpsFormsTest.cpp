// Every type and stride that the C entries of the norm and the token sort take is reachable from their
// C++ forms; host only: empty inputs, and refusals that reach no device.
#include <cstdint>
#include <cstring>

#include "Expect.hpp"
#include "litemind_b200/Gemm.hpp"
#include "litemind_b200/TokenSort.hpp"

namespace {
bool says(const char* text) { return std::strstr(lm_moe_last_error(nullptr), text) != nullptr; }
template <class T>
T* at(std::uintptr_t place) { return reinterpret_cast<T*>(place << 32); }  // an address that nothing reads
}  // namespace

int main() {
    Expect expect("OpsFormsTest");
    using litemind::b200::gemm::add_rms_norm_mx;
    auto* hidden = at<std::uint16_t>(1);
    auto* delta = at<std::uint16_t>(2);
    auto* weight = at<float>(3);
    auto* sum = at<std::uint16_t>(4);
    auto* data = at<std::uint8_t>(5);
    auto* scales = at<std::uint8_t>(6);
    expect(add_rms_norm_mx(hidden, LM_DTYPE_BF16, delta, LM_DTYPE_BF16, weight, 0, 64, 1e-6F, sum, nullptr, LM_MX_E2M1, data, scales) == LM_OK, "no bf16 rows");
    expect(add_rms_norm_mx(hidden, LM_DTYPE_F16, delta, LM_DTYPE_BF16, weight, 4, 64, 1e-6F, sum, nullptr, LM_MX_E4M3, data, scales) == LM_ERR_INVALID_ARGUMENT &&
               says("hidden and delta are f32 or bf16"), "f16 rows");
    expect(add_rms_norm_mx(hidden, LM_DTYPE_BF16, delta, LM_DTYPE_BF16, weight, 4, 64, 1e-6F, delta + 64, nullptr, LM_MX_E4M3, data, scales) == LM_ERR_INVALID_ARGUMENT &&
               says("sum overlaps a part"), "a shifted sum");
    const litemind::b200::SortPlan plan{at<int32_t>(7), at<int32_t>(8), 5, 2, 64};
    expect(plan.sort(hidden, 256, 128, sum, 512, 0) == LM_OK, "no room for rows");
    expect(plan.sort(hidden, 127, 128, sum, 512, 10) == LM_ERR_INVALID_ARGUMENT && says("stride"), "x_stride below the row");
    expect(plan.sort(hidden, 256, 128, sum, 127, 10) == LM_ERR_INVALID_ARGUMENT && says("stride"), "rows_stride below the row");
    expect(plan.sort(hidden, 256, 128, reinterpret_cast<std::uint8_t*>(hidden) + 64, 256, 10) == LM_ERR_INVALID_ARGUMENT && says("overlaps x"), "rows over x");
    expect(plan.unsort_backward_f32(nullptr, hidden, LM_DTYPE_BF16, 10, weight, 64, sum, at<float>(9)) == LM_ERR_INVALID_ARGUMENT &&
               says("lm_moe_unsort_rows_backward_f32: a null"), "no gradient");
    return expect.finish();
}
