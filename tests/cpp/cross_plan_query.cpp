// Answers what cross attention's planner (cross_attention_plan.hpp) decides, one line
// of output per line of input, integers:
//   BATCH HEADS KV_HEADS SEQ_Q SEQ_K D_HEAD CUS  ->
//     FORWARD GROUPS UNITS  BACKWARD Q_SPLITS KV_SPLITS
// FORWARD is "rows", "few_keys", "tiles128" or "tiles256" (rows of a workgroup), GROUPS 0
// where a workgroup takes a unit of rows; BACKWARD is "short_rows", "short_keys" or "tiles".
#include <iostream>

#include "cross_attention_plan.hpp"

int main() {
    int64_t batch, heads, kv, sq, sk, d, cus;
    while (std::cin >> batch >> heads >> kv >> sq >> sk >> d >> cus) {
        const nrs::CrossForwardPlan f = nrs::plan_cross_forward(batch, heads, kv, sq, sk, d, cus);
        const nrs::CrossBackwardPlan b = nrs::plan_cross_backward(batch, heads, kv, sq, sk, d, cus);
        const int64_t units = batch * kv * ((sq * (heads / kv) + f.unit_rows - 1) / f.unit_rows);
        std::cout << (f.few_keys                ? "few_keys"
                      : !f.tiles                ? "rows"
                      : f.unit_rows == 256      ? "tiles256"
                                                : "tiles128")
                  << " " << f.groups << " " << units << " "
                  << (b.short_rows ? "short_rows" : b.short_keys ? "short_keys" : "tiles") << " "
                  << b.q_splits << " " << b.kv_splits << "\n";
    }
}
