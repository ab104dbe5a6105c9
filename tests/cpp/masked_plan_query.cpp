// Answers what masked attention's planner (masked_attention_plan.hpp) decides, one line
// of output per line of input, integers:
//   BATCH HEADS KV_HEADS SEQ_Q SEQ_K D_HEAD CUS  ->
//     FORWARD SHARED Q_PARTS KV_PARTS FORWARD_BYTES BACKWARD_BYTES
// FORWARD is "rows", "tiles128" or "tiles256" (rows of a workgroup); SHARED is the number
// of workgroups of a shared line of tiles ("rows"; 0: a unit each), or of parts of a walk.
#include <iostream>

#include "masked_attention_plan.hpp"

int main() {
    int64_t batch, heads, kv, sq, sk, d, cus;
    while (std::cin >> batch >> heads >> kv >> sq >> sk >> d >> cus) {
        const auto f = nrs::plan_masked_forward(batch, heads, kv, sq, sk, d, cus);
        const auto b = nrs::plan_masked_backward(batch, heads, kv, sq, sk, d, cus);
        std::cout << (!f.tiles ? "rows" : f.unit_rows == 256 ? "tiles256" : "tiles128") << " "
                  << (f.tiles ? f.walk.parts : f.line.groups) << " " << b.q.parts << " "
                  << b.kv.parts << " " << f.bytes() << " " << b.bytes() << "\n";
    }
}
