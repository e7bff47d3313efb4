// What the calls of a layer of experts share.
#pragma once
#include "kv.h"

namespace lapis_b200 {

constexpr int MAX_EXPERTS = 1024, MAX_CHOSEN = 32;

int check_expert_lists(const char *what, const lapis_b200_expert_lists *lists);  // experts.cu; 0 or a recorded error

}  // namespace lapis_b200
