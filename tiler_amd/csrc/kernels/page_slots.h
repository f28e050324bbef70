// What the planner hands the page table kernel by value (the host packs the same
// struct).
#pragma once

#include <stdint.h>

struct TilerPageSlots {
  uint64_t sequences, tokens, free_count, width;
  uint32_t page, reserved;
};
