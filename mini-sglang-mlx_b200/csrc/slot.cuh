// Pool slots as the stores and the device-built tables write them.
#pragma once

namespace b2a {

// A slot of -1: this row has none (padding of a captured step), the stores skip it. Any other slot
// outside the pool is an error (kWdBadSlot).
constexpr int kNoSlot = -1;

}  // namespace b2a
