// Where a lane's 16 bytes of a row lie that go into LDS with a step of 128 bytes: plain arithmetic, so that
// the host can check it for every size.
#pragma once

namespace mi::adapter {

// Of a row of `width` bytes (a multiple of 16) the lane's chunk (0, 16, .. 112) of the step at `off`: its place where
// the row has it, else the row's first 16 bytes, which are readable in a row of any width (what comes from
// there meets zeros). Rows may be shorter than a step.
constexpr int ring_place(int off, int chunk, int width) { return off + chunk < width ? off + chunk : 0; }

}  // namespace mi::adapter
