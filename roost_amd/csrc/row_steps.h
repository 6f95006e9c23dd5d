// Which copies a wavefront's rows make on their way through LDS, and how far it may count on them: plain arithmetic, so that
// a program on the host can hold it against every width.
//
// Rows of `bytes` bytes go by steps of 128, of which a wavefront takes the steps at first, first + stride, ... A copy
// instruction brings eight rows' 128 bytes; rows whose steps are `sub` times as long take `sub` copies for each, one after
// another (`half`). Lanes whose 16 bytes lie past the row's end copy nothing, and an instruction with no lane left is branched
// over: it is not issued, and no counter of outstanding copies ever sees it.

#pragma once

#include <cstdint>

namespace roost {

constexpr uint32_t kStepBytes = 128;

constexpr uint32_t StepsOf(uint32_t first, uint32_t stride, uint32_t bytes) {
  return first < bytes ? (bytes - first + stride - 1) / stride : 0;
}

// Whether every lane copies in every instruction of the step at `at`.
constexpr bool WholeStep(uint32_t at, uint32_t bytes) { return at + kStepBytes <= bytes; }

// A lane's piece of its row's 128 bytes.
constexpr uint32_t PieceOfLane(uint32_t lane) { return 16 * ((lane % 8) ^ (lane / 8)); }

// Whether a lane with `piece` copies in an instruction for the half-th 128 bytes of a step of rows `sub` times as long.
constexpr bool CopiesPiece(uint32_t at, uint32_t half, uint32_t piece, uint32_t bytes, uint32_t sub) {
  return at * sub + half * kStepBytes + piece < bytes * sub;
}

// With the copies of steps i .. i + stages - 1 out (fewer at the end), step i may be awaited by leaving the copies of
// stages - 1 steps outstanding while i + stages is at most this: every step among them is a whole one and has issued all its
// copies. The last step of a row may issue fewer (rows of 8 bits beside an adapter's of 16, `sub` 2, where it holds 64 bytes
// or less), so what it leaves outstanding says nothing about the steps before it.
constexpr uint32_t StepsByCount(uint32_t first, uint32_t stride, uint32_t bytes) {
  return WholeStep(first, bytes) ? (bytes - kStepBytes - first) / stride + 1 : 0;
}

}  // namespace roost
