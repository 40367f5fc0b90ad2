// The angle of a rotation by position, for rotary.hip and paged_append.hip.
//
// A pair's frequency is a fraction of a full turn a position, held as a 0.64 fixed-point number, so that position *
// frequency modulo a turn is one 64-bit product whose overflow is the modulo: off by 2^-32 of a turn, which is dropped,
// and by position times 2^-65 of the frequency's rounding, as much again at position 2^33 (a float product loses a bit of
// the angle with every doubling: 2^-4 rad at a million). What is left after the nearest quarter turn is within pi / 4,
// where the Taylor polynomials below are off by less than 2^-29 (sine, to x^9) and 2^-32 (cosine, to x^10); in fp32 both
// come out within two of its steps.
#pragma once

#include "common.h"

MI355_DEVINL void sincos_of_turn(int64_t position, uint64_t frequency, float& sine, float& cosine) {
  const uint32_t u = static_cast<uint32_t>((static_cast<uint64_t>(position) * frequency) >> 32);
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(u - (quarter << 30))) * 1.4629180792671596e-9f;  // pi / 2^31
  const float z = x * x;
  float s = 2.7557319e-6f, c = -2.7557319e-7f;  // 1 / 9!, -1 / 10!
  s = __builtin_fmaf(s, z, -1.9841270e-4f);
  c = __builtin_fmaf(c, z, 2.4801587e-5f);
  s = __builtin_fmaf(s, z, 8.3333333e-3f);
  c = __builtin_fmaf(c, z, -1.3888889e-3f);
  s = __builtin_fmaf(s, z, -1.6666667e-1f);
  c = __builtin_fmaf(c, z, 4.1666667e-2f);
  s = __builtin_fmaf(s * z, x, x);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  sine = quarter & 1 ? c : s;
  cosine = quarter & 1 ? s : c;
  sine = quarter & 2 ? -sine : sine;
  cosine = (quarter + 1) & 2 ? -cosine : cosine;
}
