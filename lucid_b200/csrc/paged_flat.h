// Which 16-byte pieces of a flat run each lane copies (paged_decode.cu, MODE kFlat): the
// run is 16 rows of D bf16, 32 D bytes, D an odd multiple of 4.  Plain C++, so that a host
// program can walk every head dimension.
#pragma once

namespace lb {

// key chunks per lane of the kernel that takes head dimension D, and the D it takes
constexpr int flat_chunks(int D) { return D < 64 ? 4 : D < 80 ? 5 : 8; }
constexpr int flat_least_d(int nk) { return nk == 4 ? 4 : nk == 5 ? 68 : 84; }
constexpr int flat_most_d(int nk) { return nk == 4 ? 60 : nk == 5 ? 76 : 124; }

// copies per lane, each of 512 bytes in a warp
constexpr int flat_copies(int nk) { return (flat_most_d(nk) + 15) / 16; }

// whether the lane's copy u lies in the run; the first ones do for every D of the kernel,
// which the compiler sees
constexpr bool flat_copied(int nk, int D, int u, int lane) {
  return 512 * (u + 1) <= 32 * flat_least_d(nk) || 16 * (32 * u + lane) < 32 * D;
}

}  // namespace lb
