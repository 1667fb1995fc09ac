// When the sets of LDS that a tile's wavefronts stage for one another have arrived: how many of its latest loads a wavefront may
// have in flight at each barrier.
//
// Loads arrive in the order in which they are issued. A workgroup begins with both operands' scales (fd + fs loads), `ahead`
// blocks of D's operands (2 fd each) and sets 0, 1 and 2 (`staged` each). Step J then multiplies the set of its block: it issues
// 2 fd loads of D, has its barrier, behind which the next block's set is read, and issues the set three blocks on. Step 3 has
// the next four blocks' scales beside that, fd of D's before its other loads and one of S's for each fragment, half before the
// barrier and half after it. What a tile's end stores comes behind all of these and only makes a wait longer.
#pragma once

namespace plm {

struct Fp8TileLoads {
  int fd, fs, staged, ahead;
};

// Before the first step. Step 0's wait counts the D operands of two steps, and before a workgroup's first step there was none,
// so with D three blocks ahead (where no operand of the step before has to arrive first) set 1 has to be there already.
constexpr int fp8_first_wait(Fp8TileLoads z) { return z.ahead == 1 ? 2 * z.staged : z.staged; }

// At step J's barrier: behind the next block's set come the set after it and the D operands of this step and, with D three
// blocks ahead, of the one before, which with one block ahead have been multiplied by then.
constexpr int fp8_step_wait(Fp8TileLoads z, int j) {
  return z.staged + 2 * z.fd * (z.ahead == 1 ? 1 : 2) + (j == 3 ? z.fd + z.fs / 2 : 0);
}

}  // namespace plm
