// How logprob.cu cuts its work: host arithmetic only.
#pragma once

#include <stdint.h>

namespace tsr {

constexpr int kLpMost = 512;    // threads of a CTA at most
constexpr int kLpPer = 12;      // logits of a thread at a time
constexpr int kLpCluster = 16;  // CTAs of a row at most

// CTAs of a row, a cluster: twice as many while the machine has room for them (two a SM; clusters of sixteen, of which a GPC holds
// few, one a SM) and each has a quarter of a tile.  `resident(ctas)`: how many clusters of that size the device runs at a time, 0 where it
// does not take the size (a partitioned GPU); asked only for sizes that come into question.
template <typename Resident>
inline unsigned logprob_ctas(uint64_t rows, uint64_t vocab, Resident resident) {
  unsigned ctas = 1;
  while (ctas < kLpCluster && rows * (ctas * 2) <= (ctas < 8 ? 296 : 148) && vocab / (ctas * 2) >= kLpMost * kLpPer / 4) ctas *= 2;
  while (ctas > 1 && resident(ctas) == 0) ctas /= 2;
  return ctas;
}

}  // namespace tsr
