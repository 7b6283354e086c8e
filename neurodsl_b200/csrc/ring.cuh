// ring.cuh — the steps of a ring of tiles, its producer's and its consumers',
// and what each does when a wait runs out.  The waits are arguments, so the same
// steps run on the host, over barriers made of threads.
#pragma once

#ifdef __CUDACC__
#define ND_RING __device__ __forceinline__
#else
#define ND_RING inline
#endif

namespace nd {

// The producer: a tile into stage it % kStages while more(), the stage's last tile
// having been read.
//   read(stage, parity)    waits for that; false when it ran out or another role
//                          has given up
//   fill(stage)            sends the next tile's copies off
//   give_up()              tells the other roles and the host
//   landed(stage, parity)  waits for a tile's copies, whoever has given up
// On every way out the tiles still in flight land first: the consumers may be gone
// by then, and with them the block and the memory that is written.
template <int kStages, typename More, typename Read, typename Fill, typename GiveUp, typename Landed>
ND_RING void ring_produce(More&& more, Read&& read, Fill&& fill, GiveUp&& give_up, Landed&& landed) {
  int it = 0;
  for (; more(); ++it) {
    if (it >= kStages && !read(it % kStages, (it / kStages - 1) & 1)) {
      give_up();
      break;
    }
    fill(it % kStages);
  }
  for (int i = it > kStages ? it - kStages : 0; i < it; ++i) landed(i % kStages, i / kStages & 1);
}

// A consumer: whether tile `it` is there.  The first that does not come is
// reported, and from then on (`ok`) nothing is waited for; the caller neither uses
// nor releases a stage without its tile.
template <int kStages, typename Wait, typename GiveUp>
ND_RING bool ring_take(bool& ok, int it, Wait&& wait, GiveUp&& give_up) {
  if (ok && !wait(it % kStages, it / kStages & 1)) {
    ok = false;
    give_up();
  }
  return ok;
}

}  // namespace nd
