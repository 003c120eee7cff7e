// The finder of prompt attention's tiles, run by a warp on the host.
#include "warp_host.h"

#include <cstring>

#include "prompt_tiles.cuh"

using namespace mtpb;

namespace {
PaParams params(const int* starts, int S, int first, int n, int total, int hq, int hkv, int rows, long long* items) {
  PaParams p;
  std::memset(&p, 0, sizeof(p));
  p.starts = starts;
  p.S = S;
  p.first = first;
  p.n = n;
  p.total = total;
  p.hq = hq;
  p.hkv = hkv;
  *items = pa_items(&p, rows);
  return p;
}
}  // namespace

extern "C" {

// Tiles of `rows` rows by growing `numbers`: out[i] = {start, tok0, ntok}, the tokens a tile, the items that a call
// plans, and the gaps' ends as they stand after the last number. 0, or 1 when the lanes do not agree.
int pt_find(const int* starts, int S, int first, int n, int total, int hq, int hkv, int rows, const int* numbers, int count,
            int* out, int* tt, long long* items, int* gaps) {
  const PaParams p = params(starts, S, first, n, total, hq, hkv, rows, items);
  *tt = p.tt;
  int apart = 0;
  warp_host::run([&](int lane) {
    alignas(PaTiles) unsigned char memory[sizeof(PaTiles)];
    std::memset(memory, 0xA5, sizeof(memory));  // what registers may hold
    PaTiles& t = *reinterpret_cast<PaTiles*>(memory);
    t.open(p);
    for (int i = 0; i < count; ++i) {
      const PaItem it = t.find(p, numbers[i]);
      const int got[3] = {it.start, it.tok0, it.ntok};
      if (lane == 0) std::memcpy(out + 3 * i, got, sizeof(got));
      apart |= std::memcmp(out + 3 * i, got, sizeof(got)) != 0;
    }
    if (lane == 0) gaps[0] = t.gap0, gaps[1] = t.gap1;
    apart |= gaps[0] != t.gap0 || gaps[1] != t.gap1;
  });
  return apart;
}

// The same with a finder of its own for every number, as a CTA with one tile has it.
int pt_only(const int* starts, int S, int first, int n, int total, int hq, int hkv, int rows, const int* numbers, int count,
            int* out, int* tt, long long* items, int* gaps) {
  const PaParams p = params(starts, S, first, n, total, hq, hkv, rows, items);
  *tt = p.tt;
  int apart = 0;
  for (int i = 0; i < count; ++i)
    warp_host::run([&](int lane) {
      alignas(PaTiles) unsigned char memory[sizeof(PaTiles)];
      std::memset(memory, 0xA5, sizeof(memory));
      PaTiles& t = *reinterpret_cast<PaTiles*>(memory);
      const PaItem it = t.only(p, numbers[i]);
      const int got[3] = {it.start, it.tok0, it.ntok};
      if (lane == 0) {
        std::memcpy(out + 3 * i, got, sizeof(got));
        gaps[0] = t.gap0, gaps[1] = t.gap1;
      }
      apart |= std::memcmp(out + 3 * i, got, sizeof(got)) != 0 || gaps[0] != t.gap0 || gaps[1] != t.gap1;
    });
  return apart;
}
}
