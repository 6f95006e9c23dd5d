// Counts the copies that a wavefront's rows issue and the copies that it waits for (roost_amd/csrc/row_steps.h), over every
// width, and prints the first cases where a step is used while one of its copies may still be on its way.
#include <cstdio>
#include <vector>

#include "row_steps.h"

// Instructions of one step, in order: a rows (by halves), then b rows.
static unsigned Issued(unsigned at, unsigned a, unsigned b, unsigned sub, unsigned bytes) {
  if (roost::WholeStep(at, bytes)) return (a + b) / 8;
  unsigned issued = 0;
  for (unsigned i = 0; i < (a + b) / 8; ++i) {
    const bool of_a = i < a / 8;
    const unsigned half = of_a ? 8 * i / (a / sub) : 0, s = of_a ? sub : 1;
    bool any = false;
    for (unsigned lane = 0; lane < 64; ++lane) any = any || roost::CopiesPiece(at, half, roost::PieceOfLane(lane), bytes, s);
    issued += any;
  }
  return issued;
}

int main() {
  unsigned long cases = 0, wrong = 0, slack = 0;
  for (unsigned sub : {1u, 2u})
    for (unsigned ranks : {16u, 32u, 64u, 80u})
      for (unsigned b : {8u, 16u, 32u, 64u})
        for (unsigned stages : {2u, 3u, 4u})
          for (unsigned waves : {1u, 4u, 8u})
            for (unsigned bytes = 16; bytes <= 5 * 128 * waves; bytes += 16)
              for (unsigned wave = 0; wave < waves; ++wave) {
                const unsigned a = ranks * sub, copies = (a + b) / 8, first = 128 * wave, stride = 128 * waves;
                const unsigned steps = roost::StepsOf(first, stride, bytes);
                const unsigned counted = roost::StepsByCount(first, stride, bytes);
                std::vector<unsigned> out;  // outstanding instructions by their step, oldest first
                unsigned sent = 0, landed = 0;
                const auto send = [&] {
                  for (unsigned k = Issued(first + sent * stride, a, b, sub, bytes); k > 0; --k) out.push_back(sent);
                  ++sent;
                };
                while (sent < stages && sent < steps) send();
                for (unsigned i = 0; i < steps; ++i) {
                  const bool by_count = i + stages <= counted;
                  const unsigned left = by_count ? (stages - 1) * copies : 0;
                  while (out.size() - landed > left) ++landed;  // the wait
                  bool ready = true;
                  for (unsigned k = landed; k < out.size(); ++k) ready = ready && out[k] != i;
                  ++cases;
                  // A wait for everything where all the steps that are out are whole would be one too many.
                  slack += !by_count && i + stages <= steps && roost::WholeStep(first + (i + stages - 1) * stride, bytes);
                  if (!ready && wrong++ < 8)
                    std::printf("used too early: sub %u, %u + %u rows, %u stages, wave %u of %u, %u bytes, step %u of %u\n",
                                sub, a, b, stages, wave, waves, bytes, i, steps);
                  if (sent < steps) send();
                }
              }
  std::printf("%lu steps, %lu used too early, %lu waits too many\n", cases, wrong, slack);
  return wrong != 0 || slack != 0;
}
