// kv4_keys.hpp — where kv4_select_kernel has its candidates' keys in LDS (constexpr functions alone: a host compiler
// takes it too).
#pragma once
#include <cstdint>

namespace g4kv4 {

// n candidates, GROUP at a time; of a group, each wave takes as many in a row as the others, 64 * each().
struct Keys {
  static constexpr uint32_t THREADS = 1024, PER = 32, GROUP = PER * THREADS;
  uint32_t n;
  constexpr uint32_t groups() const { return (n + GROUP - 1) / GROUP; }
  constexpr uint32_t rows(uint32_t g) const { return n - g * GROUP < GROUP ? n - g * GROUP : GROUP; }
  constexpr uint32_t each(uint32_t g) const { return (rows(g) + THREADS - 1) / THREADS; }  // keys of a thread
  // Lane l of a wave has the group's candidates first + l + 64 j at places place + l + 64 j, j < each(g). The places are a
  // wave's own whatever the group: the last one's share is smaller, and a wave may fetch it while others still read
  // theirs of the group before.
  constexpr uint32_t first(uint32_t g, uint32_t wave) const { return wave * 64 * each(g); }
  static constexpr uint32_t place(uint32_t wave) { return wave * 64 * PER; }
};

}  // namespace g4kv4
