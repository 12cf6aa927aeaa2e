// Host build of the absorbed latent attention's share of workgroups
// (helix_runtime_amd/csrc/latent.hpp): prints it for 256 workgroups and each number of
// row blocks from 0 to argv[1].
#include "../../helix_runtime_amd/csrc/latent.hpp"

#include <cstdio>
#include <cstdlib>

int main(int argc, char** argv) {
  if (argc != 2) return 2;
  const std::size_t most = std::strtoul(argv[1], nullptr, 10);
  for (std::size_t n = 0; n <= most; ++n) std::printf("%zu\n", helix::hip::latent_share(256, n));
  return 0;
}
