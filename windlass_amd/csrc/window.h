// window.h — the tiles of keys that attention through a sliding window goes through,
// and which of them have to be masked: arithmetic of the kernels (tree_dev.h), for the
// host too. Not public ABI.
//
// A request has `len` tokens in the cache and `nodes` behind them; a node of position pos
// (len + the number of its ancestors) sees of the former the first `sinks` and those
// fewer than `window` positions before its own. No position or window reaches 2^31.
#pragma once
#include <stdint.h>

namespace wl {
namespace paged {

// The first key, sinks apart, that position pos sees.
constexpr uint32_t window_from(uint32_t pos, uint32_t window) { return pos >= window ? pos - window + 1u : 0u; }

// Tiles of kt keys with none that some node sees: the first of them, and how many (the
// first node sees the earliest key; the sinks' tiles are [0, at)).
struct Skip {
    uint32_t at, n;
};
constexpr Skip window_skip(uint32_t len, uint32_t window, uint32_t sinks, uint32_t kt) {
    const uint32_t from = window_from(len, window) / kt, sunk = sinks / kt + (sinks % kt ? 1u : 0u);
    return from > sunk ? Skip{sunk, from - sunk} : Skip{~0u, 0u};
}

// Whether keys [k0, k0 + n), all of them before the nodes, have to be masked. Some node may
// not see some of them where they are not all sinks and k0 is below the first key of the
// last node a chain may have. The tile that begins at that key is masked too: this
// node may have seen nothing of the tile before it, and in the first tile that a row
// sees keys of it needs its reference, which the kernels set in a walk's first tile and in
// masked ones. (Without: infinite weights, and the walk done again. 64 chains of 8 through
// 2048 keys of 16-bit rows, no sinks, which meet this at one length in 32: 364 us, and 184
// with lengths one longer.)
constexpr bool window_masks(uint32_t len, uint32_t nodes, uint32_t window, uint32_t sinks, uint32_t k0, uint32_t n) {
    return k0 + n > sinks && k0 + window <= len + nodes;
}

}  // namespace paged
}  // namespace wl
