// linear8_shape.h -- where the kernels of linear8.hip read, as plain C++ (compiled
// for the host alone by the tests).
#pragma once

namespace ember {

// Operands are read through buffers of this many bytes from a tile's first row on, no
// fewer than its rows have: 256 of at most 2^23.  A load's offset has a lane's share,
// its place in the tile, and one that all lanes have, the group of k.  The lane's is the
// one that is sure to be held against the buffer's size, so past the last group it lies
// past the buffer: such a load gives 0 and reads nothing.
constexpr unsigned kBufferBytes = 0x80000000u;
constexpr unsigned lane_offset(unsigned in_tile, bool there)
{
    return in_tile | (there ? 0u : kBufferBytes);
}

}  // namespace ember
