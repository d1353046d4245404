// Host-side state shared by the library's translation units: error text and launch accounting of
// the calling thread (read back with flexsae_last_error and flexsae_last_launch_count).
#pragma once

namespace flexsae {

// Stores the text for flexsae_last_error() and returns `code`.
int fail(int code, const char* fmt, ...);

// Kernels enqueued by the current entry point.
extern thread_local int t_launches;

}  // namespace flexsae
