// What the last launch on each stream wrote, for launches that read ahead of their wait: host arithmetic only.
#pragma once

#include <stddef.h>

namespace tsr {

class LaunchRecord {
 public:
  // Whether a launch that reads `reads` ahead of its wait may start under the last one on `stream` of `device` (a stream's handle
  // may be another device's too: the default stream's is); records `writes` as what it writes itself.
  bool next(int device, const void* stream, const void* const* reads, const size_t* read_bytes, int nreads, const void* const* writes,
            const size_t* write_bytes, int nwrites) {
    Last* slot = nullptr;
    for (Last& l : table_)
      if (l.used && l.stream == stream && l.device == device) slot = &l;
    // a stream new to the table, or one that others have pushed out of it: what its last launch wrote is not known
    bool ok = slot != nullptr || nreads <= 0;
    if (slot == nullptr) {
      slot = &table_[next_];
      next_ = (next_ + 1) % kStreams;
      *slot = Last{};
    }
    for (int i = 0; i < nreads; ++i) {
      const auto* r = static_cast<const unsigned char*>(reads[i]);
      for (int j = 0; j < slot->count; ++j)
        if (r < slot->ptr[j] + slot->bytes[j] && slot->ptr[j] < r + read_bytes[i]) ok = false;  // previous output is our weight
    }
    if (slot->count < 0) ok = false;  // more outputs than the table holds: anything may have been written
    slot->device = device;
    slot->stream = stream;
    slot->used = true;
    slot->count = nwrites <= kRanges ? nwrites : -1;
    for (int j = 0; j < slot->count; ++j) {
      slot->ptr[j] = static_cast<const unsigned char*>(writes[j]);
      slot->bytes[j] = write_bytes[j];
    }
    return ok;
  }

 private:
  static constexpr int kStreams = 16, kRanges = 12;
  struct Last {
    const void* stream;
    bool used;
    int device, count;
    const unsigned char* ptr[kRanges];
    size_t bytes[kRanges];
  };
  Last table_[kStreams] = {};
  int next_ = 0;
};

}  // namespace tsr
