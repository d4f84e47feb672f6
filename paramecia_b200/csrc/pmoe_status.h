// Which callers have heard of a failure.  The kernels of operators without a handle count their failures on the device and never
// take one back; a caller asks on a stream, and hears of what was counted since that stream's last call.  So no caller takes another
// one's failure away, whatever streams and threads they use.  Host code only.
#pragma once
#include <map>
#include <mutex>
#include <utility>

namespace pmoe {

class FailureCounts {
    std::mutex mutex;
    std::map<std::pair<int, const void *>, unsigned> heard;   // by device and stream

public:
    // whether `count`, the device's failures so far, is news for `stream`
    bool news(int device, const void *stream, unsigned count)
    {
        std::lock_guard<std::mutex> lock(mutex);
        unsigned &last = heard[{device, stream}];
        const bool more = last != count;
        last = count;
        return more;
    }
};

}  // namespace pmoe
