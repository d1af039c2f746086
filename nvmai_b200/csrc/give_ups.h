// Which stream's owner has been told of which given-up wait (nvmai_cuda_moe_int8_matmul_status).
#pragma once
#include <cstdint>
#include <map>
#include <mutex>
#include <thread>
#include <tuple>

namespace nvmai {

// The device counts the waits that its products gave up and never goes back.  Each stream has the count that its owner knows of; a
// question compares the two, so an owner's question takes nobody else's answer, and a wait given up while one asks is
// in the next answer.  A stream starts, at its first product, from the last count that anybody has read: no later than that product.
// One without products (graphs replayed on it were captured elsewhere) starts from none, and is told of all there have been.
class GiveUps {
public:
    // ahead of a product on the stream
    void product(int dev, const void *stream) {
        struct Last { const GiveUps *of; int dev; const void *stream; };
        static thread_local Last last{};                 // most products follow one on the same stream: 4 ns instead of 16
        if (last.of == this && last.dev == dev && last.stream == stream) return;
        {
            std::lock_guard<std::mutex> lock(guard_);
            known_.emplace(key(dev, stream), read_[dev]);
        }
        last = Last{this, dev, stream};
    }
    // The count read behind the stream's work: is there anything its owner does not know of?
    bool news(int dev, const void *stream, uint32_t count) {
        std::lock_guard<std::mutex> lock(guard_);
        read_[dev] = count;
        uint32_t &known = known_.emplace(key(dev, stream), 0u).first->second;
        const bool is_new = known != count;
        known = count;
        return is_new;
    }

private:
    using Key = std::tuple<int, const void *, std::thread::id>;
    static Key key(int dev, const void *stream) {
        const bool per_thread = stream == reinterpret_cast<const void *>(2);       // cudaStreamPerThread: each thread's own
        return Key{dev, stream, per_thread ? std::this_thread::get_id() : std::thread::id{}};
    }
    std::mutex guard_;
    std::map<Key, uint32_t> known_;
    std::map<int, uint32_t> read_;
};

}  // namespace nvmai
