// Memory of paged batches that are gone, kept for the next ones: a host that makes a batch for every step would otherwise pin, allocate and free for
// milliseconds each time. No CUDA in here: who gives memory back to the system does so with what gone() hands out, when it may.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <exception>
#include <mutex>
#include <vector>

namespace llamd {

struct KeptBlock {
    uint8_t *p = nullptr;
    size_t n = 0;
    void *event = nullptr;  // behind whatever still uses it, where its user made one; goes with the block
};

class Kept {
   public:
    Kept(size_t most, size_t most_bytes) : most_(most), most_bytes_(most_bytes) {}
    // What to allocate for n bytes: powers of two from 64 KB, so that lengths which grow from step to step find the blocks of those before them.
    static size_t rounded(size_t n) {
        size_t r = 1 << 16;
        while (r < n) r *= 2;
        return r;
    }
    // The smallest kept block that n bytes fit in; none that is more than four times as large as what would be allocated. Null: there is none.
    KeptBlock take(size_t n) {
        std::lock_guard<std::mutex> hold(lock_);
        size_t best = blocks_.size();
        for (size_t i = 0; i < blocks_.size(); i++)
            if (blocks_[i].n >= n && blocks_[i].n <= 4 * rounded(n) && (best == blocks_.size() || blocks_[i].n < blocks_[best].n)) best = i;
        if (best == blocks_.size()) return {};
        const KeptBlock b = blocks_[best];
        blocks_.erase(blocks_.begin() + best);
        bytes_ -= b.n;
        return b;
    }
    // Keeps b for the next batches. Too many: the smallest goes. Too many bytes: those kept longest go, or b itself where it is more than all of them may be.
    void keep(const KeptBlock &b) {
        std::lock_guard<std::mutex> hold(lock_);
        try {
            gone_.reserve(gone_.size() + blocks_.size() + 1);
            blocks_.reserve(blocks_.size() + 1);
        } catch (const std::exception &) {
            return;  // (no memory for a list entry: the block is lost)
        }
        if (b.n > most_bytes_) {
            gone_.push_back(b);
            return;
        }
        while (bytes_ + b.n > most_bytes_) drop(0);
        blocks_.push_back(b);
        bytes_ += b.n;
        if (blocks_.size() > most_) {
            size_t least = 0;
            for (size_t i = 1; i < blocks_.size(); i++)
                if (blocks_[i].n < blocks_[least].n) least = i;
            drop(least);
        }
    }
    // Everything kept is to go: memory has run short elsewhere.
    void let_go() {
        std::lock_guard<std::mutex> hold(lock_);
        try {
            gone_.reserve(gone_.size() + blocks_.size());
        } catch (const std::exception &) {
            return;
        }
        while (!blocks_.empty()) drop(blocks_.size() - 1);
    }
    // What keep() had no room for since the last time.
    std::vector<KeptBlock> gone() {
        std::lock_guard<std::mutex> hold(lock_);
        std::vector<KeptBlock> out;
        out.swap(gone_);
        return out;
    }

   private:
    void drop(size_t i) {
        gone_.push_back(blocks_[i]);
        bytes_ -= blocks_[i].n;
        blocks_.erase(blocks_.begin() + i);
    }
    const size_t most_, most_bytes_;
    std::mutex lock_;  // (batches are given back by whichever thread lets go of them last)
    size_t bytes_ = 0;
    std::vector<KeptBlock> blocks_, gone_;  // (the one kept longest first)
};

}  // namespace llamd
