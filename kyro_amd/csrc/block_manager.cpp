// Host block allocator and block-granular prefix cache (see block_manager.hpp for the
// differences from the reference and why).
#include "block_manager.hpp"

#include <algorithm>

namespace kyro {
namespace bm {

namespace {
int64_t blocks_for(int64_t tokens, int bs) { return (tokens + bs - 1) / bs; }

size_t common_prefix(const Tokens& a, const uint32_t* b, size_t nb) {
    const size_t n = std::min(a.size(), nb);
    size_t i = 0;
    while (i < n && a[i] == b[i]) ++i;
    return i;
}
}  // namespace

// ------------------------------------------------------------------------------ RadixCache

RadixCache::RadixCache(int block_size, int64_t max_capacity) : bs_(block_size), capacity_(max_capacity) {}

void RadixCache::leaf_add(Node* n) {
    if (n != &root_ && n->children.empty()) leaves_.insert({n->last_access, n});
}

void RadixCache::leaf_remove(Node* n) { leaves_.erase({n->last_access, n}); }

// The reference stamps Instant::now() on each matched node (radix_cache.rs:74); a logical clock
// gives the same order without ties between calls.
void RadixCache::touch(Node* n) {
    const bool leaf = n->children.empty();
    if (leaf) leaf_remove(n);
    n->last_access = ++clock_;
    if (leaf) leaf_add(n);
}

// radix_cache.rs:49-86 walks nodes whose token runs match in full. Here a node is one block:
// whole blocks match by key, and the walk ends at the child sharing the longest prefix with the
// next (partial or diverging) block, which the caller treats as a partially matched block.
std::pair<std::vector<int64_t>, int64_t> RadixCache::match_prefix(const uint32_t* t, int64_t n) {
    std::vector<int64_t> blocks;
    Node* node = &root_;
    int64_t pos = 0;
    while (pos < n) {
        const int64_t take = std::min<int64_t>(bs_, n - pos);
        if (take == bs_) {
            auto it = node->children.find(Tokens(t + pos, t + pos + take));
            if (it != node->children.end()) {
                Node* c = it->second.get();
                touch(c);
                blocks.push_back(c->block);
                pos += take;
                node = c;
                continue;
            }
        }
        Node* best = nullptr;
        size_t best_len = 0;
        for (auto& kv : node->children) {  // map order: ties go to the smallest key
            const size_t c = common_prefix(kv.first, t + pos, (size_t)take);
            if (c > best_len) {
                best_len = c;
                best = kv.second.get();
            }
        }
        if (best) {
            touch(best);
            blocks.push_back(best->block);
            pos += (int64_t)best_len;
        }
        break;
    }
    return {blocks, pos};
}

// radix_cache.rs:89-120 inserts the remaining tokens as one node holding every block of the
// sequence, so a later match returns blocks twice; here each block becomes its own node and a
// block already cached under the same tokens is reported as not taken. Eviction after an insert
// (:117-119) returns the evicted blocks so their references can be dropped.
std::vector<bool> RadixCache::insert(const uint32_t* t, int64_t n, const int64_t* blocks,
                                     std::vector<int64_t>* evicted) {
    const int64_t nb = blocks_for(n, bs_);
    std::vector<bool> taken((size_t)nb, false);
    Node* node = &root_;
    for (int64_t i = 0; i < nb; ++i) {
        const int64_t p0 = i * bs_, p1 = std::min<int64_t>(n, p0 + bs_);
        Tokens key(t + p0, t + p1);
        auto it = node->children.find(key);
        if (it != node->children.end()) {
            node = it->second.get();
            touch(node);
            continue;
        }
        if ((int64_t)node->key.size() < bs_ && node != &root_) break;  // partial nodes stay leaves
        auto child = std::make_unique<Node>();
        child->key = std::move(key);
        child->block = blocks[i];
        child->parent = node;
        child->last_access = ++clock_;
        Node* c = child.get();
        leaf_remove(node);  // the parent stops being a leaf
        node->children.emplace(c->key, std::move(child));
        leaf_add(c);
        ++num_cached_;
        taken[(size_t)i] = true;
        node = c;
    }
    if (num_cached_ > capacity_) {
        std::vector<int64_t> ev = evict_lru();
        if (evicted) evicted->insert(evicted->end(), ev.begin(), ev.end());
    }
    return taken;
}

// radix_cache.rs:126-155 takes the oldest leaf among the first tree level that has one, in
// HashMap order; here it is the least recently used leaf of the whole tree.
bool RadixCache::evict_one(int64_t* block) {
    if (leaves_.empty()) return false;
    Node* n = leaves_.begin()->second;
    leaves_.erase(leaves_.begin());
    *block = n->block;
    Node* parent = n->parent;
    const Tokens key = n->key;
    parent->children.erase(key);  // frees n
    --num_cached_;
    leaf_add(parent);
    return true;
}

void RadixCache::cached_blocks(std::vector<int64_t>* out) const {
    std::vector<const Node*> stack{&root_};
    while (!stack.empty()) {
        const Node* n = stack.back();
        stack.pop_back();
        if (n != &root_) out->push_back(n->block);
        for (auto& kv : n->children) stack.push_back(kv.second.get());
    }
}

std::vector<int64_t> RadixCache::evict_lru() {
    std::vector<int64_t> out;
    int64_t b;
    while (num_cached_ > capacity_ && evict_one(&b)) out.push_back(b);
    return out;
}

// ---------------------------------------------------------------------------- BlockManager

// block_manager.rs:32-50: every GPU block free (popped from the back, so block N-1 first) and a
// cache budget of a third of the GPU blocks.
BlockManager::BlockManager(int block_size, int64_t num_gpu_blocks, int64_t num_cpu_blocks)
    : bs_(block_size), num_gpu_(num_gpu_blocks), num_cpu_(num_cpu_blocks),
      ref_((size_t)num_gpu_blocks, 0), cache_(block_size, num_gpu_blocks / 3) {
    free_.reserve((size_t)num_gpu_blocks);
    for (int64_t b = 0; b < num_gpu_blocks; ++b) free_.push_back(b);
}

void BlockManager::release(int64_t block) {
    int& r = ref_[(size_t)block];
    if (r <= 0) return;  // never reached when every holder drops its reference once
    if (--r == 0) free_.push_back(block);
}

// block_manager.rs:67-76 evicts once, down to the cache budget, and may still fail; here leaves
// are evicted one at a time until n blocks are free or the cache is empty.
bool BlockManager::reserve(int64_t n) {
    int64_t b;
    while ((int64_t)free_.size() < n && cache_.evict_one(&b)) release(b);
    return (int64_t)free_.size() >= n;
}

// block_manager.rs:53-102. A match ending inside a block cannot share that block (the request
// writes its own tokens into the rest of it), so the request gets a fresh block and a pending
// copy of the cached one; the matched token count is the reference's cached_token_count.
int BlockManager::allocate_with_prefix(uint64_t rid, const uint32_t* tokens, int64_t n, int64_t* cached) {
    if (n < 0 || table_.count(rid)) return EINVAL_;
    auto match = cache_.match_prefix(tokens, n);
    const int64_t matched = match.second;
    const int64_t full = matched / bs_;
    const bool partial = matched % bs_ != 0;
    const int64_t cow_src = partial ? match.first[(size_t)full] : -1;
    for (int64_t i = 0; i < full; ++i) ++ref_[(size_t)match.first[(size_t)i]];
    if (partial) ++ref_[(size_t)cow_src];  // held until the copy is handed out
    const int64_t need = blocks_for(n, bs_) - full;
    if (!reserve(need)) {
        for (int64_t i = 0; i < full; ++i) release(match.first[(size_t)i]);
        if (partial) release(cow_src);
        return ENOSPACE;
    }
    Request r;
    r.blocks.assign(match.first.begin(), match.first.begin() + full);
    for (int64_t i = 0; i < need; ++i) {
        const int64_t b = free_.back();
        free_.pop_back();
        ref_[(size_t)b] = 1;
        r.blocks.push_back(b);
    }
    if (partial) copies_.push_back({cow_src, r.blocks[(size_t)full]});
    r.prompt.assign(tokens, tokens + n);
    r.has_prompt = true;
    r.num_tokens = n;
    table_.emplace(rid, std::move(r));
    *cached = matched;
    return OK;
}

// block_manager.rs:107-124 (no prefix caching, no eviction).
int BlockManager::allocate(uint64_t rid, int64_t num_tokens) {
    if (num_tokens < 0 || table_.count(rid)) return EINVAL_;
    const int64_t need = blocks_for(num_tokens, bs_);
    if ((int64_t)free_.size() < need) return ENOSPACE;
    Request r;
    for (int64_t i = 0; i < need; ++i) {
        const int64_t b = free_.back();
        free_.pop_back();
        ref_[(size_t)b] = 1;
        r.blocks.push_back(b);
    }
    r.num_tokens = num_tokens;
    table_.emplace(rid, std::move(r));
    return OK;
}

// Room for n more tokens (a decode token, or the k + 1 rows of a verify step). Positions at or
// past the prompt always lie in blocks the request owns alone, so they can be written.
int BlockManager::append_slots(uint64_t rid, int64_t n) {
    auto it = table_.find(rid);
    if (it == table_.end() || n < 0) return EINVAL_;
    Request& r = it->second;
    const int64_t need = blocks_for(r.num_tokens + n, bs_) - (int64_t)r.blocks.size();
    if (need > 0) {
        if (!reserve(need)) return ENOSPACE;
        for (int64_t i = 0; i < need; ++i) {
            const int64_t b = free_.back();
            free_.pop_back();
            ref_[(size_t)b] = 1;
            r.blocks.push_back(b);
        }
    }
    r.num_tokens += n;
    return OK;
}

// Drops rows after num_tokens (rejected drafts), releasing blocks no longer covered. The prompt
// is never cut: its last block may be shared with the cache. A request made private has no prompt, but
// may share blocks behind its front ones: the next row must not be written into one of them.
int BlockManager::truncate(uint64_t rid, int64_t num_tokens) {
    auto it = table_.find(rid);
    if (it == table_.end()) return EINVAL_;
    Request& r = it->second;
    const int64_t floor_len = r.has_prompt ? (int64_t)r.prompt.size() : 0;
    if (num_tokens < floor_len || num_tokens > r.num_tokens) return EINVAL_;
    if (!r.has_prompt && num_tokens % bs_ != 0 && ref_[(size_t)r.blocks[(size_t)(num_tokens / bs_)]] > 1) return EINVAL_;
    const int64_t keep = blocks_for(num_tokens, bs_);
    while ((int64_t)r.blocks.size() > keep) {
        release(r.blocks.back());
        r.blocks.pop_back();
    }
    r.num_tokens = num_tokens;
    return OK;
}

// A request whose cached tokens are about to be moved (eviction) owns the blocks of its first num_tokens
// tokens alone, the ones that are written: every one of them that another holder shares is replaced by a fresh
// block and a pending copy. Its blocks no longer hold its prompt in order, so the prompt is forgotten: it is
// not handed to the prefix cache when the request ends, and truncate may cut below it. Evicting cache leaves
// to make room can only lower reference counts, so the blocks are looked at again after it.
int BlockManager::make_private(uint64_t rid, int64_t num_tokens) {
    auto it = table_.find(rid);
    if (it == table_.end() || num_tokens < 0) return EINVAL_;
    Request& r = it->second;
    const size_t front = (size_t)blocks_for(std::min(num_tokens, r.num_tokens), bs_);
    int64_t need = 0;
    for (size_t i = 0; i < front; ++i) need += ref_[(size_t)r.blocks[i]] > 1;
    if (!reserve(need)) return ENOSPACE;
    for (size_t i = 0; i < front; ++i) {
        const int64_t b = r.blocks[i];
        if (ref_[(size_t)b] <= 1) continue;
        const int64_t fresh = free_.back();
        free_.pop_back();
        ref_[(size_t)fresh] = 1;
        copies_.push_back({b, fresh});  // the request's reference on b is the copy's from here on
        r.blocks[i] = fresh;
    }
    r.prompt.clear();
    r.has_prompt = false;
    return OK;
}

// block_manager.rs:128-153 hands the request's blocks to the cache with the prompt. Here the
// cache takes its own reference on the blocks it did not already hold, then the request drops
// its reference on all of its blocks, so each block is freed when its last holder lets go.
// cache_prompt = false (a request ended before its prompt's K/V was written) skips the cache.
int BlockManager::free(uint64_t rid, bool cache_prompt) {
    auto it = table_.find(rid);
    if (it == table_.end()) return EINVAL_;
    Request r = std::move(it->second);
    table_.erase(it);
    std::vector<int64_t> evicted;
    if (cache_prompt && r.has_prompt && !r.prompt.empty()) {
        const std::vector<bool> taken =
            cache_.insert(r.prompt.data(), (int64_t)r.prompt.size(), r.blocks.data(), &evicted);
        for (size_t i = 0; i < taken.size(); ++i)
            if (taken[i]) ++ref_[(size_t)r.blocks[i]];
    }
    for (int64_t b : r.blocks) release(b);
    for (int64_t b : evicted) release(b);
    return OK;
}

std::string BlockManager::check() const {
    std::vector<int> holders((size_t)num_gpu_, 0);
    for (auto& kv : table_)
        for (int64_t b : kv.second.blocks) ++holders[(size_t)b];
    std::vector<int64_t> cached;
    cache_.cached_blocks(&cached);
    if ((int64_t)cached.size() != cache_.num_cached_blocks()) return "cache node count disagrees";
    for (int64_t b : cached) ++holders[(size_t)b];
    for (auto& c : copies_) ++holders[(size_t)c.first];
    std::vector<char> in_free((size_t)num_gpu_, 0);
    for (int64_t b : free_) {
        if (b < 0 || b >= num_gpu_) return "free pool holds an invalid id";
        if (in_free[(size_t)b]) return "block " + std::to_string(b) + " is twice in the free pool";
        in_free[(size_t)b] = 1;
    }
    for (int64_t b = 0; b < num_gpu_; ++b) {
        if (holders[(size_t)b] != ref_[(size_t)b])
            return "block " + std::to_string(b) + ": " + std::to_string(holders[(size_t)b]) + " holders, ref count " +
                   std::to_string(ref_[(size_t)b]);
        if ((holders[(size_t)b] == 0) != (in_free[(size_t)b] != 0))
            return "block " + std::to_string(b) + (in_free[(size_t)b] ? " is free but held" : " is unheld but not free");
    }
    return "";
}

const Request* BlockManager::find(uint64_t rid) const {
    auto it = table_.find(rid);
    return it == table_.end() ? nullptr : &it->second;
}

// The copies are handed out once; the source's reference is dropped then, so the caller must
// queue the copies before anything else writes into the cache on that stream.
std::vector<std::pair<int64_t, int64_t>> BlockManager::take_copies() {
    std::vector<std::pair<int64_t, int64_t>> out;
    out.swap(copies_);
    for (auto& c : out) release(c.first);
    return out;
}

// Sorted, lists with a common start are neighbours, and the runs of neighbours that share at least d blocks nest: a tree,
// whose node of d blocks has lists and deeper runs below it. Some of its nodes are opened as groups. A list leaves out most
// in the deepest open node above it, all d of whose blocks it has in common, and an open node reads them once. So with a
// the blocks of the nearest open node above v, the most that the lists below v leave out is
//   f(v, a) = max(v's lists * a + sum of f(run, a),  (v's lists - 1) * d + sum of f(run, d)),
// worked out from the innermost runs for each node above v as the nearest open one. Those are fewer than v has blocks, so
// that all of it takes no more room or time than the lists.
std::vector<PrefixGroup> prefix_groups(const std::vector<const std::vector<int64_t>*>& lists) {
    struct Node {
        int64_t blocks;
        std::vector<int32_t> lists, runs;  // by place in the sorted order; nodes
        int32_t parent = -1, level = 0;    // nodes above it
        int32_t open_below = 0;            // it opens where the nearest open node above is at a lower level than this
        int32_t nearest = 0, group = -1;   // that node's level; the group of its lists, -1: each by itself
    };
    const size_t n = lists.size();
    std::vector<int32_t> order(n);
    for (size_t i = 0; i < n; ++i) order[i] = (int32_t)i;
    std::stable_sort(order.begin(), order.end(), [&](int32_t a, int32_t b) { return *lists[(size_t)a] < *lists[(size_t)b]; });
    // The tree, runs before what they lie in, the root of no blocks last.
    std::vector<Node> nodes, open(1);
    open[0].blocks = 0;
    for (size_t i = 0; i < n; ++i) {
        int64_t d = 0;  // blocks in common with the next list
        if (i + 1 < n) {
            const std::vector<int64_t>&a = *lists[(size_t)order[i]], &b = *lists[(size_t)order[i + 1]];
            const size_t m = std::min(a.size(), b.size());
            d = std::mismatch(a.begin(), a.begin() + (ptrdiff_t)m, b.begin()).first - a.begin();
        }
        int32_t run = -1;  // what has just ended: the list, or a run up to it
        auto put = [&](Node& to) { run < 0 ? to.lists.push_back((int32_t)i) : to.runs.push_back(run); };
        while (open.back().blocks > d) {
            put(open.back());
            run = (int32_t)nodes.size();
            nodes.push_back(std::move(open.back()));
            open.pop_back();
        }
        if (open.back().blocks < d) {
            open.emplace_back();
            open.back().blocks = d;
        }
        put(open.back());
    }
    nodes.push_back(std::move(open.back()));
    for (size_t v = nodes.size(); v-- > 0;)
        for (const int32_t r : nodes[v].runs) {
            nodes[(size_t)r].parent = (int32_t)v;
            nodes[(size_t)r].level = nodes[v].level + 1;
        }
    // best[v][j]: f(v, a) for the node at level j above v as the nearest open one.
    std::vector<std::vector<int64_t>> best(nodes.size());
    for (size_t v = 0; v + 1 < nodes.size(); ++v) {
        Node& node = nodes[v];
        best[v].resize((size_t)node.level);
        int64_t opened = ((int64_t)node.lists.size() - 1) * node.blocks;
        for (const int32_t r : node.runs) opened += best[(size_t)r][(size_t)node.level];
        int32_t above = node.parent;
        for (int32_t j = node.level; j-- > 0; above = nodes[(size_t)above].parent) {
            int64_t apart = (int64_t)node.lists.size() * nodes[(size_t)above].blocks;
            for (const int32_t r : node.runs) apart += best[(size_t)r][(size_t)j];
            best[v][(size_t)j] = std::max(apart, opened);
            if (opened > apart && node.open_below == 0) node.open_below = j + 1;  // apart falls with j
        }
        for (const int32_t r : node.runs) std::vector<int64_t>().swap(best[(size_t)r]);
    }
    // From the root: which nodes open, and the group of each list.
    std::vector<int64_t> group_blocks;
    std::vector<int32_t> group_of(n, -1);
    for (size_t v = nodes.size(); v-- > 0;) {
        Node& node = nodes[v];
        if (node.parent >= 0) {
            const Node& above = nodes[(size_t)node.parent];
            node.nearest = above.nearest;
            node.group = above.group;
            if (node.nearest < node.open_below) {
                node.nearest = node.level;
                node.group = (int32_t)group_blocks.size();
                group_blocks.push_back(node.blocks);
            }
        }
        for (const int32_t i : node.lists) group_of[(size_t)i] = node.group;
    }
    // In the order of each group's first list.
    std::vector<PrefixGroup> groups;
    std::vector<int32_t> place(group_blocks.size(), -1);
    for (size_t i = 0; i < n; ++i) {
        const int32_t g = group_of[i];
        if (g < 0) {
            groups.push_back({{order[i]}, 0});
            continue;
        }
        if (place[(size_t)g] < 0) {
            place[(size_t)g] = (int32_t)groups.size();
            groups.push_back({{}, group_blocks[(size_t)g]});
        }
        groups[(size_t)place[(size_t)g]].members.push_back(order[i]);
    }
    return groups;
}

}  // namespace bm
}  // namespace kyro
