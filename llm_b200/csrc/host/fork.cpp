// Sequences that share pages: forking a slot, what the forked sequences of a step share, compacting a pool, and which
// prompts of a batch are worth starting together.
#include <algorithm>
#include <vector>

#include "../prefix_plan.h"
#include "cache.hpp"

using namespace llmh;

namespace llmh {

// `count` children of a slot, as long as it is. Everything is checked before anything is taken. What the children share is
// theirs at once; *copies says which pages the caller has to copy before the children or the slot are stepped.
std::vector<int> Cache::fork(int slot, int count, std::vector<PageCopy>* copies) {
    require_held(slot);
    if (count < 1) throw Failure{LLMH_FORMAT, "a fork has at least one child"};
    if (count > slots.n_free())
        throw Failure{LLMH_CACHE_FULL, "slot " + std::to_string(slot) + " cannot have " + std::to_string(count) + " children: " +
                                           std::to_string(slots.n_free()) + " slots are free"};
    int length = lengths_[slot], full = length / PAGE, rest = length % PAGE;
    for (const Group& group : groups) {
        const std::vector<int>& pages = group.slot_pages[slot];
        int listed = std::min(pages_for(length), group.ring_pages);
        if ((int)pages.size() < listed)
            throw Failure{LLMH_INVARIANT, "slot " + std::to_string(slot) + " has fewer pages than positions"};
        long long need = (long long)count * (group.window ? listed : listed - full);
        if (need > group.pool.n_free())
            throw Failure{LLMH_CACHE_FULL, std::string("the ") + group.kind() + " group has " + std::to_string(group.pool.n_free()) +
                                               " free pages, the fork needs " + std::to_string(need)};
    }
    std::vector<int> children;
    for (int i = 0; i < count; ++i) children.push_back(acquire());
    for (size_t g = 0; g < groups.size(); ++g) {
        Group& group = groups[g];
        int listed = std::min(pages_for(length), group.ring_pages);
        for (int child : children) {
            lengths_[child] = length;
            for (int i = 0; i < listed; ++i) {
                int page = group.slot_pages[slot][i];
                if (!group.window && i < full) {
                    group.give(child, page);
                } else {
                    // (a ring's page may hold positions of its last turn behind the newest one: it is copied whole)
                    int own = group.pool.take();
                    group.give(child, own);
                    copies->push_back({(int)g, page, own, group.window ? PAGE : rest});
                }
            }
        }
    }
    return children;
}

// Whether new sequences of these final lengths fit beside what is held, if the first shared[i] positions of sequence i (whole pages)
// are pages of the one before it.
bool Cache::can_hold_shared(int n, const long long* lengths, const long long* shared) const {
    if (n > slots.n_free()) return false;
    for (int i = 0; i < n; ++i)
        if (lengths[i] > max_seq_len) return false;
    for (const Group& group : groups) {
        long long pages = 0;
        for (int i = 0; i < n; ++i)
            pages += group.window ? std::min(pages_for(lengths[i]), group.ring_pages)
                                  : pages_for(lengths[i]) - std::min<long long>(shared[i], lengths[i]) / PAGE;
        if (pages > group.pool.n_free()) return false;
    }
    return true;
}

// The moves that leave a group's held pages at the front of its pool: the last held pages to the first free places.
std::vector<PageCopy> Cache::plan_compact(int g) const {
    const Group& group = groups[g];
    std::vector<PageCopy> moves;
    int held = group.pool.n_held(), to = 0;
    for (int page = held; page < group.pool.count(); ++page) {
        if (!group.pool.is_held(page)) continue;
        while (group.pool.is_held(to)) ++to;
        moves.push_back({g, page, to++, PAGE});
    }
    return moves;
}

void Cache::apply_moves(int g, const std::vector<int>& from, const std::vector<int>& to) {
    Group& group = groups[g];
    group.pool.exchange(from, to);
    std::vector<int> now(group.pool.count());
    for (int page = 0; page < group.pool.count(); ++page) now[page] = page;
    for (size_t i = 0; i < from.size(); ++i) {
        now[from[i]] = to[i];
        group.holders[to[i]] = group.holders[from[i]];
        group.holders[from[i]] = 0;
    }
    for (int slot = 0; slot < max_slots; ++slot)
        for (size_t i = 0; i < group.slot_pages[slot].size(); ++i)
            group.table[(size_t)slot * group.ring_pages + i] = group.slot_pages[slot][i] = now[group.slot_pages[slot][i]];
}

// The first pages that two slots have in common, as far as both are past them (a `full` group; all of them share alike).
int Cache::common_pages(int slot_a, int slot_b) const {
    for (const Group& group : groups) {
        if (group.window) continue;
        const std::vector<int>&a = group.slot_pages[slot_a], &b = group.slot_pages[slot_b];
        size_t most = std::min({a.size(), b.size(), (size_t)(std::min(lengths_[slot_a], lengths_[slot_b]) / PAGE)});
        return (int)(std::mismatch(a.begin(), a.begin() + most, b.begin()).first - a.begin());
    }
    return 0;
}

// A position is about to be written: its page must be the slot's alone.
void Cache::require_writable(int slot, long long position) const {
    for (const Group& group : groups) {
        if (group.window) continue;
        size_t i = (size_t)(position / PAGE);
        if (i < group.slot_pages[slot].size() && group.holders[group.slot_pages[slot][i]] > 1)
            throw Failure{LLMH_INVARIANT, "position " + std::to_string(position) + " of slot " + std::to_string(slot) +
                                              " lies on a page that other slots hold"};
    }
}

}  // namespace llmh

namespace {

// Neighbours i and i + 1 have common[i] items in common, and so has a run of neighbours the least of its numbers. Cuts the n into
// runs such that the sum of (members - 1) * common items is greatest; first[k] is where run k starts, first[runs] = n. Runs are at most
// MOST_MEMBERS long. Of equal sums the one with longer runs at the end.
constexpr int MOST_MEMBERS = 1024;

int best_runs(int n, const int* common, int* first) {
    std::vector<long long> best(n + 1, 0);
    std::vector<int> from(n + 1, 0);
    for (int j = 1; j <= n; ++j) {
        best[j] = best[j - 1];
        from[j] = j - 1;
        int least = 0x7fffffff;
        for (int i = j - 2; i >= 0 && j - i <= MOST_MEMBERS; --i) {
            least = std::min(least, common[i]);
            if (least <= 0) break;
            long long sum = best[i] + (long long)(j - 1 - i) * least;
            if (sum >= best[j]) {
                best[j] = sum;
                from[j] = i;
            }
        }
    }
    int runs = 0;
    for (int j = n; j > 0; j = from[j]) ++runs;
    first[runs] = n;
    for (int j = n, k = runs; j > 0; j = from[j]) first[--k] = from[j];
    return runs;
}

}  // namespace

// children: room for `count` slots. copies: 4 ints each {group, source page, target page, rows}, up to `capacity` of them; their number
// is at most count * (1 + pages of the rings).
LLMH_EXPORT int llmh_cache_fork(void* cache, int slot, int count, int* children, int* copies, int capacity, int* n_copies) {
    return guarded([&] {
        std::vector<PageCopy> list;
        Cache* c = static_cast<Cache*>(cache);
        long long most = 0;
        for (const Group& group : c->groups) most += (long long)std::max(count, 0) * (group.window ? group.ring_pages : 1);
        if (most > capacity) throw Failure{LLMH_INVARIANT, "the list of copies has room for " + std::to_string(capacity)};
        std::vector<int> slots = c->fork(slot, count, &list);
        std::copy(slots.begin(), slots.end(), children);
        *n_copies = (int)list.size();
        for (size_t i = 0; i < list.size(); ++i) {
            copies[4 * i] = list[i].group;
            copies[4 * i + 1] = list[i].source;
            copies[4 * i + 2] = list[i].target;
            copies[4 * i + 3] = list[i].rows;
        }
    });
}
LLMH_EXPORT int llmh_cache_can_hold_shared(void* cache, int n, const long long* lengths, const long long* shared) {
    return static_cast<Cache*>(cache)->can_hold_shared(n, lengths, shared) ? 1 : 0;
}
// from, to: room for every page of the group.
LLMH_EXPORT int llmh_cache_plan_compact(void* cache, int group, int* from, int* to, int* count) {
    return guarded([&] {
        Cache* c = static_cast<Cache*>(cache);
        if (group < 0 || group >= (int)c->groups.size()) throw Failure{LLMH_INVARIANT, "no such group"};
        std::vector<PageCopy> moves = c->plan_compact(group);
        *count = (int)moves.size();
        for (size_t i = 0; i < moves.size(); ++i) {
            from[i] = moves[i].source;
            to[i] = moves[i].target;
        }
    });
}
LLMH_EXPORT int llmh_cache_apply_moves(void* cache, int group, int count, const int* from, const int* to) {
    return guarded([&] {
        Cache* c = static_cast<Cache*>(cache);
        if (group < 0 || group >= (int)c->groups.size()) throw Failure{LLMH_INVARIANT, "no such group"};
        c->apply_moves(group, std::vector<int>(from, from + count), std::vector<int>(to, to + count));
    });
}

// The groups of a step's entries that share pages: entries first[g] .. first[g + 1] - 1 have pages[g] pages in common (first: room for
// n + 1, pages: for n). summary: [groups, most new tokens of an entry, of a group, most shared pages, most positions behind them, pages that are
// read once less for each further member of a group]; groups = 0: nothing is shared.
LLMH_EXPORT int llmh_step_groups(void* cache, int n, const int* slots, const int* counts, int* first, int* pages, int* summary) {
    return guarded([&] {
        const Cache& c = *static_cast<Cache*>(cache);
        std::vector<int> common(n);
        for (int i = 0; i < n; ++i) c.require_held(slots[i]);
        for (int i = 0; i + 1 < n; ++i) common[i] = c.common_pages(slots[i], slots[i + 1]);
        int groups = best_runs(n, common.data(), first);
        int max_new = 0, max_group = 0, max_shared = 0, max_own = 0, saved = 0;
        for (int g = 0; g < groups; ++g) {
            int shared = first[g + 1] - first[g] > 1 ? 0x7fffffff : 0, tokens = 0;
            for (int i = first[g]; i + 1 < first[g + 1]; ++i) shared = std::min(shared, common[i]);
            pages[g] = shared;
            for (int i = first[g]; i < first[g + 1]; ++i) {
                tokens += counts[i];
                max_new = std::max(max_new, counts[i]);
                max_own = std::max(max_own, c.length(slots[i]) + counts[i] - shared * PAGE);
            }
            max_group = std::max(max_group, tokens);
            max_shared = std::max(max_shared, shared);
            saved += (first[g + 1] - first[g] - 1) * shared;
        }
        summary[5] = saved;
        summary[0] = max_shared > 0 ? groups : 0;
        summary[1] = max_new;
        summary[2] = max_group;
        summary[3] = max_shared;
        summary[4] = max_own;
    });
}

// Whether a step of single tokens in bfloat16 has every sequence read its shared pages itself (prefix_plan.h).
LLMH_EXPORT int llmh_prefix_reads_alone(long long walks, int shared, long long group_rows) {
    return llmb_prefix::reads_alone(walks, shared, group_rows, true, false) ? 1 : 0;
}

// About how many microseconds the attention of a prompt step in bfloat16 takes where every sequence reads its pages for itself (*apart: a block for 128
// tokens and a query head, two on an SM) and where tiles of a group's rows read the shared ones once (*once: prefix_plan.h). A page takes a
// block 0.77 apart and 0.57 of an SM's time where there are many; a tile of 256 rows 0.98, one of at most 128 rows 0.78, if its keys serve several
// query heads. Against measured steps of up to 80 sequences with 8 to 512 shared pages, 32 heads over 8 and over 32: once 0.6 to 1.3 times, apart 0.35
// (many short prompts) to 1.3 times what it took; which one is the faster it says rightly of 133 of 143.
LLMH_EXPORT int llmh_step_attention_times(void* cache, int n, const int* slots, const int* counts, int groups, const int* first, const int* pages,
                                          int n_heads, int n_kv_heads, int head_dim, double* apart, double* once) {
    return guarded([&] {
        using namespace llmb_prefix;
        const Cache& c = *static_cast<Cache*>(cache);
        const int share = n_heads / n_kv_heads;
        double all_pages = 0, chain = 0;
        std::vector<int> token(n + 1, 0);
        for (int s = 0; s < n; ++s) {
            token[s + 1] = token[s] + counts[s];
            for (int t = 0; t < counts[s]; t += 128) {
                const double seen = (c.length(slots[s]) + std::min(t + 127, counts[s] - 1)) / PAGE + 1;
                all_pages += seen * n_heads;
                chain = std::max(chain, seen);
            }
        }
        *apart = std::max(0.77 * chain, 0.57 * all_pages / SMS) + 5;

        // the tiles as the launch has them: as many for each group as the largest has, the last round cut into pieces
        int most_tokens = 0, most_shared = 0, most_own = 0;
        for (int g = 0; g < groups; ++g) {
            most_tokens = std::max(most_tokens, token[first[g + 1]] - token[first[g]]);
            most_shared = std::max(most_shared, pages[g]);
            for (int s = first[g]; s < first[g + 1]; ++s) most_own = std::max(most_own, pages_for(c.length(slots[s]) + counts[s]) - pages[g]);
        }
        const long long tiles_of = ((long long)most_tokens * share + WIDE_ROWS - 1) / WIDE_ROWS, all = tiles_of * groups * n_kv_heads;
        const long long uncut = all / SMS * SMS;
        const int pieces = wide_pieces(all - uncut, bucket(most_shared) + bucket(std::max(most_own, 1)), head_dim);
        double work = 0, longest = 0;
        long long blocks = 0;
        for (int g = 0; g < groups; ++g) {
            const long long rows = (long long)(token[first[g + 1]] - token[first[g]]) * share;
            int s = first[g];
            for (long long row = 0; row < rows; row += WIDE_ROWS) {
                const long long left = std::min<long long>(WIDE_ROWS, rows - row);
                const int t0 = token[first[g]] + (int)(row / share), t1 = token[first[g]] + (int)((row + left - 1) / share);
                while (token[s + 1] <= t0) ++s;
                int walk = pages[g];
                for (int i = s; i < first[g + 1] && token[i] <= t1; ++i)
                    if (counts[i] > 0) walk += (c.length(slots[i]) + std::min(counts[i] - 1, t1 - token[i])) / PAGE + 1 - pages[g];
                const double page = left <= TILE_ROWS && share > 1 ? 0.78 : 0.98;
                const long long at = (g * tiles_of + row / WIDE_ROWS) * n_kv_heads;
                for (int cut = 0; cut < 2; ++cut) {          // of its key heads, those before and those in the last round
                    const long long heads = cut ? std::max(at + n_kv_heads - std::max(at, uncut), 0ll) : std::max(std::min(at + n_kv_heads, uncut) - at, 0ll);
                    if (heads == 0) continue;
                    const int of = cut ? pieces : 1, part = (walk + of - 1) / of;
                    work += heads * of * (part + 10) * page;
                    longest = std::max(longest, (part + 12) * page);
                    blocks += heads * of;
                }
            }
        }
        const double rounds = (double)((blocks + SMS - 1) / SMS);
        *once = std::max(longest, blocks > 0 ? rounds * work / blocks : 0.0) + (pieces > 1 && all > uncut ? 3 : 0);
    });
}

// The same choice for n prompts (tokens flat, counts each): prompts first[k] .. first[k + 1] - 1 start together with their first common[k] tokens,
// a multiple of `unit` that leaves each of them a token, 0 for a prompt alone. first: room for n + 1, common: for n.
LLMH_EXPORT int llmh_prompt_runs(int n, const int* counts, const int* tokens, int unit, int* first, int* common, int* runs) {
    return guarded([&] {
        if (n < 0 || unit < 1) throw Failure{LLMH_FORMAT, "bad sizes"};
        std::vector<int> least(n);
        const int* a = tokens;
        for (int i = 0; i + 1 < n; ++i) {
            const int* b = a + counts[i];
            int most = std::max(std::min(counts[i], counts[i + 1]) - 1, 0);
            least[i] = (int)(std::mismatch(a, a + most, b).first - a) / unit * unit;
            a = b;
        }
        *runs = best_runs(n, least.data(), first);
        for (int k = 0; k < *runs; ++k) {
            common[k] = first[k + 1] - first[k] > 1 ? 0x7fffffff : 0;
            for (int i = first[k]; i + 1 < first[k + 1]; ++i) common[k] = std::min(common[k], least[i]);
        }
    });
}
