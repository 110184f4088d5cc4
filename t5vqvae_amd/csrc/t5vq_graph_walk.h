// Internal to libt5vq_torch.so: a walk over what a backward pass will still run.
#ifndef T5VQ_GRAPH_WALK_H_
#define T5VQ_GRAPH_WALK_H_
#include <unordered_set>
#include <vector>

namespace t5vq_graph {

// The first node behind `from` (not `from` itself) that `found` picks, among those that `runs` admits and that are reached
// through admitted ones; null if there is none.  Every node is looked at once, however many paths lead to it, and the walk
// keeps its own stack.  Node: anything whose next_edges() holds smart pointers to nodes as `function`, null where an edge leads
// nowhere.
template <class Node, class Runs, class Found>
const Node* first_behind(const Node& from, Runs runs, Found found) {
    std::unordered_set<const Node*> seen{&from};
    std::vector<const Node*> open{&from};
    while (!open.empty()) {
        const Node* node = open.back();
        open.pop_back();
        for (const auto& edge : node->next_edges()) {
            Node* next = edge.function.get();
            if (!next || !seen.insert(next).second || !runs(next)) continue;
            if (found(next)) return next;
            open.push_back(next);
        }
    }
    return nullptr;
}

}  // namespace t5vq_graph
#endif
