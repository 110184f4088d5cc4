"""The walk behind the refusal of a captured backward pass that would reach an eager graph on the default stream, on nodes of
its own: no device, no torch."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <memory>
#include <unordered_set>
#include <vector>
#include "t5vq_graph_walk.h"
struct Node;
struct Edge { std::shared_ptr<Node> function; };
struct Node {
    std::vector<Edge> edges;
    bool eager = false;
    const std::vector<Edge>& next_edges() const { return edges; }
};
typedef std::shared_ptr<Node> P;
static std::vector<std::unique_ptr<Node>> all;                    // edges do not own: a long chain would be freed by recursion
static P make(std::vector<P> next = {}, bool eager = false) {
    all.push_back(std::make_unique<Node>());
    Node* n = all.back().get();
    for (auto& p : next) n->edges.push_back({p});
    n->eager = eager;
    return P(n, [](Node*) {});
}
static size_t looked;
static const Node* walk(const P& from, std::unordered_set<const Node*>* wanted = nullptr) {
    looked = 0;
    return t5vq_graph::first_behind(*from, [&](const Node* n) { return !wanted || wanted->count(n); },
                                    [&](const Node* n) { ++looked; return n->eager; });
}
#define CHECK(c) do { if (!(c)) { std::printf("failed at line %d: %s\n", __LINE__, #c); std::exit(1); } } while (0)
int main() {
    const P leaf = make({}, true), other = make();
    CHECK(walk(make()) == nullptr && looked == 0);
    CHECK(walk(make({nullptr, other, nullptr})) == nullptr && looked == 1);
    CHECK(walk(make({other, leaf})) == leaf.get());                       // a leaf handed to the operator itself
    const P cast = make({leaf}), view = make({cast});
    CHECK(walk(make({other, cast})) == leaf.get());                       // behind one operation
    CHECK(walk(make({nullptr, view})) == leaf.get());                     // behind two
    CHECK(walk(leaf) == nullptr);                                          // the running node itself is not behind itself
    const P mul = make({make()}, true);
    CHECK(walk(make({mul})) == mul.get());                                // an eager operation, not only a leaf
    // only what the pass runs: another leaf is asked for, or the way to the eager one is not taken
    const P asked = make(), both = make({cast, asked});
    std::unordered_set<const Node*> wanted{asked.get()};
    CHECK(walk(both, &wanted) == nullptr && looked == 1);
    wanted.insert(leaf.get());
    CHECK(walk(both, &wanted) == nullptr && looked == 1);                 // not through a node that does not run
    wanted.insert(cast.get());
    CHECK(walk(both, &wanted) == leaf.get());
    // 2^200 paths, each node once; then an eager leaf at their end
    P top = make();
    for (int i = 0; i < 200; ++i) top = make({make({top}), make({top})});
    CHECK(walk(make({top})) == nullptr && looked == 601);
    top = leaf;
    for (int i = 0; i < 200; ++i) top = make({make({top}), make({top})});
    CHECK(walk(make({top})) == leaf.get());
    // a long chain
    top = leaf;
    for (int i = 0; i < 1000000; ++i) top = make({top});
    CHECK(walk(top) == leaf.get() && looked == 1000000);
    std::printf("walk ok\n");
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_walk(tmp_path):
    source, program = tmp_path / "walk.cpp", tmp_path / "walk"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "t5vqvae_amd", "csrc"), "-o", str(program), str(source)], check=True, timeout=120)
    got = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0 and got.stdout == "walk ok\n", got.stdout + got.stderr
