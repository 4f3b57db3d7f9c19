"""Attention over the paged 4-bit cache where a CTA's share ends one kv head and begins the next, and both are cut into so many shares that they are joined in groups: one long sequence
among short ones."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import paged_oracle as P
from test_paged import check, cuda, filled, on_torch  # noqa: F401  (a fixture)


# Random batches dealt out by the kernel's own arithmetic: every word that counts has one owner (a triple, or a group of a triple's shares), and as many arrivals as its owner waits for.
WORDS = r"""
#include <cstdio>
#include <map>
#include <random>
#include <utility>
#include <vector>
#include "kv4_shares.cuh"
using namespace lmb::kv4;
int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  long long grouped = 0, met = 0;
  for (int batch = 0; batch < 6000; ++batch) {
    const int grids[] = {148, 296, 444, 592, 740, 1024}, ctas = grids[rng() % 6], heads = pick(1, 20), n_seq = pick(1, 40);
    std::vector<int> triples;
    int64_t U = 0;
    for (int b = 0; b < n_seq; ++b) {
      const int units = rng() % 4 ? pick(1, 30) : pick(1, 2000), tiles = rng() % 5 ? 1 : pick(1, 4);
      for (int t = 0; t < tiles * heads; ++t) { triples.push_back(units); U += units; }
    }
    const int shares = (int)(U < ctas ? U : ctas);
    for (int s = 0; s < shares; ++s)
      if (share_begin(s, U, shares) >= share_begin(s + 1, U, shares)) return printf("an empty share\n"), 1;
    std::map<int, std::pair<int, int>> owner;                  // word -> triple, group (-1: the triple's)
    std::map<int, int> arrivals, wanted;
    auto count = [&](int word, int triple, int group, int of) {
      if (word < 0 || word >= kCounters) return false;
      const auto o = owner.emplace(word, std::make_pair(triple, group)).first->second;
      wanted[word] = of;
      ++arrivals[word];
      return o == std::make_pair(triple, group);
    };
    int64_t item0 = 0;
    std::vector<int> first_of_group(shares, 0);
    for (int i = 0; i < (int)triples.size(); item0 += triples[i++]) {
      const int a = share_of(item0, U, shares), z = share_of(item0 + triples[i] - 1, U, shares);
      if (share_begin(a, U, shares) > item0 || share_begin(a + 1, U, shares) <= item0) return printf("a piece in another share\n"), 1;
      if (a == z) continue;
      for (int s = a; s <= z; ++s) {
        const Part q = part_of(item0, triples[i], s, U, shares);
        const bool many = q.groups > 1;
        if (q.sa != a || s < q.first || s >= q.first + q.count) return printf("a share outside its group\n"), 1;
        if (!count(part_counter(q), i, many ? (s - a) / kJoin : -1, q.count)) return printf("batch %d: two owners of word %d\n", batch, part_counter(q)), 1;
        if (many && s == q.first && !count(triple_counter(q), i, -1, q.groups)) return printf("batch %d: two owners of word %d\n", batch, triple_counter(q)), 1;
        grouped += many;
        if (many && s == q.first && first_of_group[s]++) ++met;
      }
    }
    for (const auto& w : wanted)
      if (arrivals[w.first] != w.second) return printf("word %d: %d arrivals of %d\n", w.first, arrivals[w.first], w.second), 1;
  }
  if (grouped < 100000 || met < 100) return printf("the batches are too small: %lld, %lld\n", grouped, met), 1;
  return 0;
}
"""


def test_every_counter_has_one_owner(tmp_path):
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "luminal.jl_b200", "csrc")
    src = tmp_path / "words.cpp"
    src.write_text(WORDS)
    subprocess.run([shutil.which("g++") or "c++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", csrc, str(src), "-o", str(tmp_path / "words")], check=True)
    r = subprocess.run([str(tmp_path / "words")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def plain(q, cu, lens, table, pages, page, scale):
    """The oracle's (out, size) for one row a sequence, in 64 bits on the GPU: sequences of many tokens."""
    import torch
    n, heads, D = len(pages) * page, pages.shape[1], q.shape[-1]
    every = np.arange(n)
    (k, v), (kn, vn) = ([cuda(x) for x in P.load(pages, every, page, D, size=s)] for s in (False, True))
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for b, l in enumerate(lens):
        pos = np.arange(l)
        slots = cuda(table[b, pos // page].astype(np.int64) * page + pos % page)
        x = q[cu[b]].double().unflatten(0, (heads, -1))                          # [heads, G, D]
        e = torch.softmax(scale * torch.einsum("hgd,khd->hgk", x, k[slots]), -1)
        most = 1 + abs(scale) * torch.einsum("hgd,khd->hgk", x.abs(), kn[slots]).amax(-1, keepdim=True)
        out[cu[b]] = torch.einsum("hgk,khd->hgd", e, v[slots]).flatten(0, 1).cpu().numpy()
        size[cu[b]] = (most * torch.einsum("hgk,khd->hgd", e, vn[slots])).flatten(0, 1).cpu().numpy()
    return out, size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,lens", [(8, [56320] + [300] * 23), (8, [53760] + [1000] * 27), (8, [60000] + [1000] * 31), (18, [24000]), (18, [9000] * 2 + [100000]), (13, [40000, 30000]),
                                        (5, [700, 90000, 20])])
def test_one_long_sequence_among_short_ones(on_torch, dtype, heads, lens):
    """Twenty calls with one workspace: the oracle's numbers, the same bits every time, and counters of 0 behind each."""
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(heads + len(lens))
    D, G, page, held = 128, 4, 64, 40
    lens = np.array(lens, np.int32)
    table = rng.integers(0, held, (len(lens), -(-int(lens.max()) // page))).astype(np.int32)       # sequences read the same pages, in other orders
    pages = filled(rng, held, heads, page, D)
    cu = np.arange(len(lens) + 1).astype(np.int32)
    q = cuda(rng.standard_normal((len(lens), heads * G, D)).astype(np.float32), torch.float32 if dtype == "f32" else torch.bfloat16)
    want, size = plain(q, cu, lens, table, pages, page, D ** -0.5)
    ws = torch.zeros(L.kv4_attention_workspace(dev, D), dtype=torch.uint8, device="cuda")
    args = cuda(cu), cuda(lens), cuda(table), cuda(pages)
    first = None
    for _ in range(20):
        out = torch.full_like(q, 7.0)
        L.kv4_attention(dev, q, out, *args, page_size=page, workspace=ws)
        dev.sync()
        if first is None:
            first = out
            check(out, want, size, dtype)
        assert torch.equal(out, first)
        assert not ws[:4 * 3 * 1024].any()                            # the counters come first
