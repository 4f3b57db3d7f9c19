"""Verification of drafts where probabilities leave every number's range."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import cuda, on_torch  # noqa: F401  (a fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [6, 5000, 50000])
@pytest.mark.parametrize("draft_logits", [True, False])
@pytest.mark.parametrize("top,T", [(10000, 1e-6), (1000, 7e-8), (20, 2e-9), (1.0, 3e-10), (-50, 4e-9), (3.0e38, 1e28)])
def test_verify_logits_one_step_apart_at_temperatures_near_0(on_torch, vocab, draft_logits, top, T):
    """Two logits that are neighbours among the floats, so cold that the lower one's probability is far below any number: the higher one is the token, as a draft and as the new token."""
    import torch
    L, dev = on_torch
    top = np.float32(top)
    below = np.nextafter(top, np.float32(-np.inf))
    n, per = 6, 2
    rows = n * per
    rng = np.random.default_rng(41)
    target = np.full((rows, vocab), -np.inf, np.float32)
    draft = target.copy()
    best = rng.integers(0, vocab, rows)
    other = (best + rng.integers(1, vocab, rows)) % vocab
    r = np.arange(rows)
    target[r, best], target[r, other] = top, below
    draft[r, other], draft[r, best] = top, below                                 # the draft model takes the two the other way round
    cu = (np.arange(n + 1) * per).astype(np.int32)
    tokens = np.zeros(rows, np.int32)
    tokens[1::2] = np.where(np.arange(n) % 2 == 0, best[0::2], other[0::2])            # every second draft is refused
    temperature = np.full(n, T, np.float32)
    accept_u, sample_u = np.full(rows, 0.5, np.float32), np.linspace(0, 1 - 2 ** -24, n).astype(np.float32)
    use = draft if draft_logits else None
    want = P.verify(target, use, cu, tokens, temperature, accept_u, sample_u, np.full(rows, 55, np.int32))
    out, n_out, drop = (torch.full((k,), 55, dtype=torch.int32, device="cuda") for k in (rows, n, n))
    ws = torch.zeros(L.verify_drafts_workspace(rows), dtype=torch.uint8, device="cuda")
    L.verify_drafts(dev, cuda(target), None if use is None else cuda(draft), cuda(cu), cuda(tokens), cuda(temperature), cuda(accept_u), cuda(sample_u), out, n_out, drop, workspace=ws)
    dev.sync()
    for got, w in zip((out, n_out, drop), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert (want[0] >= 0).sum() >= n and (want[1] == np.where(np.arange(n) % 2 == 0, 2, 1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 50000])
@pytest.mark.parametrize("temperature", [None, 0.0, 1.0])
@pytest.mark.parametrize("cu", [[0, 4, 2, 1], [0, 6, 3, 6], [2, 6, 0, 5], [0, 5, 9, 6]])
def test_verify_offsets_that_share_rows_give_tokens_of_the_vocabulary(on_torch, vocab, temperature, cu):
    """Whatever the workspace held: a row that offsets give to two sequences holds a token or -1, the call is told of, and the next one is right."""
    import torch
    L, dev = on_torch
    rows, n = 6, 3
    rng = np.random.default_rng(42)
    target = cuda(rng.standard_normal((rows, vocab)).astype(np.float32))
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    tokens[1:] = target.argmax(1).cpu().numpy()[:-1]                        # every draft is the largest logit
    t = None if temperature is None else torch.full((n,), temperature, device="cuda")
    u = cuda(rng.random(rows).astype(np.float32))
    ints = lambda k: torch.full((k,), -1, dtype=torch.int32, device="cuda")  # noqa: E731
    for fill in (0x7f, 0x3f, 0xff):
        ws = torch.full((L.verify_drafts_workspace(rows),), fill, dtype=torch.uint8, device="cuda")
        out, n_out, drop = ints(rows), ints(n), ints(n)
        L.verify_drafts(dev, target, None, cuda(np.array(cu, np.int32)), cuda(tokens), t, u, u, out, n_out, drop, workspace=ws)
        with pytest.raises(L.LuminalB200Error) as e:
            dev.sync()
        assert e.value.code == -1
        assert ((out >= -1) & (out < vocab)).all() and ((n_out >= 0) & (n_out <= rows)).all() and ((drop >= 0) & (drop < rows)).all()
        good = np.array([0, 2, 2, 6], np.int32)
        want = P.verify(target.cpu().numpy(), None, good, tokens, None if t is None else t.cpu().numpy(), u.cpu().numpy(), u.cpu().numpy(), np.full(rows, 55, np.int32))
        L.verify_drafts(dev, target, None, cuda(good), cuda(tokens), t, u, u, out, n_out, drop, workspace=ws)
        dev.sync()
        for got, w in zip((out, n_out, drop), want):
            assert np.array_equal(got.cpu().numpy(), w)


# Logits below a top one at many temperatures: this exponential, CUDA's, and how far apart they may be.
EXP64 = r"""
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>
#include "exp64.cuh"
__global__ void both(const float* x, const float* top, const double* inv_T, double* ours, double* cudas, int n) {
  __shared__ double table[32];
  lmb::fill_table(table);
  __syncthreads();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    ours[i] = lmb::Power(table, top[i], inv_T[i])(x[i]);
    cudas[i] = exp(((double)fminf(x[i], 3.402823466e38f) - (double)top[i]) * inv_T[i]);
  }
}
int main() {
  const int n = 1 << 22;
  std::mt19937_64 rng(3);
  std::uniform_real_distribution<double> u(0, 1);
  std::vector<float> x(n), top(n);
  std::vector<double> inv(n), ours(n), cudas(n);
  for (int i = 0; i < n; ++i) {
    inv[i] = std::exp2(40 * u(rng) - 20);
    top[i] = (float)((2 * u(rng) - 1) * std::exp2(20 * u(rng) - 8));
    const double y = i % 4 == 0 ? -640 * u(rng) : i % 4 == 1 ? -u(rng) : i % 4 == 2 ? -30 * u(rng) : -std::exp2(-50 * u(rng));
    x[i] = std::fmin(top[i], (float)(top[i] + y / inv[i]));
  }
  x[0] = top[0]; x[1] = -INFINITY; x[2] = NAN; x[3] = INFINITY; top[3] = 3.402823466e38f; x[4] = -3.402823466e38f; top[4] = x[4];
  float *dx, *dt; double *di, *da, *db;
  cudaMalloc(&dx, n * 4); cudaMalloc(&dt, n * 4); cudaMalloc(&di, n * 8); cudaMalloc(&da, n * 8); cudaMalloc(&db, n * 8);
  cudaMemcpy(dx, x.data(), n * 4, cudaMemcpyHostToDevice);
  cudaMemcpy(dt, top.data(), n * 4, cudaMemcpyHostToDevice);
  cudaMemcpy(di, inv.data(), n * 8, cudaMemcpyHostToDevice);
  both<<<512, 256>>>(dx, dt, di, da, db, n);
  cudaMemcpy(ours.data(), da, n * 8, cudaMemcpyDeviceToHost);
  cudaMemcpy(cudas.data(), db, n * 8, cudaMemcpyDeviceToHost);
  if (cudaDeviceSynchronize() != cudaSuccess) return printf("%s\n", cudaGetErrorString(cudaGetLastError())), 1;
  if (ours[0] != 1 || ours[1] != 0 || ours[2] != 0 || ours[3] != 1 || ours[4] != 1) return printf("edges: %g %g %g %g %g\n", ours[0], ours[1], ours[2], ours[3], ours[4]), 1;
  int counted = 0;
  double worst = 0;
  const double half = std::exp2(-53.0);
  for (int i = 5; i < n; ++i) {
    const double y = std::fabs((x[i] - (double)top[i]) * inv[i]);               // in units of e
    if (y > 620) continue;                                                       // 2^-895: nearly all that counts
    // this one's 2.2e-15 + 6 + 3 |y| roundings, and CUDA's own: its argument's two, its result's one unit in the last place
    const double limit = 2.3e-15 + (6 + 2 + 5 * y) * half, off = std::fabs(ours[i] / cudas[i] - 1);
    worst = std::fmax(worst, off / limit);
    ++counted;
    if (!(off <= limit)) return printf("x %.9g top %.9g 1/T %.17g: %.17g, CUDA %.17g\n", x[i], top[i], inv[i], ours[i], cudas[i]), 1;
  }
  printf("%d compared, at most %.2f of the limit\n", counted, worst);
  return counted < n / 2;
}
"""


@pytest.mark.gpu
def test_the_exponential_beside_cudas(lib_built, device, tmp_path):
    import os
    import subprocess
    from importlib import import_module
    build = import_module("luminal_jl_b200._build")
    (tmp_path / "exp64.cu").write_text(EXP64)
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, str(tmp_path / "exp64.cu"), "-o", str(tmp_path / "exp64")], check=True)
    r = subprocess.run([str(tmp_path / "exp64")], capture_output=True, text=True, timeout=300, env={**os.environ})
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
