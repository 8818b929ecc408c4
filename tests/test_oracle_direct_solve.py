"""The oracle's direct solve is the yardstick of the GPU parity tests (P(k) and samples to 1e-6): it has to be well
inside that itself, on every CPU and thread count."""
import numpy as np
import pytest
import scipy.linalg

from oracle import pspec_ref as R


def _system(N, T, M, frac):
    from hydra_pspec_amd import synthetic
    d = synthetic.make_baselines(N, T, M, k0=1, nbl=1, flag_frac=frac, dense=True)
    fl, S, Fm = d["flags"][0], d["S_initial"], d["fgmodes"]
    Ni = fl.T * d["Ninv"] * fl
    A = np.zeros((N + M, N + M), dtype=complex)
    A[:N, :N] = np.eye(N) + S @ Ni
    A[:N, N:] = S @ Ni @ Fm
    A[N:, :N] = Fm.T.conj() @ Ni
    A[N:, N:] = Fm.T.conj() @ Ni @ Fm
    ops = np.array([scipy.linalg.sqrtm(S), S, Ni, scipy.linalg.sqrtm(Ni)])
    return d["vis"][0] * fl, fl, Fm, [ops, np.array([A, A])]      # (the direct solve does not use the pseudo-inverse)


@pytest.mark.parametrize("N,T,M,frac", [(1024, 32, 12, 0.15), (1024, 32, 12, 0.0), (120, 20, 6, 0.1)])
def test_direct_solve_is_row_scale_independent(N, T, M, frac):
    """A's last M rows are larger than the rest by Ninv / 1, and an LU's error is relative to the largest rows.  With the
    error of a solve whose every row is solved to working accuracy, |r| <= g (|A| |x| + |b|) with g = (n + 2) 2 sqrt(2) u,
    the solution is off by at most |A^-1| |r| <= 2 g |A^-1| |A| |x| (|b| <= |A| |x|): the bound below, which does not
    change when a row of A is scaled.  Reference: the same system, refined with residuals in extended precision."""
    vis, fl, Fm, mats = _system(N, T, M, frac)
    A = mats[1][0]
    AL, lu = A.astype(np.clongdouble), scipy.linalg.lu_factor(A)
    inv = np.abs(np.linalg.inv(A))
    for t in (0, T // 2):
        x, _, info = R.gcr_fgmodes_1d(t, vis[t], fl, mats, Fm, solver="direct")
        assert info == 0
        b = _rhs(t, vis[t], fl, mats, Fm).astype(np.clongdouble)
        ref = scipy.linalg.lu_solve(lu, b.astype(complex)).astype(np.clongdouble)
        for _ in range(4):
            ref = ref + scipy.linalg.lu_solve(lu, (b - AL @ ref).astype(complex))
        bound = 2 * (N + M + 2) * 2 * 2 ** 0.5 * 2.0 ** -53 * (inv @ (np.abs(A) @ np.abs(x)))
        err = np.abs(x - ref).astype(float)
        print(f"t {t}: largest error {err.max() / np.abs(x).max():.2e} of the largest entry, signal part "
              f"{err[:N].max() / np.abs(x[:N]).max():.2e}, largest error / bound {np.max(err / bound):.2e}")
        assert np.all(err <= bound)
        assert err[:N].max() < 1e-8 * np.abs(x[:N]).max()         # a hundredth of the GPU tests' tolerance


def _rhs(idx, vis, w, mats, Fm):
    """b of the oracle's system, from its draws (four real normals per channel, in order)."""
    (Sh, S, Ni, Nih), N = mats[0], len(vis)
    state = np.random.get_state()
    np.random.seed(R.GCR_SEED0 + idx)
    z = [np.random.randn(N, 1) for _ in range(4)]
    np.random.set_state(state)
    oma, omb = (z[0] + 1j * z[1]) / 2 ** 0.5, (z[2] + 1j * z[3]) / 2 ** 0.5
    d = (w * vis).reshape(N, 1)
    top = S @ Ni @ d + Sh @ oma + S @ Nih @ omb
    return np.concatenate([top[:, 0], (Fm.T.conj() @ (Ni @ d + Nih @ omb))[:, 0]])
