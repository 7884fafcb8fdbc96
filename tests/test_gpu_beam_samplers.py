"""The samplers on the beam selection and the quantised history: LAIR with its history in 8 or 4 bits, and with the
proposals of the largest weights in the place of the final draws."""
import numpy as np
import pytest
import torch

from oracle import cs_oracle_beam as O
from tests.helpers import seeded_inputs
from tests.test_gpu_options_rng import check_imputations, model, run_sampler  # noqa: F401
from vae_conditional_sampling_amd import _lib

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "mxfp8", "mxfp4"]


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantised_queue_gives_what_a_float_queue_of_the_quantised_states_gives(fmt):
    from vae_conditional_sampling_amd.sampling.utils import ImputationHistoryQueue
    g = torch.Generator().manual_seed(5)
    B, K, D, T = 7, 4, 43, 5
    q = ImputationHistoryQueue(T, (B, K, D), storage=fmt)
    f = ImputationHistoryQueue(T, (B, K, D))
    assert q.history_queue.dtype == torch.uint8 and q.history_queue.numel() < 0.3 * 4 * f.history_queue.numel()
    group = 64 if fmt == "int8" else 32
    for t in range(8):                                   # (past the ring's end)
        X = torch.randn(B, K, D, generator=g) * 3
        q.enqueue_batch(X.cuda())
        f.enqueue_batch(torch.from_numpy(O.quantised(X.numpy(), fmt, group).astype(np.float32)).cuda())
        assert (q.tail_idx, q.full, len(q)) == (f.tail_idx, f.full, len(f))
    X = torch.randn(B, K, D, generator=g).cuda()
    coe = torch.randint(0, K, (B,), generator=g)
    rng = _lib.make_rng(9, 4, 1000)
    for kw in (dict(chain_of_proposal=[0, 2, 3]), dict(chain_of_example=coe), dict(rng=rng), dict()):
        a, b = q.concat_history(X, [1, 4, 2], **kw), f.concat_history(X, [1, 4, 2], **kw)
        assert torch.equal(a, b)
    out = torch.empty(B, K + 3, D, device="cuda")
    assert q.concat_history(X, [0, 0, 3], rng=rng, out=out) is out and torch.equal(out, f.concat_history(X, [0, 0, 3], rng=rng))
    with pytest.raises(NotImplementedError):
        ImputationHistoryQueue(T, (B, K, D), dtype=torch.bool, storage=fmt)
    with pytest.raises(NotImplementedError):
        ImputationHistoryQueue(T, (B, K, D), storage="int5")


@pytest.mark.parametrize("fmt", FORMATS)
def test_lair_with_its_history_in_few_bits(model, fmt):  # noqa: F811
    from vae_conditional_sampling_amd.sampling.test_step_vae_sampling import TestVAELatentAdaptiveImportanceResampling as S
    B, K, D = 130, 4, 9
    X, M = seeded_inputs(B, K, D, 31)
    X, M = X.cuda(), M.cuda()
    kw = dict(num_iterations=9, num_imp_samples=1, weighting_scheme="dmis", resampling_scheme="gr",
              resampling_method="multinomial", num_prior_replenish_proposals=1, num_pseudo_warmup_iterations=2,
              num_historical_proposals=3, no_historic_proposals_iterations=4, imputation_history_length=5)
    _, plain = run_sampler(S, model, X, M, **kw)
    s, outs = run_sampler(S, model, X, M, imputation_history_format=fmt, **kw)
    _, again = run_sampler(S, model, X, M, imputation_history_format=fmt, **kw)
    assert len(outs) == 11 and all(torch.equal(a["X"], b["X"]) for a, b in zip(outs, again))
    for o in outs:
        check_imputations(o["X"], X, M)
    # the same chains up to the first use of the history, others after it
    assert all(torch.equal(a["X"], b["X"]) for a, b in zip(outs[:5], plain[:5]))
    assert not torch.equal(outs[-1]["X"], plain[-1]["X"])
    kw.update(resampling_scheme="glr", weighting_scheme="dmis_within_groups", glr_cluster_size=4, num_prior_replenish_proposals=0,
              num_historical_proposals=4, no_historic_proposals_iterations=5, imputation_history_length=6, num_iterations=10)
    _, outs = run_sampler(S, model, X, M, imputation_history_format=fmt, **kw)
    for o in outs:
        check_imputations(o["X"], X, M)


@pytest.mark.parametrize("n", [1, 5, 64])
def test_the_proposals_of_the_largest_weights(model, n):  # noqa: F811
    from vae_conditional_sampling_amd.sampling.test_step_vae_sampling import TestVAELatentAdaptiveImportanceResampling as S
    B, K, D, T, R, I = 21, 4, 9, 6, 1, 2
    X, M = seeded_inputs(B, K, D, 13)
    X, M = X.cuda(), M.cuda()
    kw = dict(num_iterations=T, num_imp_samples=I, weighting_scheme="dmis", resampling_scheme="gr",
              resampling_method="multinomial", num_prior_replenish_proposals=R, resample_final_imps=True,
              resample_final_imps_num_samples=n)
    s, _ = run_sampler(S, model, X, M, resample_final_imps_method="top", **kw)
    Zp, lw = s._proposals
    lw[1, 0, 3] = lw[0, 0, 3]                             # equal weights: the earlier iteration first
    lw[:, :, 4] = float("-inf")                           # one proposal with a weight
    lw[2, 1, 4, 3] = -3.0
    lw[:, :, 5] = float("nan")                            # none
    imps, Z, idx = s.final_resampling(X[:, 0].cpu(), M)
    Kp = K + R
    flat = lw.reshape(T * I, B, Kp).permute(1, 0, 2).reshape(B, -1).cpu()
    order = torch.sort(flat, dim=1, descending=True, stable=True).indices[:, :n]
    order = torch.cat([order, order[:, :1].expand(B, n - order.shape[1])], dim=1)   # (T I K' = 60 proposals: then the best again)
    order[4] = (2 * I + 1) * Kp + 3
    order[5] = 0
    assert torch.equal(idx.cpu(), order)
    want = Zp.reshape(T * I, B, Kp, -1).cpu()[order // Kp, torch.arange(B)[:, None], order % Kp]
    assert torch.equal(Z.cpu(), want) and imps.shape == (1, B, n, D)
    obs = M[:, 0].cpu()
    assert all(torch.equal(imps[0, b, i].cpu()[obs[b]], X[b, 0].cpu()[obs[b]]) for b in range(B) for i in range(n))
    # the draws of the multinomial method are what they were
    a, _ = run_sampler(S, model, X, M, **kw)
    b, _ = run_sampler(S, model, X, M, resample_final_imps_method="multinomial", **kw)
    assert torch.equal(a.final_resampling(X[:, 0].cpu(), M)[2], b.final_resampling(X[:, 0].cpu(), M)[2])


def test_both_options_through_the_yaml_driver(tmp_path):
    """top: the whole run and two shards of it write the same; the history in 8 bits: the run ends and keeps what is
    observed."""
    import os
    from tests.helpers import ROOT
    from vae_conditional_sampling_amd import distributed, driver
    common = ["data.synthetic_num_test=90", "data.num_first_datapoints_test=61", "data.batch_size=32",
              "test_class.init_args.num_iterations=12"]
    top = common + ["test_class.init_args.resample_final_imps_method=top"]
    load = lambda name, extra, root: driver.load_config(os.path.join(ROOT, name), extra + [f"trainer.default_root_dir={root}"])
    name = "configs/uci_hepmass/sampling_u50/lair_k16_dmis_gr_mult_1replenish_wholedataset.yaml"
    whole, _ = driver.run(load(name, top, tmp_path / "one"))
    shards = [driver.run(load(name, top, tmp_path / "two"), rank=r, world_size=2)[0].collector.shard_arrays() for r in range(2)]
    out = str(tmp_path / "two" / "merged")
    distributed.write_batches(distributed.merge_shards(shards), 32, out)
    files = [n for n in os.listdir(whole.out_dir) if n.startswith("irwg_imputations_after_final_resampling_")]
    assert len(files) == 2
    for n in files:
        a, b = np.load(os.path.join(whole.out_dir, n)), np.load(os.path.join(out, n))
        assert a["imputations"].shape[2] == 5 and all(np.array_equal(a[k], b[k]) for k in a.files)
        m = np.broadcast_to(a["masks"][None], a["imputations"].shape)
        assert np.array_equal(a["imputations"][m], np.broadcast_to(a["true_X"][None], m.shape)[m])
    name = "configs/uci_miniboone/sampling_u50/lair_k4_dmis_gr_mult_1replenish.yaml"
    past = common + ["test_class.init_args.resample_final_imps=False", "test_class.init_args.num_historical_proposals=2",
                     "test_class.init_args.no_historic_proposals_iterations=3", "test_class.init_args.imputation_history_length=6",
                     "test_class.init_args.imputation_history_format=int8"]
    tester, outs = driver.run(load(name, past, tmp_path / "past"))
    f = np.load(os.path.join(tester.out_dir, "imputations_0.npz"))
    m = np.broadcast_to(f["masks"][None], f["imputations"].shape)
    assert np.isfinite(f["imputations"]).all()
    assert np.array_equal(f["imputations"][m], np.broadcast_to(f["true_X"][None], m.shape)[m])


def test_binary_data_keep_their_uint8_history():
    from tests.helpers import conv_weights, make_conv_model
    from tests.test_gpu_samplers import BASE_KW
    from vae_conditional_sampling_amd.sampling import test_step_vae_sampling as T
    enc_w, dec_w = conv_weights("omni_like", 7)
    g = torch.Generator().manual_seed(5)
    B, K, D = 3, 4, 784
    X0 = (torch.rand(B, 1, D, generator=g) < 0.3).float().repeat(1, K, 1)
    M = torch.rand(B, 1, D, generator=g) < 0.5
    runs = []
    for fmt in (None, "int8"):
        s = T.TestVAELatentAdaptiveImportanceResampling(
            num_iterations=6, num_imp_samples=1, weighting_scheme="dmis", resampling_scheme="gr", resampling_method="multinomial",
            num_prior_replenish_proposals=1, num_pseudo_warmup_iterations=1, num_historical_proposals=2,
            no_historic_proposals_iterations=3, imputation_history_length=4, imputation_history_format=fmt, num_copies=K, **BASE_KW)
        s.set_model(make_conv_model("omni_like", enc_w, dec_w, "normal", "bern"))
        s.on_test_start()
        s.rng_seed = 11
        s.on_test_batch_start(None, 0)
        Xi = s.basic_imputation(X0.cuda(), M.cuda())
        runs.append([d["X"].clone() for d in s.sampler(Xi, M.cuda())])
    assert len(runs[0]) == len(runs[1]) and all(torch.equal(a, b) for a, b in zip(*runs))
    assert not torch.equal(runs[0][0], runs[0][-1])
