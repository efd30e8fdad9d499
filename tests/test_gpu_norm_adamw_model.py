"""enable_LN and optimizer="adamw" of the model: engine steps against the oracle, in every update mode, on the bf16 path,
sharded, captured, through fit() and through checkpoints.

With 32-bit states the bars are those of the other optimizers' step tests (1e-5 for losses; 2e-4 of the tensor's scale
for parameters after Adam-like steps, which divide rounding noise by sqrt(v))."""
import copy

import numpy as np
import pytest
import torch

from oracle import xdeepfm_oracle as X
from recommenders_amd.models.deeprec.models._engine import XDeepFMEngine
from recommenders_amd.models.deeprec.models._sharded import ShardedXDeepFMEngine
from tests.util import make_hp, random_batch, random_features, write_libffm

pytestmark = pytest.mark.gpu


def close(got, exp, rtol, what):
    got, exp = np.asarray(got, dtype=np.float64), np.asarray(exp, dtype=np.float64)
    assert got.shape == exp.shape, (what, got.shape, exp.shape)
    scale, err = max(float(np.abs(exp).max()), 1e-30), float(np.abs(got - exp).max())
    assert err <= rtol * scale, "%s: %.3e of scale %.3e" % (what, err, scale)


def upload(eng, b):
    return eng.upload(b["labels"], b["dnn_feat_indices"], b["dnn_feat_values"], b["dnn_feat_weights"])


def start(hp, seed):
    """Initial tensors, the norms' weights away from 1 and 0."""
    p = X.init_params(hp, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    return {k: v + 0.2 * torch.randn(v.shape, generator=gen) if k.startswith("ln_") else v for k, v in p.items()}


def engine(hp, p, **kw):
    eng = XDeepFMEngine(hp, **kw)
    eng.load_state({k: v.clone() for k, v in p.items()})
    return eng


def check_params(sd, p64, rtol, skip=()):
    for k, v in p64.items():
        if not k.startswith(tuple(skip)):
            close(sd[k].float().cpu().numpy().reshape(v.shape), v.numpy(), rtol, "param " + k)


@pytest.mark.parametrize("optimizer", ["adam", "adamw", "sgd"])
@pytest.mark.parametrize("mode", ["dense_exact", "sparse_rows"])
@pytest.mark.parametrize("variant", ["plain", "dropout", "softmax"])
def test_steps_match_the_oracle(optimizer, mode, variant):
    kw = dict(enable_LN=True, optimizer=optimizer, learning_rate=0.01, FEATURE_COUNT=300, weight_decay=0.05,
              loss="cross_entropy_loss")
    if mode == "dense_exact" and optimizer == "adamw":
        kw["embed_weight_decay"] = 0.02
    if optimizer == "adam":
        kw.update(layer_l2=0.01 if mode == "dense_exact" else 0.0, cross_l2=0.01)
    if variant == "dropout":
        kw.update(user_dropout=True, dropout=[0.2, 0.3])
    if variant == "softmax":
        kw["activation"] = ["softmax", "elu"]
    hp = make_hp(**kw)
    rng = np.random.default_rng(15)
    p32 = start(hp, 6)
    eng = engine(hp, p32, embedding_update=mode)
    p64 = {k: v.double() for k, v in p32.items()}
    st = X.new_opt_state(p64, hp)
    for step in range(4):
        B = 128 if step != 1 else 77
        b = random_batch(rng, hp, B)
        loss, dloss = eng.train_step(upload(eng, b))
        masks = None
        if variant == "dropout":
            masks = [eng.ws["drop_%d" % k][:B].cpu().numpy().astype(np.float64) for k in range(2)]
        o_loss, o_dl, _, _ = X.train_step(p64, st, b, hp, dropout_masks=masks, adam_rows=mode != "dense_exact")
        close(float(dloss), o_dl, 2e-5, "data loss step %d" % step)
        close(float(loss), o_loss, 2e-5, "total loss step %d" % step)
    eng.check_errors()
    # a bias in front of a norm moves the row's mean alone where the norm follows at once: what is left of its gradient
    # is not zero (the norm is over the units), so every parameter is compared
    check_params(eng.state_dict(), p64, 5e-4 if optimizer != "sgd" else 5e-5)
    # scoring: the same norm, no statistics of its own
    b = random_batch(rng, hp, 50)
    eng.forward(upload(eng, b), with_loss=False)
    own = {k: eng.state_dict()[k].detach().cpu().double().reshape(v.shape) for k, v in p64.items()}
    logit, _ = X.forward(own, b, hp)
    close(eng.ws["logit"][:50].cpu().numpy(), logit.numpy()[:, 0], 1e-5, "logit")


@pytest.mark.parametrize("mode", ["dense_exact", "sparse_rows"])
def test_adamw_without_a_norm_matches_the_oracle(mode):
    hp = make_hp(optimizer="adamw", learning_rate=0.01, FEATURE_COUNT=300)
    rng = np.random.default_rng(2)
    p32 = X.init_params(hp, seed=3)
    eng = engine(hp, p32, embedding_update=mode)
    p64 = {k: v.double() for k, v in p32.items()}
    st = X.new_opt_state(p64, hp)
    for step in range(4):
        b = random_batch(rng, hp, 64)
        loss, _ = eng.train_step(upload(eng, b))
        close(float(loss), X.train_step(p64, st, b, hp, adam_rows=mode != "dense_exact")[0], 1e-5, "loss")
    check_params(eng.state_dict(), p64, 5e-4)


@pytest.mark.parametrize("mode", ["dense_exact", "sparse_rows"])
def test_8_bit_states_take_the_step_of_their_values(mode):
    """A step reads the values its codes stand for and rounds only what it writes back: a 32-bit engine that is handed
    parameters and state values of an 8-bit one takes the same next step, in every bit of the parameters."""
    kw = dict(enable_LN=True, optimizer="adamw", learning_rate=0.01, FEATURE_COUNT=300)
    hp32, hp8 = make_hp(**kw), make_hp(adamw_state_bits=8, **kw)
    rng = np.random.default_rng(4)
    p = start(hp32, 5)
    coded = engine(hp8, p, embedding_update=mode)
    assert coded.dense_m is None and (mode != "dense_exact" or coded.table_m is None)
    for step in range(4):
        plain = XDeepFMEngine(hp32, embedding_update=mode)
        plain.load_state({k: v.clone() if torch.is_tensor(v) else v for k, v in coded.state_dict().items()
                          if not k.startswith("slot8/")})
        batch = random_batch(rng, hp32, 64)
        la, lb = plain.train_step(upload(plain, batch))[0], coded.train_step(upload(coded, batch))[0]
        assert float(la) == float(lb)
        sa, sb = plain.state_dict(), coded.state_dict()
        for k in p:
            assert torch.equal(sa[k], sb[k]), (k, step)
        if step:  # ... and what is written back is rounded
            assert not torch.equal(sa["slot/dense_m"], sb["slot/dense_m"].float())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("mode", ["dense_exact", "sparse_rows"])
def test_checkpoints_resume_in_every_bit(bits, mode):
    hp = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=bits, learning_rate=0.01, FEATURE_COUNT=300)
    rng = np.random.default_rng(9)
    p = start(hp, 1)
    a = engine(hp, p, embedding_update=mode, seed=3)
    batches = [random_batch(rng, hp, 40) for _ in range(4)]
    for x in batches[:2]:
        a.train_step(upload(a, x))
    saved = {k: v.clone() if torch.is_tensor(v) else v for k, v in copy.copy(a.state_dict()).items()}
    b = XDeepFMEngine(hp, embedding_update=mode, seed=3)
    b.load_state(saved)
    for x in batches[2:]:
        a.train_step(upload(a, x))
        b.train_step(upload(b, x))
    sa, sb = a.state_dict(), b.state_dict()
    assert set(sa) == set(sb)
    for k, v in sa.items():
        assert torch.equal(v, sb[k]) if torch.is_tensor(v) else v == sb[k], k
    # the other kind of states: from the values
    other = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=40 - bits, learning_rate=0.01, FEATURE_COUNT=300)
    c = XDeepFMEngine(other, embedding_update=mode, seed=3)
    c.load_state(saved)
    sc = c.state_dict()
    assert c.step == 2 and float(c.opt_state[3]) == 2
    names = ["slot/dense_m", "slot/dense_v"] + (["slot/table_m", "slot/table_v", "slot/lin_v"] if mode == "dense_exact" else [])
    for k in names:
        # half a step of the codes (a sixteenth of the value), and half a unit: 2^-17 of the block's largest m, 2^-33 of v
        x, y = saved[k].float().cpu(), sc[k].float().cpu()
        assert ((x - y).abs() <= x.abs() / 16 + 2.0 ** -17 * x.abs().max()).all(), k
        assert float(y.abs().max()) > 0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(bits):
    hp = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=bits, learning_rate=0.01, FEATURE_COUNT=300,
                 batch_size=64)
    rng = np.random.default_rng(3)
    p = start(hp, 2)

    def one_token_per_field():
        labels, feats = random_features(rng, 64, hp.FIELD_COUNT, hp.FEATURE_COUNT, multi_p=0.0, missing_p=0.0)
        from oracle import ffm_iterator_oracle as O
        return O.convert(labels, feats, hp.FIELD_COUNT, hp.FEATURE_COUNT)

    batches = [one_token_per_field() for _ in range(5)]
    for mode in ("dense_exact", "sparse_rows"):
        a, b = engine(hp, p, embedding_update=mode, seed=1), engine(hp, p, embedding_update=mode, seed=1)

        def arrays(eng, x):
            idx = torch.from_numpy(np.ascontiguousarray(x["dnn_feat_indices"])).cuda()
            return (torch.from_numpy(np.asarray(x["labels"], dtype=np.float32).reshape(-1)).cuda(), idx,
                    torch.from_numpy(np.asarray(x["dnn_feat_values"])).cuda(),
                    torch.from_numpy(np.asarray(x["dnn_feat_weights"], dtype=np.float32)).cuda())

        gs = b.capture_step(*arrays(b, batches[0]))
        a.train_step(upload(a, batches[0]))
        for k, x in enumerate(batches[1:]):
            la = a.train_step(upload(a, x))[0]
            lb = gs.run(*arrays(b, x))[0]
            if k % 2:
                torch.cuda.synchronize()
            assert float(la) == float(lb)
        sa, sb = a.state_dict(), b.state_dict()
        for k, v in sa.items():
            assert torch.equal(v, sb[k]) if torch.is_tensor(v) else v == sb[k], (mode, k)


def test_bf16_products_with_a_norm():
    """compute_dtype bf16: products of bf16 operands (2^-8 each, 2e-2 in all as for the plain tower), norm in fp32."""
    hp = make_hp(enable_LN=True, optimizer="adamw", learning_rate=0.001, FEATURE_COUNT=300, FIELD_COUNT=8, dim=16,
                 layer_sizes=[64, 48], cross_layer_sizes=[16, 16], activation=["tanh", "sigmoid"],
                 loss="cross_entropy_loss")
    rng = np.random.default_rng(8)
    p = start(hp, 4)
    eng = engine(hp, p, compute_dtype="bf16", embedding_update="sparse_rows")
    b = random_batch(rng, hp, 97)
    eng.forward(upload(eng, b), with_loss=True, with_grad=True)
    db = upload(eng, b)
    eng.forward(db, with_loss=True, with_grad=True)
    eng.backward(db)
    eng.join_late()
    p64 = {k: v.double().requires_grad_(True) for k, v in p.items()}
    logit, _ = X.forward(p64, b, hp)
    close(eng.ws["logit"][:97].cpu().numpy(), logit.detach().numpy()[:, 0], 2e-2, "logit")
    labels = torch.as_tensor(np.asarray(b["labels"])).double()
    X.data_loss(logit, X.pred_from_logit(logit, hp), labels, hp).backward()
    for k in ("ln_dnn_g_0", "ln_dnn_o_0", "ln_dnn_g_1", "ln_dnn_o_1", "dnn_w_1"):
        got, exp = eng.grad_views[k].double().cpu(), p64[k].grad
        assert float((got - exp).norm() / exp.norm()) <= 2e-2, k


def test_sharded_engine_takes_the_same_steps():
    """One rank holding all rows: both modes, both kinds of states, against the plain engine."""
    for bits in (32, 8):
        for mode in ("dense_exact", "sparse_rows"):
            hp = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=bits, learning_rate=0.01,
                         FEATURE_COUNT=301, embed_weight_decay=0.1 if mode == "dense_exact" else 0.0)
            rng = np.random.default_rng(6)
            p = start(hp, 7)
            a = engine(hp, p, embedding_update=mode, seed=5)
            s = ShardedXDeepFMEngine(hp, seed=5, embedding_update=mode)
            s.load_global_state({k: v.clone() for k, v in p.items()})
            for _ in range(3):
                b = random_batch(rng, hp, 64)
                la, ls = a.train_step(upload(a, b))[0], s.train_step(upload(s, b))[0]
                close(float(ls), float(la), 1e-5 if bits == 32 else 1e-3, "loss")
            sa, ss = a.state_dict(), s.state_dict()
            for k in p:
                # (8 bits: sums in another order may cross a code's border and the steps part: no more than both
                # runs' steps together, 1.01 lr each for states in 32 bits and, with two roundings of m up and of v
                # down by an eighth, (9/8)^2 / (7/8) = 1.45 times that)
                d = float((sa[k].float() - ss[k].float().reshape(sa[k].shape)).abs().max())
                assert d <= (max(2e-4 * float(sa[k].abs().max()), 1e-6) if bits == 32 else 2 * 2 * 1.47 * 0.01), k


def _two_rank_worker(rank, world, port, bits, mode, out):
    """One rank of two processes that share cuda:0 and talk over gloo with host-staged exchanges."""
    import os

    import torch.distributed as dist

    from oracle import ffm_iterator_oracle as O

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        hp = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=bits, learning_rate=0.01, FEATURE_COUNT=301,
                     loss="cross_entropy_loss")
        p32 = start(hp, 9)
        eng = ShardedXDeepFMEngine(hp, seed=7, embedding_update=mode)
        eng.load_global_state({k: v.clone() for k, v in p32.items()})
        p64 = {k: v.double() for k, v in p32.items()}
        st = X.new_opt_state(p64, hp)
        rng = np.random.default_rng(21)  # every rank draws the same global batches
        per = 48
        for step in range(4):
            labels, feats = random_features(rng, per * world, hp.FIELD_COUNT, hp.FEATURE_COUNT)
            mine = slice(rank * per, (rank + 1) * per)
            loss, dloss = eng.train_step(upload(eng, O.convert(labels[mine], feats[mine], hp.FIELD_COUNT,
                                                               hp.FEATURE_COUNT)))
            tot = torch.stack([loss, dloss]).double().cpu()
            dist.all_reduce(tot)
            if bits == 32:
                o = X.train_step(p64, st, O.convert(labels, feats, hp.FIELD_COUNT, hp.FEATURE_COUNT), hp,
                                 adam_rows=mode != "dense_exact")
                close(float(tot[0]), o[0], 2e-5, "loss step %d" % step)
        eng.check_errors()
        # the replicated variables and their states: the same bits on every rank
        flat = [eng.dense.cpu()] + [t.cpu() for n, t in sorted(eng.state_dict().items()) if "/dense_" in n]
        for t in flat:
            both = [torch.empty_like(t) for _ in range(world)]
            dist.all_gather(both, t)
            assert torch.equal(both[0], both[1])
        if bits == 32:
            table, lin = eng.gather_global_table()
            check_params({**{k: eng.views[k] for k in eng.dense_shapes}, "embedding": table, "lin_w": lin}, p64, 5e-4)
        out.put((rank, "ok"))
    except Exception:  # noqa: BLE001
        import traceback

        out.put((rank, traceback.format_exc()))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("mode", ["dense_exact", "sparse_rows"])
def test_two_ranks_stay_together(bits, mode):
    """World size 2: the norm needs no exchange (its weights' gradients ride in the all-reduce of the dense ones), the
    replicated variables take the same step on every rank, rounding of 8-bit states included."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    procs = [ctx.Process(target=_two_rank_worker, args=(r, 2, port, bits, mode, out)) for r in range(2)]
    for p in procs:
        p.start()
    res = [out.get(timeout=100) for _ in procs]
    for p in procs:
        p.join(timeout=30)
    assert sorted(res) == [(r, "ok") for r in range(2)], res


def test_fit_with_a_norm_and_adamw(tmp_path):
    from recommenders_amd.models.deeprec.io.iterator import FFMTextIterator
    from recommenders_amd.models.deeprec.models.xDeepFM import XDeepFMModel

    rng = np.random.default_rng(11)
    labels, feats = random_features(rng, 500, 7, 300, multi_p=0.0, missing_p=0.0)
    train = write_libffm(str(tmp_path / "train.txt"), labels, feats)
    for bits in (32, 8):
        hp = make_hp(enable_LN=True, optimizer="adamw", adamw_state_bits=bits, FEATURE_COUNT=300, batch_size=50,
                     epochs=2, learning_rate=0.01, save_model=True, save_epoch=1, MODEL_DIR=str(tmp_path))
        model = XDeepFMModel(hp, FFMTextIterator, seed=2)
        model.fit(train, train)
        res = model.run_eval(train)
        assert set(res) == {"auc", "logloss"} and all(np.isfinite(v) for v in res.values())
        again = XDeepFMModel(hp, FFMTextIterator, seed=9)
        again.load_model(str(tmp_path / "epoch_2"))
        assert again.run_eval(train) == res


def test_what_the_engine_refuses():
    for kw, text in ((dict(enable_LN=True, enable_BN=True), "exclude"), (dict(layer_l2=0.1), "must be 0"),
                     (dict(cross_l1=0.1), "must be 0"), (dict(is_clip_norm=1), "clip"),
                     (dict(adamw_state_bits=16), "32 or 8")):
        with pytest.raises(ValueError, match=text):
            XDeepFMEngine(make_hp(optimizer="adamw", **kw))
    with pytest.raises(ValueError, match="dense_exact"):
        XDeepFMEngine(make_hp(optimizer="adamw", embed_weight_decay=0.1), embedding_update="sparse_rows")
