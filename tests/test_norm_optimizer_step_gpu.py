"""Group norm and orthogonalised updates as a training step uses them: nets with 'act_nm': 'gn' against the fp64 oracle, the
'muon' optimiser's update against its formula on the engine's own gradients, both together over launch modes, checkpoints and
the SNGan / driver entry points."""
import math

import numpy as np
import pytest
import torch

from oracle import restatement as R
from test_muon_gpu import orth64, tolerance

pytestmark = pytest.mark.gpu

AK = float(np.power(64.0, 0.125))


def nhwc(a):
    return torch.as_tensor(np.ascontiguousarray(np.transpose(a, (0, 2, 3, 1)))).cuda()


def dcgan_gn(groups=None):
    """a DCGAN pair with group norm where G has batch norm, and in D (which batch norm would couple across rows)"""
    g = {'act_nm': 'gn', **({'groups': groups} if groups else {})}
    return {'input': [(3, 16, 16)], 'code': [(24, 'linear')],
            'generator': [{'name': 'l1', 'out': 64 * 4 * 4, 'op': 'd', 'act': 'lrelu', 'out_reshape': [64, 4, 4], **g},
                          {'name': 'l2_up', 'out': 32, 'op': 'tc', 'act': 'lrelu', 'kernel': 4, 'strides': 2, **g},
                          {'name': 'l3_up', 'out': 24, 'op': 'tc', 'act': 'tanh', 'kernel': 4, 'strides': 2, **g},
                          {'name': 'l4_t', 'out': 3, 'act': 'tanh'}],
            'discriminator': [{'name': 'l1', 'out': 16, 'act': 'lrelu', 'act_k': AK, 'w_nm': 's', **g},
                              {'name': 'l2_ds', 'out': 32, 'act': 'lrelu', 'kernel': 4, 'strides': 2, **g},
                              {'name': 'l3', 'out': 40, 'act': 'tanh', 'act_k': AK, 'w_nm': 's', 'out_reshape': [8 * 8 * 40], **g},
                              {'name': 'l4', 'op': 'd', 'out': 32, 'act': 'lrelu', 'act_nm': 'gn', 'groups': 4},
                              {'name': 'l5_s', 'out': 16, 'op': 'd', 'act_k': AK, 'bias': 'b', 'w_nm': 's'}]}


def resnet_gn():
    k = [3, 3, 1]
    # (D: four channels or more per group.  One channel per group takes a constant per channel out of a block's branch, the losses do not
    # see one added to every score: a shortcut's bias would have no gradient at all)
    return {'input': [(3, 16, 16)], 'code': [(16, 'linear')],
            'generator': [{'name': 'l1', 'out': 32 * 4 * 4, 'op': 'd', 'out_reshape': [32, 4, 4]},
                          {'name': 'l2_res', 'type': 'res', 'out': 32, 'act': 'lrelu', 'act_nm': 'gn', 'kernel': k, 'scale': ['unpool', 2]},
                          {'name': 'l3_res', 'type': 'res', 'out': 16, 'act': 'lrelu', 'act_nm': 'gn', 'groups': 4, 'kernel': k, 'scale': ['unpool', 2]},
                          {'name': 'l4_gn', 'op': 'i', 'act': 'lrelu', 'act_nm': 'gn', 'groups': 2}, {'name': 'l5_t', 'out': 3, 'act': 'tanh'}],
            'discriminator': [{'name': 'l1_res', 'type': 'res_v1', 'out': 16, 'act': 'lrelu', 'act_k': AK, 'w_nm': 's', 'kernel': k,
                               'scale': ['avg', -2], 'act_nm': 'gn', 'groups': 4},
                              {'name': 'l2_res', 'type': 'res', 'out': 32, 'act': 'lrelu', 'kernel': k, 'scale': ['avg', -2], 'act_nm': 'gn', 'groups': 4},
                              {'name': 'l3_res', 'type': 'res_i', 'out': 32, 'act': 'lrelu', 'act_k': AK, 'w_nm': 's', 'act_nm': 'gn', 'groups': 8,
                               'out_reshape': [4 * 4 * 32]},
                              {'name': 'l4_s', 'out': 16, 'op': 'd', 'act_k': AK, 'w_nm': 's'}]}


def engine(arch, B=8, **kw):
    from mmdgan_hip.tape import TapeEngine
    return TapeEngine(arch, kw.pop('loss', 'rep'), (5e-4, 2e-4), batch_size=B, seed=3, **kw)


def floor(eng, name):
    """the losses depend on differences of scores only: the last bias's gradient is zero, and its computed value the sum of 2B score
    gradients (the first two blocks of the loss's four), each rounded to 2^-24 of itself and added in fp32"""
    return 2.0 ** -22 * float(eng._loss.grads[:2].abs().double().sum()) if name.endswith('_s/bias/bias') else 0.0


def batch(arch, B, rs):
    c, h, w = arch['input'][0]
    return rs.randn(B, arch['code'][0][0]).astype(np.float32), rs.uniform(-1, 1, (B, c, h, w)).astype(np.float32)


@pytest.mark.parametrize('make,mode', [(dcgan_gn, 'eager'), (lambda: dcgan_gn(8), 'plan'), (resnet_gn, 'eager'), (resnet_gn, 'plan')])
def test_step_with_group_norm_matches_the_oracle(make, mode):
    """three steps, each from the oracle's variables: images, scores, losses and every gradient at the bars of the other engine tests
    (1e-4 of a tensor in L2; the losses' floor of 4e-7 of their kernel means).  lrelu and tanh: no activation whose derivative
    a rounding could switch off entirely.
    What a loss may be off by has two parts.  |L - ref| <= |L - L64(s)| + |L64(s) - L64(s_ref)| with s the engine's scores, L64 the loss in
    64 bits: the first is the loss kernel's, the second what scores that are right to fp32 make of a loss that amplifies them.
    First: the kernel forms d^2 = |x|^2 + |y|^2 - 2 x y from sums of 16 fp32 products, each off by 16 * 2^-24 of its terms at most, and adds
    them with two more roundings: off by 18 * 2^-24 * (|x|^2 + |y|^2); exp(-d^2 / 2) by half of that relatively, 18 * 2^-24 * max |s|^2.  (The
    4e-7 of the other tests is for scores of norm 1: here d^2 is about 16, the kernel means being 5e-4.)
    Second: d^2 / 2 about 8, a relative error e of the distances is one of 16 e in every mean; the loss is a difference of means 15 times
    as large: 240 e.  Ten layers of sums of up to 512 fp32 terms leave e = 4e-6 (sqrt(512) roundings each, in quadrature), the loss
    1e-3.  The scores themselves are held in L2."""
    arch, B = make(), 8
    eng = engine(arch, B, launch_mode=mode)
    ora = R.OracleGan(arch, 'rep', (5e-4, 2e-4), dtype=torch.float64, params=eng.get_variables())
    assert sorted(ora.params) == sorted(eng.variable_names())
    assert any('/GN/gamma' in n for n in eng.variable_names()) and eng._d_joint      # (rows of D stay independent under group norm)
    launch, seen = eng._loss.launch, []

    def keep_scores(scores, *a, **kw):                       # (a plan calls it once: its replays write the same buffer)
        seen[:] = [scores, scores.clone()]
        return launch(scores, *a, **kw)
    eng._loss.launch = keep_scores
    rs = np.random.RandomState(5)
    for step in range(3):
        z, real = batch(arch, B, rs)
        eng.set_variables({k: v.numpy().copy() for k, v in ora.params.items()})
        zt, rt = torch.tensor(z, dtype=torch.float64), torch.tensor(real, dtype=torch.float64)
        lg, ld, stats, upd, gd, gg, (gen, s_x, s_gen) = ora.grads(zt, rt)
        ora.step(zt, rt)
        eng.step(nhwc(real), torch.as_tensor(z).cuda())
        fake = np.transpose(eng._dis_in[B:].cpu().numpy(), (0, 3, 1, 2))
        assert np.abs(fake - gen.detach().numpy()).max() <= 1e-4 * np.abs(gen.detach().numpy()).max()
        got = eng.losses.cpu().numpy().astype(np.float64)
        assert mode == 'plan' and step or torch.equal(*seen)                             # (the scores outlive the step)
        s, s64 = seen[0].cpu().double(), torch.cat([s_x, s_gen]).detach()
        assert (s - s64).norm() <= 1e-4 * s64.norm(), step
        own = R.gan_loss(s[B:], s[:B], 'rep', B, rep_weights=eng.rep_weights)
        for i, (ref, mine) in enumerate(zip((float(lg), float(ld)), own)):
            bar = (4e-7 + 18 * 2.0 ** -24 * float((s * s).sum(1).max())) * float(max(got[2:5]))
            assert abs(got[i] - float(mine)) <= 1e-4 * abs(float(mine)) + bar, (step, i, got[i], float(mine))
            assert abs(float(mine) - ref) <= 1e-3 * abs(ref) + bar, (step, i, float(mine), ref)
        if step == 0:
            continue                                     # (gradients of un-normalised start vectors: rounding noise, as in the other step tests)
        grads = eng.get_variables(grad=True)
        for name, ref in {**gd, **gg}.items():
            ref = ref.numpy()
            err = np.linalg.norm(grads[name].astype(np.float64) - ref)
            assert err <= 1e-4 * np.linalg.norm(ref) + floor(eng, name) + 1e-12, (step, name, err, np.linalg.norm(ref))


def test_group_norm_in_d_row_restricted_and_joint_passes_agree(monkeypatch):
    """D's two backward passes together (3B rows) and one by one (B rows of the fake half) give the same gradients"""
    arch, B = resnet_gn(), 6
    z, real = batch(arch, B, np.random.RandomState(1))
    got = []
    for joint in ('1', '0'):
        monkeypatch.setenv('MMDGAN_TAPE_JOINT', joint)
        eng = engine(arch, B)
        assert eng._d_joint == (joint == '1')
        eng.step(nhwc(real), torch.as_tensor(z).cuda())
        got.append(eng.get_variables(grad=True))
    for name in got[0]:
        a, b = got[0][name].astype(np.float64), got[1][name].astype(np.float64)
        assert np.linalg.norm(a - b) <= 1e-4 * np.linalg.norm(a) + 2 * floor(eng, name) + 1e-12, name


def test_inference_and_front_end_run_group_norm():
    """generate / discriminate in inference mode and Routine.__call__: the training forward (group norm has one form)"""
    from GeneralTools.layer_func import Net, Routine
    arch, B = dcgan_gn(), 4
    eng = engine(arch, B)
    z = torch.randn(B, 24, device='cuda')
    img = eng.generate(z, is_training=False).clone()
    ora = R.OracleGan(arch, 'rep', (5e-4, 2e-4), dtype=torch.float64, params=eng.get_variables())
    ref = R.net_forward(ora.gen_specs, ora.params, z.cpu().double(), False)[0]
    assert torch.allclose(img.permute(0, 3, 1, 2).cpu().double(), ref, rtol=1e-4, atol=1e-5)
    net = Net(arch['generator'], net_name='gen')
    r = Routine(net)
    r.add_input_layers([B, 24], [0])
    r.seq_links(list(range(len(arch['generator']))))
    r.add_output_layers([len(arch['generator']) - 1])
    r(z, is_training=False)
    for name, v in eng.get_variables().items():
        if name.startswith('gen/'):
            net.network.set_variable(name, v)
    assert torch.allclose(r(z, is_training=False)['x'], img.permute(0, 3, 1, 2), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize('mode', ['eager', 'plan'])
def test_muon_step_applies_its_formula_to_the_gradients(mode):
    """kernels: momentum, orthogonalised, RMS-matched step; vectors: Adam - from the gradients that the engine itself formed"""
    arch, B = dcgan_gn(), 8
    eng = engine(arch, B, launch_mode=mode, optimizer='muon')
    rs = np.random.RandomState(2)
    mom = {}
    for step in range(3):
        z, real = batch(arch, B, rs)
        before = {k: v.copy() for k, v in eng.get_variables(eng.variable_names(trainable_only=True)).items()}
        m0, v0, t0 = eng.get_adam_state()
        eng.step(nhwc(real), torch.as_tensor(z).cuda())
        after, grads = eng.get_variables(list(before)), eng.get_variables(grad=True)
        for name, p in before.items():
            lr = 5e-4 if name.startswith('dis/') else 2e-4
            g, p = torch.as_tensor(grads[name]).double(), torch.as_tensor(p).double()
            got = torch.as_tensor(after[name]).double()
            if name.endswith('/kernel') or '/kernel_' in name:
                m = 0.95 * torch.as_tensor(m0[name]).double() + g
                u = (g + 0.95 * m).reshape(-1, p.shape[-1])
                o = orth64(u)
                c = lr * 0.2 * math.sqrt(max(u.shape))
                tol = 2 * c * tolerance(u, o) + 2.0 ** -23 * float(2 * p.norm())
                # (grads: the fix-up applied in torch, a rounding or two away from the kernel's)
                assert float((got - (p - (c * o).reshape(p.shape))).norm()) <= tol, (step, name)
                mom[name] = m
            else:
                t = t0 + 1
                m = 0.5 * torch.as_tensor(m0[name]).double() + 0.5 * g
                v = 0.999 * torch.as_tensor(v0[name]).double() + 0.001 * g * g
                ref = p - lr * math.sqrt(1 - 0.999 ** t) / (1 - 0.5 ** t) * m / (v.sqrt() + 1e-8)
                assert (got - ref).abs().max() <= 1e-4 * lr + 2.0 ** -23 * p.abs().max(), (step, name)
        m1, _, t1 = eng.get_adam_state()
        assert t1 == t0 + 1
        for name, m in mom.items():
            assert float((torch.as_tensor(m1[name]).double() - m).norm()) <= 1e-5 * float(m.norm()) + 1e-12, name


def test_launch_modes_checkpoints_and_refusals():
    """a run of both together: eager and plan issue reach the same state to rounding (convolutions sum with atomics; the last bias,
    whose gradient is all rounding, goes where Adam's signs send it and is left out); a restored run continues as the saved
    one; another optimiser's checkpoint is refused"""
    from mmdgan_hip.engine import GanEngine
    arch, B = resnet_gn(), 6
    a, b = engine(arch, B, launch_mode='eager', optimizer='muon'), engine(arch, B, launch_mode='plan', optimizer='muon')
    rs = np.random.RandomState(4)
    data = [batch(arch, B, rs) for _ in range(5)]
    run = lambda e, d: [e.step(nhwc(real), torch.as_tensor(z).cuda()) for z, real in d]
    run(a, data[:3])
    run(b, data[:3])
    va, vb = a.get_variables(), b.get_variables()
    for k in (k for k in va if not k.endswith('_s/bias/bias')):
        assert np.linalg.norm(va[k] - vb[k]) <= 1e-3 * np.linalg.norm(va[k]) + 1e-6, k
    sd = a.state_dict()
    assert sd['optimizer'] == 'muon'
    c = engine(arch, B, launch_mode='plan', optimizer='muon')
    c.load_state_dict(sd)
    assert all(np.array_equal(x, y) for x, y in zip(c.get_adam_state()[0].values(), a.get_adam_state()[0].values()))
    run(a, data[3:])
    run(c, data[3:])
    va, vc = a.get_variables(), c.get_variables()
    for k in (k for k in va if not k.endswith('_s/bias/bias')):
        assert np.linalg.norm(va[k] - vc[k]) <= 1e-3 * np.linalg.norm(va[k]) + 1e-6, k
    with pytest.raises(ValueError, match='optimizer muon'):
        engine(arch, B).load_state_dict(sd)
    with pytest.raises(ValueError, match='optimizer adam'):
        a.load_state_dict(engine(arch, B).state_dict())
    plain = {'input': [(3, 16, 16)], 'code': [(16, 'linear')], 'generator': [{'name': 'l1', 'out': 3 * 16 * 16, 'op': 'd', 'act': 'tanh', 'out_reshape': [3, 16, 16]}],
             'discriminator': [{'name': 'l1', 'out': 8, 'act': 'lrelu', 'out_reshape': [16 * 16 * 8]}, {'name': 'l2', 'out': 4, 'op': 'd'}]}
    with pytest.raises(ValueError, match='runs adam'):
        GanEngine(plain, 'rep', (1e-4, 1e-4), batch_size=4).load_state_dict({**sd})
    with pytest.raises(NotImplementedError, match='optimizer sgd'):
        engine(arch, B, optimizer='sgd')


def test_a_net_without_vectors_and_bad_groups():
    arch = {'input': [(3, 8, 8)], 'code': [(16, 'linear')],
            'generator': [{'name': 'l1', 'out': 3 * 8 * 8, 'op': 'd', 'act': 'tanh', 'bias': None, 'out_reshape': [3, 8, 8]}],
            'discriminator': [{'name': 'l1', 'out': 8, 'act': 'lrelu', 'bias': None, 'out_reshape': [8 * 8 * 8]},
                              {'name': 'l2', 'out': 4, 'op': 'd', 'bias': None}]}
    eng = engine(arch, 4, optimizer='muon')
    z, real = batch(arch, 4, np.random.RandomState(0))
    before = eng.get_variables()
    eng.step(nhwc(real), torch.as_tensor(z).cuda())
    after = eng.get_variables()
    assert all(np.isfinite(after[k]).all() and not np.array_equal(after[k], before[k]) for k in after)
    for groups in (5, 0, 2.0):
        bad = dcgan_gn()
        bad['discriminator'][0]['groups'] = groups
        with pytest.raises(ValueError, match='groups'):
            engine(bad, 4)


def test_sngan_trains_with_muon(tmp_path):
    """the public entry point: SNGan(optimizer='muon').training on synthetic data, through an Agent, and a resumed round"""
    from GeneralTools.misc_fun import FLAGS
    from GeneralTools.graph_func import Agent
    from DeepLearning.my_sngan import SNGan
    saved = (FLAGS.DEFAULT_OUT, FLAGS.SYNTHETIC_DATA)
    FLAGS.DEFAULT_OUT, FLAGS.SYNTHETIC_DATA = str(tmp_path) + '/', True
    try:
        arch = dcgan_gn()
        for round_ in range(2):
            mdl = SNGan(arch, num_class=0, loss_type='rep', optimizer='muon')
            agent = Agent('toy', 'sub', load_ckpt=True, do_save=True, query_step=4, print_loss=False)
            mdl.training('toy', agent, 64, [5e-4, 2e-4], max_step=8, batch_size=8)
            assert mdl.engine.optimizer == 'muon' and mdl.engine.global_step == 8 * (round_ + 1)
        assert all(np.isfinite(v).all() for v in mdl.engine.get_variables().values())
        with pytest.raises(NotImplementedError):
            SNGan(arch, optimizer='rmsprop')
    finally:
        FLAGS.DEFAULT_OUT, FLAGS.SYNTHETIC_DATA = saved
