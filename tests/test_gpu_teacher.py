"""lib/teacher.py (models/train_rels.py -distill) and the label decoder's sampled answers (models/eval_rels.py -sample) on the GPU, at the
size smoke() runs: a teacher's records of a batch's rows, the student's loss and gradients against them, labels drawn step by step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def world():
    from dataloaders.synthetic import SyntheticVG, make_blob
    from lib.rel_model import RelModel
    torch.manual_seed(0)
    ds = SyntheticVG(num_images=2, seed=5, n_boxes=6, n_rels=6, im_size=224)

    def model():
        m = RelModel(classes=ds.ind_to_classes, rel_classes=ds.ind_to_predicates, mode='sgcls', num_gpus=1, hidden_dim=128, pooling_dim=4096,
                     nl_obj=2, nl_edge=2, order='leftright', rec_dropout=0.1, use_bias=True, pass_in_obj_feats_to_decoder=False,
                     pass_in_obj_feats_to_edge=False, use_tanh=False, limit_vision=False)
        for p in m.detector.parameters():
            p.requires_grad = False
        m.post_lstm.weight.data.mul_(0.1)
        return m.cuda()
    return ds, make_blob, model


def test_a_student_learns_from_a_teachers_records(world):
    from lib.losses import relation_losses
    from lib.teacher import RelTeacher
    ds, make_blob, model = world
    student = model().train()
    net = model()
    stats = {k: v.clone() for k, v in net.state_dict().items() if 'running' in k}
    teacher = RelTeacher(net, k_obj=16, k_rel=8, temperature=2.0)
    blob = make_blob(ds, [0, 1], is_train=True)
    records = teacher.records(blob, np.random.RandomState(3))
    again = teacher.records(blob, np.random.RandomState(3))
    for a, b in zip(records.obj + records.rel, again.obj + again.rel):
        assert torch.equal(a, b)                                    # no dropout
    for k, v in net.state_dict().items():
        if k in stats:
            assert torch.equal(v, stats[k])                         # no statistics of its own
    student.sampler_rs = np.random.RandomState(3)
    result = student[blob]
    obj, rel = teacher.losses(result, records, scale=0.5)
    assert records.obj.values.shape == (result.rm_obj_dists.shape[0], 16) and records.rel.values.shape == (result.rel_dists.shape[0], 8)
    # the divergences by their definition, in 64 bits
    for got, logits, rec in ((obj, result.rm_obj_dists, records.obj), (rel, result.rel_dists, records.rel)):
        p = torch.softmax(torch.cat((rec.values.double() / 2, rec.rest.double()[:, None]), 1), 1)
        q = torch.softmax(logits.detach().double() / 2, 1)
        qk = q.gather(1, rec.indices.long())
        others = q.scatter(1, rec.indices.long(), 0.0).sum(1, keepdim=True)
        ref = 0.5 * 4.0 * (p * (p.log() - torch.cat((qk, others), 1).log())).sum(1).mean()
        span = float((logits.max(1)[0] - logits.min(1)[0]).max()) / 2 + 7.0 + float(rec.rest.abs().max())
        assert abs(got.item() - ref.item()) <= 0.5 * 4 * 2.0 ** -24 * (16 * span + 8 * span * span)
    (relation_losses(result).sum() + obj + rel).backward()
    grads = [p.grad for p in student.parameters() if p.requires_grad]
    assert all(g is not None and torch.isfinite(g).all() for g in grads)
    assert all(p.grad is None for p in net.parameters())
    student.sampler_rs = np.random.RandomState(4)                   # other rows: refused
    if student[blob].rel_labels.shape != records.rel_labels.shape or not torch.equal(student[blob].rel_labels, records.rel_labels):
        student.sampler_rs = np.random.RandomState(4)
        with pytest.raises(RuntimeError, match='sampler state'):
            teacher.losses(student[blob], records)


def test_sampled_decoding(world):
    ds, make_blob, model = world
    m = model().eval()
    blob = make_blob(ds, [0], is_train=False)
    dec = m.context.decoder_rnn
    m.eval_on_device = True

    def labels():
        with torch.no_grad():
            return m[blob][1].clone()
    greedy = labels()
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(temperature=1e-4, top_p=0.5)):
        dec.sampling = kw
        assert torch.equal(labels(), greedy)
    runs = []
    for seed in (1, 1, 2, 3, 4):
        g = torch.Generator(device='cuda')
        g.manual_seed(seed)
        dec.sampling = dict(temperature=5.0, generator=g)
        runs.append(labels())
    assert torch.equal(runs[0], runs[1])
    assert any(not torch.equal(runs[0], r) for r in runs[2:])
    for r in runs:
        assert int(r.min()) >= 1 and int(r.max()) < m.num_classes
    dec.sampling = None
    assert torch.equal(labels(), greedy)
    from torch.nn.utils.rnn import PackedSequence
    dec.sampling = dict(top_k=3)
    with pytest.raises(ValueError, match='sgdet'):
        dec(PackedSequence(torch.zeros(2, dec.inputs_dim, device='cuda'), torch.tensor([1, 1])), boxes_for_nms=torch.zeros(2, m.num_classes, 4, device='cuda'))
    dec.sampling = None


def test_train_and_eval_commands(tmp_path):
    """models/train_rels.py with a teacher it wrote itself, then models/eval_rels.py with sampled labels, as subprocesses"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, 'neural-motifs_amd')
    base = ['-m', 'sgcls', '-model', 'motifnet', '-order', 'leftright', '-nl_obj', '1', '-nl_edge', '1', '-hidden_dim', '64', '-pooling_dim', '4096', '-ngpu', '1',
            '-synthetic', '8', '-val_size', '2', '-lr', '1e-5', '-p', '1']
    save = str(tmp_path / 'rel')

    def run(script, *more):
        r = subprocess.run([sys.executable, os.path.join(pkg, 'models', script)] + base + list(more), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                           timeout=300, cwd=pkg, env=dict(os.environ, PYTHONPATH=pkg))
        assert r.returncode == 0, r.stdout[-3000:]
        return r.stdout
    run('train_rels.py', '-b', '2', '-nepoch', '1', '-max_iters', '1', '-save_dir', save)
    ckpt = os.path.join(save, 'vgrel-0.tar')
    out = run('train_rels.py', '-b', '2', '-nepoch', '1', '-max_iters', '3', '-distill', ckpt, '-distill_k', '8')
    assert 'distill_loss' in out
    out = run('eval_rels.py', '-b', '1', '-ckpt', ckpt, '-sample', '-sample_temp', '1.5', '-sample_top_k', '20', '-sample_top_p', '0.9')
    assert 'R@100' in out
