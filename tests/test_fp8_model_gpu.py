"""--precision fp8 through the model and the engine: the encoder layers' linears on e4m3 operands, GELU
with an int8 checkpoint, 8-bit segment inputs, flat gradient slots, graph-captured updates."""
import pytest
import torch

from hetseq_9cme_amd import ops

pytestmark = pytest.mark.gpu


def _encoder(layers=2, hidden=128, inter=384):
    from hetseq_9cme_amd.models.bert import BertConfig, BertEncoder, BertLayer
    torch.manual_seed(0)
    enc = BertEncoder(BertConfig(64, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=hidden // 64,
                                 intermediate_size=inter, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0)).cuda()
    for m in enc.modules():
        if isinstance(m, BertLayer):
            for part in (m.attention.self, m.attention.output, m.intermediate.dense_act, m.output):
                part.fp8 = True
    return enc.train()


def _inputs(B=3, S=40, H=128):
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(B, S, H, generator=g, device='cuda').to(torch.bfloat16)
    mask = torch.ones(B, S, device='cuda')
    mask[1, S // 2:] = 0
    d = torch.randn(B, S, H, generator=g, device='cuda')
    return x, (1 - mask) * -10000.0, d


def _grads(enc, x, bias, d, **kw):
    enc.zero_grad(set_to_none=True)
    x = x.detach().clone().requires_grad_(True)
    out = enc(x, bias, output_all_encoded_layers=False, **kw)[-1]
    out.backward(d.to(out.dtype))
    return out.detach(), x.grad, {n: p.grad for n, p in enc.named_parameters()}


def _near(a, b, rel, what):
    e = ((a.float() - b.float()).norm() / b.float().norm()).item()
    assert e <= rel, (what, e)


def test_encoder_against_reference_path(dev):
    """Kernels against the plain torch path of the same operators (fp32 between them).  The two round
    differently between operators (bf16: 2^-9 of a value); a twentieth of an operand's entries then
    fall on the other side of an e4m3 border and move by a step (2^-4 .. 2^-3): 0.02 of an operand's
    norm, 0.03 of a product of two, and 0.03 sqrt(16) = 0.12 through 2 layers forward and back."""
    enc = _encoder()
    x, bias, d = _inputs()
    out, dx, g = _grads(enc, x, bias, d)
    ops.set_fused(False)
    try:
        rout, rdx, rg = _grads(enc, x, bias, d)
    finally:
        ops.set_fused(True)
    _near(out, rout, 0.06, 'out')
    _near(dx, rdx, 0.12, 'dx')
    for n in g:
        if 'key.bias' in n:   # zero in exact arithmetic: softmax does not see a constant per query
            continue
        _near(g[n], rg[n], 0.12, n)


def test_encoder_8bit_checkpoints(dev):
    """checkpoint_activations=8: the same forward bit for bit; gradients from a recompute on the int8
    copy of a segment's input (error 2^-8 of a block's largest entry, 1 % of a value)."""
    enc = _encoder(layers=4)
    x, bias, d = _inputs()
    out, dx, g = _grads(enc, x, bias, d)
    out8, dx8, g8 = _grads(enc, x, bias, d, checkpoint_activations=8)
    assert torch.equal(out, out8)
    _near(dx8, dx, 0.15, 'dx')
    for n in g:
        if 'key.bias' in n:
            continue
        _near(g8[n], g[n], 0.15, n)


def test_checkpoint_memory(dev):
    """What a checkpointed forward keeps: one byte per element of each segment's input (4 segments of 3
    layers), a little over half of the bf16 copies."""
    enc = _encoder(layers=9)
    x, bias, _ = _inputs(B=8, S=128)
    kept = {}
    for mode in (True, 8):
        h = x.clone().requires_grad_(True)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        out = enc(h, bias, output_all_encoded_layers=False, checkpoint_activations=mode)[-1]
        kept[mode] = torch.cuda.memory_allocated() - base - out.numel() * out.element_size()
        del out, h
    elems = x.numel()
    assert kept[8] <= 3 * elems * (1 + 1 / 128) + 64 * 1024, kept
    assert kept[8] < kept[True], kept


def _ctrl(tmp_path, extra=()):
    from hetseq_9cme_amd import options, tasks
    from hetseq_9cme_amd.controller import Controller
    from hetseq_9cme_amd.data import iterators
    from hetseq_9cme_amd.data.synthetic import BERT_TINY, write_bert_config, write_synthetic_bert_shards
    d = tmp_path / 'data'
    if not d.exists():
        write_synthetic_bert_shards(str(d), n_files=1, samples_per_file=96, seq_len=128, max_pred=20, vocab_size=1024,
                                    split='train')
    cfg = write_bert_config(str(tmp_path / 'c.json'), **BERT_TINY)
    args = options.parse_training_args(['--task', 'bert', '--data', str(d), '--config_file', cfg, '--max-sentences', '8',
                                        '--fast-stat-sync', '--lr', '1e-3', '--num-workers', '1', '--precision', 'fp8',
                                        '--no-save', '--disable-validation', '--distributed-world-size', '1'] + list(extra))
    args.device_id, args.distributed_rank = 0, 0
    torch.manual_seed(args.seed)
    task = tasks.setup_task(args)
    ctrl = Controller(args, task, task.build_model(args))
    itr = iterators.GroupedIterator(ctrl.get_train_iterator(epoch=0, load_dataset=True).next_epoch_itr(shuffle=False), 1)
    return ctrl, itr


def test_engine_updates(dev, tmp_path):
    """Updates through the engine: every encoder linear on the 8-bit path, gradients straight into the
    flat slots, the bf16 shadow of the other weights in sync."""
    ctrl, itr = _ctrl(tmp_path)
    from hetseq_9cme_amd.ops import fp8
    seen = []
    split = fp8.C().split8_weights
    p0 = ctrl.flat.param_flat.clone()

    class Spy(object):
        def __getattr__(self, name):
            f = getattr(ops.C(), name)
            if name != 'split8_weights':
                return f
            return lambda Ws, grad: seen.append(len(Ws)) or split(Ws, grad)
    old, fp8.C = fp8.C, lambda: Spy()
    try:
        for _ in range(3):
            out = ctrl.train_step(next(itr))
    finally:
        fp8.C = old
    torch.cuda.synchronize()
    assert seen == [8, 8, 8]          # 2 layers x 4 weights, one launch per forward
    assert torch.isfinite(out['loss']).all() and not torch.equal(p0, ctrl.flat.param_flat)
    assert torch.equal(ctrl.flat.param_bf16, ctrl.flat.param_flat.to(torch.bfloat16))


def test_slots_hold_the_gradients_autograd_would(dev):
    """The same layer with flat gradient slots (written by the products) and without: equal bits."""
    from hetseq_9cme_amd.parallel.flat_params import FlatParamSpace
    enc = _encoder(layers=1)
    x, bias, d = _inputs()
    _, dx, g = _grads(enc, x, bias, d)
    g = {n: t.clone() for n, t in g.items()}
    enc.zero_grad(set_to_none=True)
    groups = [['layer.0.attention.self.' + n + '.' + k for n in ('query', 'key', 'value')] for k in ('weight', 'bias')]
    flat = FlatParamSpace(enc, dev, contiguous_groups=groups)
    flat.zero_grad()
    h = x.detach().clone().requires_grad_(True)
    out = enc(h, bias, output_all_encoded_layers=False)[-1]
    out.backward(d.to(out.dtype))
    flat.adopt_all()
    torch.cuda.synchronize()
    assert torch.equal(h.grad, dx)
    for n, p in enc.named_parameters():
        assert torch.equal(p.grad, g[n]), n


def test_side_stream_weight_gradients(dev):
    """Weight gradients on the side stream (slots) equal those on the compute stream."""
    from hetseq_9cme_amd.parallel.flat_params import FlatParamSpace
    enc = _encoder(layers=2)
    x, bias, d = _inputs(B=8, S=128)
    flat = FlatParamSpace(enc, dev)
    res = []
    for mode in ('off', 'on'):
        ops.set_side_stream(mode)
        try:
            flat.zero_grad()
            h = x.detach().clone().requires_grad_(True)
            out = enc(h, bias, output_all_encoded_layers=False)[-1]
            out.backward(d.to(out.dtype))
            flat.adopt_all()
        finally:
            ops.set_side_stream('auto')
        torch.cuda.synchronize()
        res.append({n: p.grad.clone() for n, p in enc.named_parameters()})
    for n in res[0]:
        # (the plan for a stream that leaves CUs free may split a reduction differently: fp32 sums of 1024
        # tokens in another order, 64 steps of 2^-23 of the sum of magnitudes, far inside 1e-4 of the norm)
        _near(res[1][n], res[0][n], 1e-4, n)


def test_graph_captured_updates_match_eager(dev, tmp_path):
    from test_train_graph_gpu import _compare

    def run(extra):
        ctrl, itr = _ctrl(tmp_path, extra)
        losses = [float(ctrl.train_step(next(itr))['loss']) for _ in range(8)]
        torch.cuda.synchronize()
        return ctrl, losses, {k: v.detach().float().cpu().clone() for k, v in ctrl.get_model().state_dict().items()}
    eager, graph = run([]), run(['--graph-train-step'])
    # the word-embedding scatter's float atomics reorder between runs; an activation that lands on the
    # other side of a rounding border then moves by an e4m3 step, as in two eager runs: the bound of the
    # bf16 engine (2e-3 of lr-sized updates) widened by the e4m3 step over the bf16 one, capped at 2 %
    _compare(eager, graph, 2e-2)


def test_kept_weights_serve_captured_and_alone(dev):
    """Serving with weights brought to 8 bits once: the outputs of a forward that makes its own codes, for a
    batch and for one short sentence, and from a captured forward replayed on new inputs."""
    enc = _encoder().eval()
    with torch.no_grad():
        ins = [_inputs()[:2], tuple(t[:1, :5].contiguous() for t in _inputs()[:2])]
        ref = [enc(x, b, output_all_encoded_layers=False)[-1] for x, b in ins]
        enc.keep_fp8_weights()
        for (x, b), r in zip(ins, ref):
            assert torch.equal(enc(x, b, output_all_encoded_layers=False)[-1], r)
        x, b = ins[0]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            enc(x, b, output_all_encoded_layers=False)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = enc(x, b, output_all_encoded_layers=False)[-1]
        for i in range(3):
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device='cuda').manual_seed(i), device=dev))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, enc(x, b, output_all_encoded_layers=False)[-1]), i


def test_two_threads_two_streams_one_encoder(dev):
    """One encoder in two threads with a stream each, a training pass beside serving forwards: each result is what
    it is alone."""
    import threading
    enc = _encoder(layers=3)
    for p in enc.parameters():
        p.data = p.data.clone()
    x, bias, d = _inputs(B=4, S=64)
    xs = [x.detach().clone().requires_grad_(True), torch.randn(x.shape, generator=torch.Generator(device='cuda').manual_seed(9), device=dev).to(x.dtype)]

    def train():
        h = xs[0].detach().clone().requires_grad_(True)
        out = enc(h, bias, output_all_encoded_layers=False)[-1]
        return (out.detach(),) + torch.autograd.grad(out, [h] + list(enc.parameters()), d.to(out.dtype))

    def serve():
        with torch.no_grad():
            return (enc(xs[1], bias, output_all_encoded_layers=False)[-1],)
    jobs = [train, serve]
    alone = [job() for job in jobs]
    torch.cuda.synchronize()
    gate, got, errors = threading.Barrier(2), [[], []], []

    def loop(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(12):
                    gate.wait(30)
                    got[i].append(jobs[i]())
            st.synchronize()
        except Exception as e:
            errors.append(e)
            gate.abort()
    ts = [threading.Thread(target=loop, args=(i,)) for i in (0, 1)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors, errors
    for i in (0, 1):
        assert len(got[i]) == 12
        for k, run in enumerate(got[i]):
            assert all(torch.equal(a, b) for a, b in zip(run, alone[i])), (i, k)


def test_captured_forwards_serve_the_weights_kept_last(dev):
    """A forward captured on kept weights, replayed after the weights changed and were kept again, with other
    tensors allocated in between: the new weights' results, without a new capture; after keep=False the last ones."""
    enc = _encoder().eval()
    x, b = _inputs()[:2]
    with torch.no_grad():
        enc.keep_fp8_weights()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            enc(x, b, output_all_encoded_layers=False)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = enc(x, b, output_all_encoded_layers=False)[-1]
        last, others = None, []
        for i in range(3):
            for p in enc.parameters():
                if p.dim() == 2:
                    p.add_(0.02 * torch.randn(p.shape, generator=torch.Generator(device='cuda').manual_seed(i), device=dev))
            with torch.inference_mode(i == 1):
                enc.keep_fp8_weights()
            others += [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (128 * 128, 128 * 384, 384 * 128, 512) for _ in range(16)]
            graph.replay()
            torch.cuda.synchronize()
            ref = enc(x, b, output_all_encoded_layers=False)[-1]
            assert torch.equal(out, ref) and (last is None or not torch.equal(ref, last)), i
            last = ref
        enc.keep_fp8_weights(False)
        others += [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (128 * 128, 128 * 384, 384 * 128, 512) for _ in range(16)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, last)
        graph2 = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match='not inside a graph capture'):
            with torch.cuda.graph(graph2):
                enc.keep_fp8_weights()
