// Attention over a 4-bit cache through the JavaScript host. 'cpu': over the
// stand-in addon, what the host checks and what it hands to the library.
// 'gpu': a layer's prompt and one more token on the device; the inputs (f32)
// and the expected outputs come from tests/test_js_kv4.py in the directory
// named by argv[3].
import assert from 'assert';
import fs from 'fs';
import path from 'path';
import {test, run} from './harness.js';
import {HipBackend, loadAddon} from '../../stratacuda_amd/src/backend.js';
import {fakeAddon} from './fake_addon.js';

if (process.argv[2] === 'cpu') {
    const real = loadAddon(), launches = ['qkNormRope', 'kv4Write', 'kv4Read', 'kv4Attention'];
    const make = async () => {
        const addon = fakeAddon(real);
        addon.kv4Bytes = (...a) => real.kv4Bytes(...a);
        addon.kv4AttentionWorkspace = (...a) => real.kv4AttentionWorkspace(...a);
        for (const f of launches) addon[f] = (ctx, ...args) => addon.calls.push({name: f, args});
        const b = await HipBackend.create({addon});
        const s = {count: 2, tokens: 5, longest: 4, tablePages: 6, starts: b.alloc(3), lengths: b.alloc(2), table: b.alloc(12)};
        return {addon, b, s, ids: [5, 2, 4, s.starts.id, s.lengths.id, s.table.id, 6]};
    };
    test('the addon exports the entries', () => {
        for (const f of ['kv4Bytes', 'kv4AttentionWorkspace', ...launches]) assert.strictEqual(typeof real[f], 'function', f);
        assert.strictEqual(real.kv4Bytes(7, 3, 200), 7 * 3 * 68 * 256);
        assert.throws(() => real.kv4Bytes(0, 3, 200), RangeError);
        assert.strictEqual(real.kv4AttentionWorkspace(5, 3, 4, 4, 6, 2, 72), 0);
        assert.ok(real.kv4AttentionWorkspace(5, 3, 4, 400, 6, 2, 72) > 0);
        assert.throws(() => real.kv4AttentionWorkspace(5, 3, 4, 4, 6, 4, 72), RangeError);
        for (const f of launches) assert.throws(() => real[f](1, 2), TypeError);
    });
    test('arguments in the library\'s order', async () => {
        const {addon, b, s, ids} = await make(), [Q, K, V, G, Y, c, n, at] = [1, 2, 3, 4, 5, 6, 7, 8].map(() => b.alloc(4000));
        const cache = b.kv4Cache(9, 2, 72), ws = b.allocBytes(64);
        assert.strictEqual(cache.pool.byteLength, 9 * 2 * 68 * 128);
        b.qkNormRope({Q, K, qView: [900, 144, 0], tokens: 5, heads: 6, kvHeads: 2, dim: 72, qGamma: c, kGamma: n, eps: 1e-6, cos: c,
            sin: n, rotary: 36, context: 100, positions: at, Yq: Y, Yk: V});
        b.kv4Write({K, V, vView: [300, 100, 7], type: 'bf16', sequences: s, cache});
        b.kv4Read({K, V, kView: [300, 100, 7], sequences: s, cache});
        b.kv4Attention({Q, sequences: s, cache, heads: 6, scale: 0.1, Y});
        b.kv4Attention({Q, qView: [900, 144, 0], gate: G, gateView: [900, 144, 72], type: 'bf16', sequences: s, cache, heads: 6,
            scale: 0.1, window: 33, Y, workspace: ws});
        const p = cache.pool.id;
        assert.deepStrictEqual(addon.calls.map(v => v.args), [
            [Q.id, [900, 144, 0], K.id, null, 0, 5, 6, 2, 72, c.id, n.id, 1e-6, c.id, n.id, 36, 100, at.id, Y.id, V.id],
            [K.id, null, V.id, [300, 100, 7], 1, ...ids, 2, 72, p, 9],
            [p, 9, 2, 72, ...ids, K.id, [300, 100, 7], V.id, null, 0],
            [Q.id, null, 0, ...ids, p, 9, 6, 2, 72, 0.1, 0, 0, null, Y.id, 0, 0],
            [Q.id, [900, 144, 0], 1, ...ids, p, 9, 6, 2, 72, 0.1, 33, G.id, [900, 144, 72], Y.id, ws.id, ws.byteLength],
        ]);
        assert.strictEqual(b.dispatches, 5);
    });
    test('refusals', async () => {
        const {addon, b, s} = await make(), X = b.alloc(4000), cache = b.kv4Cache(9, 2, 72);
        const a = {Q: X, sequences: s, cache, heads: 6, scale: 0.1, Y: X};
        assert.throws(() => b.kv4Cache(0, 2, 72), RangeError);
        assert.throws(() => b.kv4Attention({...a, type: 'f16'}), RangeError);
        assert.throws(() => b.kv4Attention({...a, Q: {id: 1}}), /Invalid HIP Q/);
        assert.throws(() => b.kv4Attention({...a, cache: undefined}), /Invalid HIP cache/);
        assert.throws(() => b.kv4Attention({...a, sequences: undefined}), /Invalid HIP sequences/);
        assert.throws(() => b.kv4Write({K: X, V: X, sequences: {...s, table: null}, cache}), /Invalid HIP table/);
        assert.throws(() => b.kv4Read({K: X, V: {id: 3}, sequences: s, cache}), /Invalid HIP V/);
        assert.throws(() => b.kv4AttentionWorkspaceBytes(s, 7, cache), RangeError);
        b.free(cache.pool);
        assert.throws(() => b.kv4Attention(a), /Invalid HIP pool/);
        assert.strictEqual(addon.calls.length, 0);
    });
} else {
    const dir = process.argv[3], m = JSON.parse(fs.readFileSync(path.join(dir, 'shape.json'), 'utf8'));
    const load = (name, Type) => { const b = fs.readFileSync(path.join(dir, name)); return new Type(b.buffer, b.byteOffset, b.byteLength / 4); };
    test('a layer\'s attention, ' + m.tokens + ' tokens and one more', async () => {
        const b = await HipBackend.create({device: 0}), {heads, kvHeads, dim, rotary, context} = m;
        const f32 = name => b.alloc(load(name, Float32Array)), i32 = v => b.alloc(Int32Array.from(v), 'i32');
        const cache = b.kv4Cache(m.pages, kvHeads, dim), weights = {qGamma: f32('qg.bin'), kGamma: f32('kg.bin'), cos: f32('cos.bin'), sin: f32('sin.bin')};
        const tokens = m.tokens, table = i32(m.table), both = [[0, tokens, 'y0.bin'], [tokens, 1, 'y1.bin']];
        const full = load('q.bin', Float32Array), keys = load('k.bin', Float32Array), values = load('v.bin', Float32Array);
        for (const [first, n, want] of both) {
            const Q = b.alloc(full.slice(first * heads * 2 * dim, (first + n) * heads * 2 * dim));
            const K = b.alloc(keys.slice(first * kvHeads * dim, (first + n) * kvHeads * dim));
            const V = b.alloc(values.slice(first * kvHeads * dim, (first + n) * kvHeads * dim));
            const Yq = b.alloc(n * heads * dim), Yk = b.alloc(n * kvHeads * dim), Y = b.alloc(n * heads * dim);
            const sequences = {count: 1, tokens: n, longest: n, tablePages: m.table.length, starts: i32([0, n]), lengths: i32([first + n]), table};
            const view = [heads * 2 * dim, 2 * dim, 0], gateView = [heads * 2 * dim, 2 * dim, dim];
            b.qkNormRope({Q, qView: view, K, tokens: n, heads, kvHeads, dim, ...weights, eps: 1e-6, rotary, context,
                positions: i32(Array.from({length: n}, (_, i) => first + i)), Yq, Yk});
            b.kv4Write({K: Yk, V, sequences, cache});
            const bytes = b.kv4AttentionWorkspaceBytes(sequences, heads, cache);
            b.kv4Attention({Q: Yq, sequences, cache, heads, scale: m.scale, gate: Q, gateView, Y, workspace: bytes ? b.allocBytes(bytes) : undefined});
            b.kv4Read({K: Yk, V, sequences, cache});
            const read = await b.read(V), held = load(want === 'y0.bin' ? 'v0.bin' : 'v1.bin', Float32Array);
            assert.deepStrictEqual(Array.from(read), Array.from(held));
            const y = await b.read(Y), expected = load(want, Float32Array);
            let worst = 0, size = 0;
            for (let i = 0; i < expected.length; i++) { worst += (y[i] - expected[i]) ** 2; size += expected[i] ** 2; }
            assert.ok(Math.sqrt(worst / size) < m.bound, 'off by ' + Math.sqrt(worst / size));
            assert.throws(() => b.kv4Attention({Q: Yq, sequences, cache, heads, scale: m.scale, Y: b.alloc(4),
                workspace: bytes ? b.allocBytes(bytes) : undefined}), e => e.code === 'SM_E_BOUNDS');
        }
        await b.dispose();
    });
}

run();
