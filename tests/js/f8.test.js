// The 8-bit floating-point operators through the JavaScript host. 'cpu': over
// the stand-in addon, what the host checks and what it hands to the library.
// 'gpu': a feed-forward block on the device; the inputs (f32) and the expected
// outputs come from tests/test_js_f8.py in the directory named by argv[3].
import assert from 'assert';
import fs from 'fs';
import path from 'path';
import {test, run} from './harness.js';
import {HipBackend, loadAddon} from '../../stratacuda_amd/src/backend.js';
import {fakeAddon} from './fake_addon.js';

if (process.argv[2] === 'cpu') {
    const real = loadAddon();
    const make = async () => {
        const addon = fakeAddon(real);
        addon.f8Bytes = (...a) => real.f8Bytes(...a);
        addon.f8GateUpWorkspace = (...a) => real.f8GateUpWorkspace(...a);
        for (const f of ['f8Quantize', 'f8Norm', 'f8Project', 'f8GateUp']) addon[f] = (ctx, ...args) => addon.calls.push({name: f, args});
        return {addon, b: await HipBackend.create({addon})};
    };
    test('the addon exports the f8 entries', () => {
        for (const f of ['f8Bytes', 'f8Quantize', 'f8Norm', 'f8Project', 'f8GateUpWorkspace', 'f8GateUp'])
            assert.strictEqual(typeof real[f], 'function', f);
        assert.deepStrictEqual(real.f8Bytes(130, 300, 128), [130 * 384, 8]);
        assert.throws(() => real.f8Bytes(1, 1, 2), RangeError);
        assert.throws(() => real.f8GateUpWorkspace(0, 5), RangeError);
    });
    test('arguments in the library\'s order', async () => {
        const {addon, b} = await make(), X = b.alloc(5 * 300), R = b.alloc(5 * 300), g = b.alloc(300);
        const x = b.f8Matrix(5, 300), w = b.f8Matrix(200, 300, 128), out = b.f8Matrix(5, 200), Y = b.alloc(5 * 210 + 7);
        const ws = b.allocBytes(b.f8GateUpWorkspaceBytes(5, 200));
        assert.strictEqual(w.scales.byteLength, 8);
        b.f8Quantize(X, x); b.f8Quantize(X, w, 'bf16');
        b.f8Norm({X, gamma: g, eps: 1e-6, R, H: R, out: x});
        b.f8Norm({X, type: 'bf16', gamma: g, eps: 0, out: x});
        b.f8Project({X: x, W: w, Y, R: Y, stride: 210, offset: 7});
        b.f8Project({X: x, W: w, Y, type: 'bf16'});
        b.f8GateUp({X: x, Wg: w, Wu: w, out, workspace: ws});
        const c = addon.calls.map(v => v.args);
        assert.deepStrictEqual(c[0], [X.id, 0, 5, 300, 1, x.codes.id, x.scales.id]);
        assert.deepStrictEqual(c[1], [X.id, 1, 200, 300, 128, w.codes.id, w.scales.id]);
        assert.deepStrictEqual(c[2], [X.id, 0, R.id, g.id, 1e-6, 5, 300, R.id, x.codes.id, x.scales.id]);
        assert.deepStrictEqual(c[3], [X.id, 1, 0, g.id, 0, 5, 300, 0, x.codes.id, x.scales.id]);
        assert.deepStrictEqual(c[4], [x.codes.id, x.scales.id, 5, 300, w.codes.id, w.scales.id, 200, Y.id, Y.id, 0, 210, 7]);
        assert.deepStrictEqual(c[5], [x.codes.id, x.scales.id, 5, 300, w.codes.id, w.scales.id, 200, 0, Y.id, 1, 200, 0]);
        assert.deepStrictEqual(c[6], [x.codes.id, x.scales.id, 5, 300, w.codes.id, w.scales.id, w.codes.id, w.scales.id, 200,
            out.codes.id, out.scales.id, ws.id, ws.byteLength]);
        assert.strictEqual(b.dispatches, 7);
    });
    test('refusals', async () => {
        const {addon, b} = await make(), X = b.alloc(1500), Y = b.alloc(1000), ws = b.alloc(1000);
        const x = b.f8Matrix(5, 300), w = b.f8Matrix(200, 300, 128), v = b.f8Matrix(200, 128, 128);
        assert.throws(() => b.f8Quantize(X, x, 'f16'), RangeError);
        assert.throws(() => b.f8Quantize({id: 1}, x), /Invalid HIP X/);
        assert.throws(() => b.f8Quantize(X), /Invalid HIP f8 output/);
        assert.throws(() => b.f8Norm({X, gamma: X, eps: 1e-6, out: w}), /Invalid HIP f8 output/);
        assert.throws(() => b.f8Project({X: w, W: w, Y}), /Invalid HIP f8 X/);
        assert.throws(() => b.f8Project({X: x, W: x, Y}), /Invalid HIP f8 W/);
        assert.throws(() => b.f8Project({X: x, W: v, Y}), RangeError);
        assert.throws(() => b.f8Project({X: x, W: w, Y, offset: -1}), RangeError);
        assert.throws(() => b.f8GateUp({X: x, Wg: w, Wu: v, out: b.f8Matrix(5, 200), workspace: ws}), RangeError);
        assert.throws(() => b.f8GateUp({X: x, Wg: w, Wu: w, out: b.f8Matrix(5, 201), workspace: ws}), RangeError);
        b.free(x.codes);
        assert.throws(() => b.f8Project({X: x, W: w, Y}), /Invalid HIP X/);
        assert.strictEqual(addon.calls.length, 0);
    });
} else {
    const dir = process.argv[3], m = JSON.parse(fs.readFileSync(path.join(dir, 'shape.json'), 'utf8'));
    const load = name => { const b = fs.readFileSync(path.join(dir, name)); return new Float32Array(b.buffer, b.byteOffset, b.byteLength / 4); };
    test('a feed-forward block of ' + m.tokens + ' tokens', async () => {
        const b = await HipBackend.create({device: 0}), {tokens, width, ff} = m;
        const up = name => b.alloc(load(name)), weight = (name, rows, cols) => {
            const out = b.f8Matrix(rows, cols, 128);
            b.f8Quantize(up(name), out);
            return out;
        };
        const Wg = weight('wg.bin', ff, width), Wu = weight('wu.bin', ff, width), Wd = weight('wd.bin', width, ff);
        const n = b.f8Matrix(tokens, width), a = b.f8Matrix(tokens, ff), H = b.alloc(tokens * width);
        b.f8Norm({X: up('x.bin'), R: up('r.bin'), gamma: up('gamma.bin'), eps: 1e-6, H, out: n});
        b.f8GateUp({X: n, Wg, Wu, out: a, workspace: b.allocBytes(b.f8GateUpWorkspaceBytes(tokens, ff))});
        b.f8Project({X: a, W: Wd, Y: H, R: H});
        const y = await b.read(H), want = load('y.bin');
        let worst = 0, size = 0;
        for (let i = 0; i < want.length; i++) { worst += (y[i] - want[i]) ** 2; size += want[i] ** 2; }
        assert.ok(Math.sqrt(worst / size) < m.bound, 'off by ' + Math.sqrt(worst / size));
        assert.throws(() => b.f8Project({X: a, W: Wd, Y: b.alloc(4)}), e => e.code === 'SM_E_BOUNDS');
        await b.dispose();
    });
}

run();
